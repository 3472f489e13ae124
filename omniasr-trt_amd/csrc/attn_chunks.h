// One wave's attention of up to 16 query columns over 32-key tiles, 128 dimensions (a chunk) of K or V at a time, in
// bf16 or e4m3 (gfx950).
//
// The products and lane layouts are those of attn_tiles.h (S^T = K Q^T and O = P V on v_mfma_f32_16x16x32_bf16), with the
// key rows behind pointers of each lane's own: lane (c = lane % 16, g = lane / 16) reads K rows 8 (c / 4) + 4 mb + c % 4
// (mb = 0, 1) and V rows 8g + j (j < 8) of a tile, each within 8 keys in a row, so that a page of 16 or more positions
// holds them.  e4m3 is multiplied as bf16: code * 2^e is exact there.
#pragma once

#include "attn_tiles.h"
#include "paged.h"

namespace omni {

// A chunk of a tile: bf16 8 x 16 bytes a lane, e4m3 4.
template <bool kF8>
struct KvChunk {
  u32x4_t r[kF8 ? 4 : 8];
};

// K: bf16 row mb at r[4 mb + s], dimensions 32s + 8g ..; e4m3 at r[2 mb + p], dimensions 64p + 16g ...
template <bool kF8>
__device__ __forceinline__ void load_k_chunk(KvChunk<kF8>& t, const char* row0, const char* row1, int ch, int g) {
  if constexpr (kF8) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      t.r[p] = ld16(row0 + ch * 128 + 64 * p + g * 16);
      t.r[2 + p] = ld16(row1 + ch * 128 + 64 * p + g * 16);
    }
  } else {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      t.r[s] = ld16(row0 + ch * 256 + 64 * s + g * 16);
      t.r[4 + s] = ld16(row1 + ch * 256 + 64 * s + g * 16);
    }
  }
}

// V row j: dimensions 8c .. + 7 of the chunk; rows past ``last`` (of the 8) as row ``last``.  ``row_bytes``: between rows.
template <bool kF8>
__device__ __forceinline__ void load_v_chunk(KvChunk<kF8>& t, const char* rows, int64_t row_bytes, int last, int ch,
                                             int c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const char* row = rows + (j < last ? j : last) * row_bytes;
    if constexpr (kF8) {
      const u32x2_t w = *reinterpret_cast<const u32x2_t*>(row + ch * 128 + c * 8);
      t.r[j >> 1][2 * (j & 1)] = w[0];
      t.r[j >> 1][2 * (j & 1) + 1] = w[1];
    } else {
      t.r[j] = ld16(row + ch * 256 + c * 16);
    }
  }
}

// Query operands of a row of D elements for the scores of the chunks: in the dimensions' order of load_k_chunk.
template <int D, bool kF8>
__device__ __forceinline__ void load_q(u32x4_t (&q)[D / 32], const uint16_t* row, bool live, int g) {
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const int at = kF8 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g;
    q[i] = live ? *reinterpret_cast<const u32x4_t*>(row + at) : u32x4_t{0u, 0u, 0u, 0u};
  }
}

// S^T += K_ch Q_ch^T (``scale``: of rows mb = 0, 1; e4m3 only).
template <bool kF8>
__device__ __forceinline__ void chunk_scores(const KvChunk<kF8>& t, const u32x4_t* q, const float (&scale)[2],
                                             f32x4_t (&acc)[2]) {
#pragma unroll
  for (int mb = 0; mb < 2; ++mb)
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      u32x4_t k;
      if constexpr (kF8) {
        const u32x4_t w = t.r[2 * mb + (s >> 1)];
        k = e4m3x8_to_bf16(u32x2_t{w[2 * (s & 1)], w[2 * (s & 1) + 1]}, scale[mb]);
      } else {
        k = t.r[4 * mb + s];
      }
      acc[mb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, k),
                                                        __builtin_bit_cast(bf16x8_t, q[s]), acc[mb], 0, 0, 0);
    }
}

// The softmax step of a tile: lane (c, g) holds query c's raw scores of keys key0 + j (key0 this lane's), seen below
// ``lim``; probabilities relative to the lazy reference maximum (see attend_scored).
template <int NB>
__device__ __forceinline__ void tile_softmax(const f32x4_t (&acc)[2], float c_scale, SoftmaxState& st, f32x4_t (&o)[NB],
                                             int g, int64_t key0, int64_t lim, float (&p)[8]) {
  float sv[8];
  bool over = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    sv[j] = key0 + j < lim ? acc[j >> 2][j & 3] : -INFINITY;
    over |= sv[j] > st.thr;
  }
  if (__any(over)) {
    float mx = sv[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mx = fmaxf(mx, sv[j]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, kWave));
    mx = fmaxf(mx, __shfl_xor(mx, 32, kWave));
    const float m_new = fmaxf(st.m_ref, mx * c_scale);
    rescale<NB>(st.m_ref, m_new == -INFINITY ? 0.f : m_new, st.l_run, o, g);
    st.m_ref = m_new;
    st.thr = m_new == -INFINITY ? -INFINITY : (m_new + kLazyLog2) / c_scale;
  }
  const float m_use = st.m_ref == -INFINITY ? 0.f : st.m_ref;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[j], c_scale, -m_use));
    st.l_run += p[j];
  }
}

__device__ __forceinline__ bool has_nonfinite(u32x4_t w) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  return bad;
}

// O += P V for a chunk: ``o`` [8], block e column c is dimension 8c + e.  ``edge`` (wave-uniform): some query does not see
// some key of the tile.  Its probability there is 0, but 0 times an infinity or NaN would reach its output, so V rows that
// hold one are left out of the product and added to the queries that see them one by one.
template <bool kF8>
__device__ __forceinline__ void chunk_values(const KvChunk<kF8>& t, const float (&p)[8], const float (&scale)[8],
                                             f32x4_t* o, bool edge, int64_t key0, int64_t lim, int c, int g) {
  u32x4_t v[8], pop;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (kF8) {
      v[j] = e4m3x8_to_bf16(u32x2_t{t.r[j >> 1][2 * (j & 1)], t.r[j >> 1][2 * (j & 1) + 1]}, scale[j]);
    } else {
      v[j] = t.r[j];
    }
  }
#pragma unroll
  for (int w = 0; w < 4; ++w)
    pop[w] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{p[2 * w], p[2 * w + 1]}), bf16x2_t));
  if (edge) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint64_t bad = __ballot(has_nonfinite(v[j]));
      if (!bad) continue;
      const u32x4_t zero = {0u, 0u, 0u, 0u}, row = v[j];
      for (int gk = 0; gk < 4; ++gk) {  // key 8 gk + j of the tile, in lanes 16 gk ..
        if (!((bad >> (16 * gk)) & 0xffffu)) continue;
        if (g == gk) v[j] = zero;
        u32x4_t all;
#pragma unroll
        for (int i = 0; i < 4; ++i) all[i] = (uint32_t)__shfl((int)row[i], 16 * gk + c, kWave);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int from = 16 * gk + 4 * g + i;  // the lane of query 4g + i and this key
          const bool seen = __shfl((int)(key0 + j < lim), from, kWave);
          const float w = round_through_bf16(__shfl(p[j], from, kWave));
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e][i] += seen ? w * bf16x8_elem(all, e) : 0.f;
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    u32x4_t b;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      b[w] = __builtin_amdgcn_perm(v[2 * w + 1][e >> 1], v[2 * w][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
    o[e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, pop), __builtin_bit_cast(bf16x8_t, b),
                                                   o[e], 0, 0, 0);
  }
}

// Query c's probability sum, in every lane (c, .).
__device__ __forceinline__ float column_sum(float l_run) {
  l_run += __shfl_xor(l_run, 16, kWave);
  return l_run + __shfl_xor(l_run, 32, kWave);
}

}  // namespace omni
