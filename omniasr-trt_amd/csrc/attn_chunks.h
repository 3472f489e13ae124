// One wave's attention of up to 16 query columns over 32-key tiles, 128 dimensions (a chunk) of K or V at a time, in
// bf16 or e4m3 (gfx950).
//
// The products and lane layouts are those of attn_tiles.h (S^T = K Q^T and O = P V on v_mfma_f32_16x16x32_bf16), with the
// key rows behind pointers of each lane's own: lane (c = lane % 16, g = lane / 16) reads K rows 8 (c / 4) + 4 mb + c % 4
// (mb = 0, 1) and V rows 8g + j (j < 8) of a tile, each within 8 keys in a row, so that a page of 16 or more positions
// holds them.  e4m3 is multiplied as bf16, which holds code * 2^e (e4m3x2_to_bf16).
#pragma once

#include "attn_tiles.h"
#include "paged.h"

namespace omni {

// Inclusive sum over the lanes of a wave.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, true);  // row_bcast 15, 31
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, true);
  return v;
}

// A chunk of a tile: bf16 8 x 16 bytes a lane, e4m3 4.
template <bool kF8>
struct KvChunk {
  u32x4_t r[kF8 ? 4 : 8];
};

// kOnce: memory that no other workgroup reads, loaded past the caches that others' data would stay in.
template <bool kOnce, typename T>
__device__ __forceinline__ T load_as(const char* p) {
  if constexpr (kOnce) return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
  return *reinterpret_cast<const T*>(p);
}

// K: bf16 row mb at r[4 mb + s], dimensions 32s + 8g ..; e4m3 at r[2 mb + p], dimensions 64p + 16g ...  ``row``: row
// c % 4 of the lane's 8 keys, 16g bytes on; rows are kRowB bytes apart.
template <bool kF8, int kRowB, bool kOnce>
__device__ __forceinline__ void load_k_chunk(KvChunk<kF8>& t, const char* row) {
  constexpr int kSteps = kF8 ? 2 : 4;
#pragma unroll
  for (int mb = 0; mb < 2; ++mb)
#pragma unroll
    for (int s = 0; s < kSteps; ++s) t.r[kSteps * mb + s] = load_as<kOnce, u32x4_t>(row + 4 * mb * kRowB + 64 * s);
}

// V row j: dimensions 8c .. + 7 of the chunk.  ``row``: the first of the lane's 8 keys, at its dimensions.
template <bool kF8, int kRowB, bool kOnce>
__device__ __forceinline__ void load_v_chunk(KvChunk<kF8>& t, const char* row) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (kF8) {
      const u32x2_t w = load_as<kOnce, u32x2_t>(row + j * kRowB);
      t.r[j >> 1][2 * (j & 1)] = w[0];
      t.r[j >> 1][2 * (j & 1) + 1] = w[1];
    } else {
      t.r[j] = load_as<kOnce, u32x4_t>(row + j * kRowB);
    }
  }
}

// S^T = K Q^T over a chunk for NB blocks of 16 queries (``scale``: of rows mb = 0, 1; e4m3 only).
template <bool kF8, int NB>
__device__ __forceinline__ void chunk_scores(const KvChunk<kF8>& t, const u32x4_t (&q)[NB][4], const float (&scale)[2],
                                             f32x4_t (&acc)[NB][2]) {
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
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        acc[nb][mb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            __builtin_bit_cast(bf16x8_t, k), __builtin_bit_cast(bf16x8_t, q[nb][s]),
            s == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : acc[nb][mb], 0, 0, 0);
    }
}

// The softmax step of a tile: lane (c, g) holds query c's raw scores of its 8 keys, of which it sees the first ``seen``;
// returns their probabilities relative to the lazy reference maximum (see attend_scored) as the P operand: bf16, what the
// matrix instruction takes, each rounded once (2^-8 of itself at most); their sum stays in fp32, of the unrounded ones.
template <int NB>
__device__ __forceinline__ u32x4_t tile_softmax(const f32x4_t (&acc)[2], float c_scale, SoftmaxState& st,
                                                f32x4_t (&o)[NB], int g, int seen) {
  float sv[8];
  bool over = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    sv[j] = j < seen ? acc[j >> 2][j & 3] : -INFINITY;
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
  float p[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[j], c_scale, -m_use));
    st.l_run += p[j];
  }
  u32x4_t pop;
#pragma unroll
  for (int w = 0; w < 4; ++w)
    pop[w] = __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{p[2 * w], p[2 * w + 1]}), bf16x2_t));
  return pop;
}

// A chunk of V on a tile with keys that some query does not see: their probability is 0, but 0 times an infinity or NaN of
// V would reach the query's output, so the products run without those.  True where there was any: the caller adds them to
// the queries that see them, whose output they make infinite or NaN whatever their weight.  ``vs``: e4m3, the exponent bytes
// of the 8 keys.  A code of e4m3 is a NaN at 0x7f; with an exponent byte b above 246 it is infinite in bf16 from 2^(255-b) on,
// the code 8 * (262 - b); with 255 (never written, but a place not written yet may hold it) all are, 0 too.
template <bool kF8>
__device__ __forceinline__ bool only_finite(KvChunk<kF8>& t, u32x2_t& vs) {
  // What, added to a magnitude that is not finite, carries into the sign's place.
  constexpr uint32_t kField = kF8 ? 0x7f7f7f7fu : 0x7f807f80u, kTop = kF8 ? 0x80808080u : 0x80008000u;
  auto carry = [&](int i, int w) {
    if constexpr (!kF8) return 0x00800080u;
    const int j = 2 * i + (w >> 1), b = (vs[j >> 2] >> (8 * (j & 3))) & 0xff;
    return 0x01010101u * (uint32_t)(b == 255 ? 0x80 : max(8 * (b - 246), 1));
  };
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < (kF8 ? 4 : 8); ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w) any |= (t.r[i][w] & kField) + carry(i, w);
  if (!__any((any & kTop) != 0)) return false;
#pragma unroll
  for (int i = 0; i < (kF8 ? 4 : 8); ++i)
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t top = ((t.r[i][w] & kField) + carry(i, w)) & kTop;
      t.r[i][w] &= ~((top << 1) - (top >> (kF8 ? 7 : 15)));  // every bit of such an element
    }
  if constexpr (kF8) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (((vs[j >> 2] >> (8 * (j & 3))) & 0xff) == 0xff) vs[j >> 2] -= 0x80u << (8 * (j & 3));
  }
  return true;
}

// O += P V over a chunk for NB blocks of 16 queries: block e of o, column c is dimension 8c + e.
template <bool kF8, int NB>
__device__ __forceinline__ void chunk_values(const KvChunk<kF8>& t, const u32x4_t (&pop)[NB], const float (&scale)[8],
                                             f32x4_t (&o)[NB][8]) {
  u32x4_t v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (kF8) {
      v[j] = e4m3x8_to_bf16(u32x2_t{t.r[j >> 1][2 * (j & 1)], t.r[j >> 1][2 * (j & 1) + 1]}, scale[j]);
    } else {
      v[j] = t.r[j];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    u32x4_t b;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      b[w] = __builtin_amdgcn_perm(v[2 * w + 1][e >> 1], v[2 * w][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
      o[nb][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, pop[nb]),
                                                         __builtin_bit_cast(bf16x8_t, b), o[nb][e], 0, 0, 0);
  }
}

// Query c's probability sum, in every lane (c, .).
__device__ __forceinline__ float column_sum(float l_run) {
  l_run += __shfl_xor(l_run, 16, kWave);
  return l_run + __shfl_xor(l_run, 32, kWave);
}

}  // namespace omni
