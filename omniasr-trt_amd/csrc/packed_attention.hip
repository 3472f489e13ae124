// Causal attention of packed prompts of different lengths on gfx950.
//
// Sequence s: queries starts[s] .. starts[s + 1] - 1 of q [queries, H, D], keys k_starts[s] .. k_starts[s + 1] - 1 of k / v
// [keys, kv, D].  Its query i of nq sees its keys [0, i + nk - nq] of nk (nk > nq: cached keys before the prompt); none
// gives zeros.  Query head h reads kv head h / (H / kv).
#include <math.h>

#include "attn_chunks.h"

namespace omni {

struct PackedAttn {
  const uint16_t* q;  // [queries, H, D]
  const uint16_t* k;  // element strides of a key and of a head
  const uint16_t* v;
  int64_t k_pos, k_head, v_pos, v_head;
  const int64_t* starts;    // [sequences + 1]
  const int64_t* k_starts;  // [sequences + 1]
  int64_t queries, keys;
  int sequences, longest, H, group;
  float scale_log2;
  uint16_t* out;  // [queries, H, D]
};

// Sequence s: its first query and key, and how many there are (within q and k, at most ``longest`` queries).
struct PackedSpan {
  int64_t q0, k0;
  int nq;
  int64_t nk;
};
__device__ __forceinline__ PackedSpan packed_span(const PackedAttn& a, int s) {
  PackedSpan p;
  p.q0 = clamp64(a.starts[s], 0, a.queries);
  p.k0 = clamp64(a.k_starts[s], 0, a.keys);
  const int64_t nq = clamp64(a.starts[s + 1], p.q0, a.queries) - p.q0;
  p.nq = (int)(nq < a.longest ? nq : a.longest);
  p.nk = clamp64(a.k_starts[s + 1], p.k0, a.keys) - p.k0;
  return p;
}

// One wave per (16 queries, head, sequence).
template <int D>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(1))) void packed_attn_kernel(PackedAttn a) {
  constexpr int kChunks = D / 128;
  const int lane = threadIdx.x, c = lane & 15, g = lane >> 4;
  const int h = blockIdx.y, head = h / a.group;
  const PackedSpan sp = packed_span(a, blockIdx.z);
  const int qb = ((int)gridDim.x - 1 - (int)blockIdx.x) * 16;  // the longest blocks first
  if (qb >= sp.nq) return;
  const bool live = qb + c < sp.nq;
  const int64_t before = sp.nk - sp.nq;
  const int64_t lim = live ? clamp64(qb + c + 1 + before, 0, sp.nk) : 0;
  const int64_t total = clamp64(min(qb + 16, sp.nq) + before, 0, sp.nk);  // keys the block's last query sees
  u32x4_t q[D / 32];
  load_q<D, false>(q, a.q + ((sp.q0 + qb + (live ? c : 0)) * a.H + h) * D, live, g);
  f32x4_t o[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  SoftmaxState st{-INFINITY, -INFINITY, 0.f};
  const char* kbase = reinterpret_cast<const char*>(a.k + sp.k0 * a.k_pos + head * a.k_head);
  const char* vbase = reinterpret_cast<const char*>(a.v + sp.k0 * a.v_pos + head * a.v_head);
  const float one[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f}, one2[2] = {1.f, 1.f};
  for (int64_t t = 0; t * 32 < total; ++t) {
    const int64_t rk = t * 32 + 8 * (c >> 2) + (c & 3);
    const char* krow[2] = {kbase + min(rk, total - 1) * a.k_pos * 2, kbase + min(rk + 4, total - 1) * a.k_pos * 2};
    const int64_t vfirst = min(t * 32 + 8 * g, total - 1);
    const int vlast = (int)min(total - 1 - vfirst, (int64_t)7);
    f32x4_t acc[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int ch = 0; ch < kChunks; ++ch) {
      KvChunk<false> k;
      load_k_chunk<false>(k, krow[0], krow[1], ch, g);
      chunk_scores<false>(k, q + 4 * ch, one2, acc);
    }
    float p[8];
    const int64_t key0 = t * 32 + 8 * g;
    tile_softmax<D / 16>(acc, a.scale_log2, st, o, g, key0, lim, p);
    const bool edge = t * 32 + 31 > qb + before;
#pragma unroll
    for (int ch = 0; ch < kChunks; ++ch) {
      KvChunk<false> v;
      load_v_chunk<false>(v, vbase + vfirst * a.v_pos * 2, a.v_pos * 2, vlast, ch, c);
      chunk_values<false>(v, p, one, o + 8 * ch, edge, key0, lim, c, g);
    }
  }
  const float l = column_sum(st.l_run);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float li = __shfl(l, 4 * g + i, kWave);
    if (qb + 4 * g + i >= sp.nq) continue;
    const float div = li == 0.f ? 1.f : li;
    uint16_t* row = a.out + ((sp.q0 + qb + 4 * g + i) * a.H + h) * D + 8 * c;
#pragma unroll
    for (int ch = 0; ch < kChunks; ++ch) {
      u32x4_t w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(o[8 * ch + 2 * e][i] / div, o[8 * ch + 2 * e + 1][i] / div);
      *reinterpret_cast<u32x4_t*>(row + 128 * ch) = w;
    }
  }
}

}  // namespace omni

using namespace omni;

extern "C" int omni_packed_attention(const void* q, const void* k, const void* v, int64_t k_stride_pos,
                                     int64_t k_stride_head, int64_t v_stride_pos, int64_t v_stride_head,
                                     const int64_t* starts, const int64_t* k_starts, int32_t sequences,
                                     int64_t queries, int64_t keys, int32_t longest, int32_t heads, int32_t kv_heads,
                                     int32_t head_dim, float scale, void* out, int32_t dtype, void* stream) {
  if (dtype != OMNI_BF16) return OMNI_ERR_DTYPE;
  if (sequences < 0 || queries < 0 || keys < 0 || longest < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads)
    return OMNI_ERR_INVALID;
  if (head_dim != 128 && head_dim != 256 && head_dim != 512) return OMNI_ERR_SHAPE;
  if (!(scale > 0.f) || scale == INFINITY) return OMNI_ERR_INVALID;
  if (sequences == 0 || queries == 0 || longest == 0) return OMNI_OK;
  if (!q || !starts || !k_starts || !out || (keys > 0 && (!k || !v))) return OMNI_ERR_INVALID;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k | (uintptr_t)v) & 15u) return OMNI_ERR_INVALID;
  if ((k_stride_pos | k_stride_head | v_stride_pos | v_stride_head) & 7) return OMNI_ERR_INVALID;
  if (k_stride_pos < 0 || k_stride_head < 0 || v_stride_pos < 0 || v_stride_head < 0) return OMNI_ERR_INVALID;
  if (sequences > 65535 || heads > 65535) return OMNI_ERR_SHAPE;
  const PackedAttn a{(const uint16_t*)q, (const uint16_t*)k, (const uint16_t*)v, k_stride_pos, k_stride_head,
                     v_stride_pos, v_stride_head, starts, k_starts, queries, keys, sequences, longest, heads,
                     heads / kv_heads, scale * 1.4426950408889634f, (uint16_t*)out};
  const dim3 grid((longest + 15) / 16, heads, sequences);
  const hipStream_t s = (hipStream_t)stream;
  if (head_dim == 128) packed_attn_kernel<128><<<grid, 64, 0, s>>>(a);
  else if (head_dim == 256) packed_attn_kernel<256><<<grid, 64, 0, s>>>(a);
  else packed_attn_kernel<512><<<grid, 64, 0, s>>>(a);
  return omni_launch_status();
}
