// Attention of a step's new tokens over a paged key-value cache on gfx950.
//
// Query i of row b (i < T) sees keys [0, lengths[b] + i) of the row's pages:
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q.k_j,  m = max_j s_j, zeros where there is no key.
// The unit of work is (row, kv head, block of 16 query columns): the T * group queries that read one kv head's keys are
// its columns, column i * group + j being token i's head kv * group + j, so that grouped heads and drafts share one read of
// the keys.  A unit's 32-key tiles are split over workgroups of one wave; each leaves (O, m, l) in fp32 and a second launch
// joins them: w_s = exp(m_s - max m), out = sum w_s O_s / sum w_s l_s.
#include <math.h>

#include "attn_chunks.h"

namespace omni {

struct PagedAttn {
  const uint16_t* q;  // [rows * T, H, D]
  PagedCache cache;
  const int64_t* lengths;
  int T, H, group, cols, qblocks, splits;
  float scale_log2;
  float* part_o;   // [unit][split][16][D]
  float* part_ml;  // [unit][split][16][2]
  uint16_t* out;   // [rows * T, H, D]
};

// Keys that the row's first and last query see.
struct PagedReach {
  int64_t first, last;
};
__device__ __forceinline__ PagedReach paged_reach(const PagedAttn& a, int b) {
  const int64_t n = clamp64(a.lengths[b], 0, a.cache.positions);
  const int64_t last = n + a.T - 1;
  return {n, last < a.cache.positions ? last : a.cache.positions};
}

template <int D, bool kF8>
__global__ __launch_bounds__(64) __attribute__((amdgpu_waves_per_eu(1))) void paged_attn_kernel(PagedAttn a) {
  constexpr int kChunks = D / 128, kRowB = D * (kF8 ? 1 : 2);
  const int lane = threadIdx.x, c = lane & 15, g = lane >> 4;
  const int sp = blockIdx.x, head = blockIdx.y / a.qblocks, qblk = blockIdx.y % a.qblocks, b = blockIdx.z;
  const int col = 16 * qblk + c, token = col / a.group;
  const bool live = col < a.cols;
  const PagedReach reach = paged_reach(a, b);
  const int64_t tiles = (reach.last + 31) / 32;
  const int64_t t0 = tiles * sp / a.splits, t1 = tiles * (sp + 1) / a.splits;
  const int64_t lim = live ? (reach.first + token < reach.last ? reach.first + token : reach.last) : 0;

  u32x4_t q[D / 32];
  load_q<D, kF8>(q, a.q + (((int64_t)b * a.T + (live ? token : 0)) * a.H + head * a.group + col % a.group) * D, live, g);
  f32x4_t o[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  SoftmaxState st{-INFINITY, -INFINITY, 0.f};
  const int64_t last_group = (reach.last - 1) >> 3;  // 8 keys in a row: all on one page
  // The cell of a group's first key (a page number out of the table's range is held in it).
  auto cell = [&](int64_t group) {
    const int64_t p = group * 8;
    int page = a.cache.table[b * a.cache.table_stride + (p >> a.cache.page_log2)];
    page = min(max(page, 0), a.cache.pages - 1);
    return (((int64_t)page * a.cache.kv + head) << a.cache.page_log2) + (p & ((1 << a.cache.page_log2) - 1));
  };
  for (int64_t t = t0; t < t1; ++t) {
    // Groups past the last key are read as the last one, keys past it as it: a key in use, masked.
    const int64_t kgroup = min(t * 4 + (c >> 2), last_group), vgroup = min(t * 4 + g, last_group);
    const int klast = (int)min(reach.last - 1 - kgroup * 8, (int64_t)7);
    const int vlast = (int)min(reach.last - 1 - vgroup * 8, (int64_t)7);
    const int64_t kcell = cell(kgroup), vcell = cell(vgroup);
    const int r0 = min(c & 3, klast), r1 = min(4 + (c & 3), klast);
    const char* krow[2] = {a.cache.k + (kcell + r0) * kRowB, a.cache.k + (kcell + r1) * kRowB};
    const char* vrows = a.cache.v + vcell * kRowB;
    float kscale[2] = {1.f, 1.f}, vscale[8];
    if constexpr (kF8) {
      kscale[0] = scale_of(a.cache.k_scale[kcell + r0]);
      kscale[1] = scale_of(a.cache.k_scale[kcell + r1]);
      const u32x2_t w = *reinterpret_cast<const u32x2_t*>(a.cache.v_scale + vcell);
#pragma unroll
      for (int j = 0; j < 8; ++j) vscale[j] = scale_of((w[j >> 2] >> (8 * (j & 3))) & 0xffu);
    }
    f32x4_t acc[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int ch = 0; ch < kChunks; ++ch) {
      KvChunk<kF8> k;
      load_k_chunk<kF8>(k, krow[0], krow[1], ch, g);
      chunk_scores<kF8>(k, q + 4 * ch, kscale, acc);
    }
    float p[8];
    const int64_t key0 = t * 32 + 8 * g;
    tile_softmax<D / 16>(acc, a.scale_log2, st, o, g, key0, lim, p);
    const bool edge = t * 32 + 31 >= reach.first;
#pragma unroll
    for (int ch = 0; ch < kChunks; ++ch) {
      KvChunk<kF8> v;
      load_v_chunk<kF8>(v, vrows, kRowB, vlast, ch, c);
      chunk_values<kF8>(v, p, vscale, o + 8 * ch, edge, key0, lim, c, g);
    }
  }
  const int64_t part = (((int64_t)b * gridDim.y + blockIdx.y) * a.splits + sp) * 16;
  const float l = column_sum(st.l_run);
  if (g == 0) {
    a.part_ml[(part + c) * 2] = st.m_ref;
    a.part_ml[(part + c) * 2 + 1] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (16 * qblk + 4 * g + i >= a.cols) continue;
    float* row = a.part_o + (part + 4 * g + i) * D + 8 * c;
#pragma unroll
    for (int ch = 0; ch < kChunks; ++ch)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<f32x4_t*>(row + 128 * ch + 4 * h) =
            f32x4_t{o[8 * ch + 4 * h][i], o[8 * ch + 4 * h + 1][i], o[8 * ch + 4 * h + 2][i], o[8 * ch + 4 * h + 3][i]};
  }
}

// One workgroup per (query, head): the splits' partials joined, 8 dimensions a thread.
template <int D>
__global__ __launch_bounds__(D / 8) void paged_attn_merge_kernel(PagedAttn a) {
  const int64_t row = blockIdx.x;
  const int h = blockIdx.y, token = (int)(row % a.T), head = h / a.group, col = token * a.group + h % a.group;
  const int64_t unit = ((row / a.T) * (a.H / a.group) + head) * a.qblocks + col / 16;
  const int64_t part = unit * a.splits * 16 + col % 16;
  float m = -INFINITY;
  for (int s = 0; s < a.splits; ++s) {
    const float ms = a.part_ml[(part + 16 * s) * 2];
    m = ms > m || ms != ms ? ms : m;
  }
  float l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const float ms = a.part_ml[(part + 16 * s) * 2];
    if (ms == -INFINITY) continue;  // no key seen
    const float w = __builtin_amdgcn_exp2f(ms - m);
    l += w * a.part_ml[(part + 16 * s) * 2 + 1];
    const f32x4_t* po = reinterpret_cast<const f32x4_t*>(a.part_o + (part + 16 * s) * D + 8 * threadIdx.x);
    const f32x4_t p0 = po[0], p1 = po[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      o[e] += w * p0[e];
      o[4 + e] += w * p1[e];
    }
  }
  const float div = l == 0.f ? 1.f : l;
  u32x4_t out;
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = pack_bf16x2(o[2 * i] / div, o[2 * i + 1] / div);
  *reinterpret_cast<u32x4_t*>(a.out + (row * a.H + h) * D + 8 * threadIdx.x) = out;
}

// Splits of a unit: enough one-wave workgroups for four waves on each CU, at most one for every 64 keys of the table.
inline int paged_splits(int64_t units, int64_t positions) {
  const int64_t want = 1024 / (units < 1 ? 1 : units), most = (positions + 63) / 64;
  const int64_t s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 128 ? 128 : s);
}

}  // namespace omni

using namespace omni;

static int64_t paged_attn_units(int64_t rows, int32_t tokens, int32_t heads, int32_t kv_heads) {
  const int64_t cols = (int64_t)tokens * (heads / kv_heads);
  return rows * kv_heads * ((cols + 15) / 16);
}

extern "C" size_t omni_paged_attention_workspace(int64_t rows, int32_t tokens, int32_t heads, int32_t kv_heads,
                                                 int32_t head_dim, int32_t page, int32_t width) {
  if (rows <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || head_dim <= 0) return 0;
  const int64_t units = paged_attn_units(rows, tokens, heads, kv_heads);
  const int64_t parts = units * paged_splits(units, (int64_t)width * page) * 16;
  return (size_t)(parts * (head_dim + 2) * 4);
}

extern "C" int omni_paged_attention(const void* q, const void* k_pages, const void* v_pages, const void* k_scale,
                                    const void* v_scale, int32_t pages, int32_t page, const int32_t* table,
                                    int64_t table_stride, int32_t width, const int64_t* lengths, int32_t rows,
                                    int32_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim, float scale,
                                    void* out, void* workspace, size_t workspace_bytes, int32_t cache_dtype,
                                    int32_t dtype, void* stream) {
  if (dtype != OMNI_BF16) return OMNI_ERR_DTYPE;
  if (rows < 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return OMNI_ERR_INVALID;
  if (tokens > 16 || heads > 4096) return OMNI_ERR_SHAPE;
  if (!(scale > 0.f) || scale == INFINITY) return OMNI_ERR_INVALID;
  if (rows == 0) return OMNI_OK;
  const int status = omni_check_pages(k_pages, v_pages, k_scale, v_scale, pages, page, kv_heads, head_dim, table,
                                      table_stride, rows, width, cache_dtype);
  if (status != OMNI_OK) return status;
  if (pages == 0 || width == 0) return OMNI_ERR_INVALID;
  if (!q || !lengths || !out || (((uintptr_t)q | (uintptr_t)out) & 15u)) return OMNI_ERR_INVALID;
  if (rows > 65535) return OMNI_ERR_SHAPE;
  if (!workspace || ((uintptr_t)workspace & 255u) ||
      workspace_bytes < omni_paged_attention_workspace(rows, tokens, heads, kv_heads, head_dim, page, width))
    return OMNI_ERR_WORKSPACE;
  PagedAttn a;
  a.q = (const uint16_t*)q;
  a.cache = omni_paged_cache(k_pages, v_pages, k_scale, v_scale, pages, page, kv_heads, table, table_stride, rows, width);
  a.lengths = lengths;
  a.T = tokens;
  a.H = heads;
  a.group = heads / kv_heads;
  a.cols = tokens * a.group;
  a.qblocks = (a.cols + 15) / 16;
  const int64_t units = paged_attn_units(rows, tokens, heads, kv_heads);
  a.splits = paged_splits(units, a.cache.positions);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + units * a.splits * 16 * head_dim;
  a.out = (uint16_t*)out;
  const hipStream_t s = (hipStream_t)stream;
  const dim3 grid(a.splits, kv_heads * a.qblocks, rows), merge((unsigned)(rows * tokens), heads);
  const bool f8 = cache_dtype == OMNI_E4M3;
  if (head_dim == 128) {
    if (f8) paged_attn_kernel<128, true><<<grid, 64, 0, s>>>(a);
    else paged_attn_kernel<128, false><<<grid, 64, 0, s>>>(a);
    paged_attn_merge_kernel<128><<<merge, 16, 0, s>>>(a);
  } else if (head_dim == 256) {
    if (f8) paged_attn_kernel<256, true><<<grid, 64, 0, s>>>(a);
    else paged_attn_kernel<256, false><<<grid, 64, 0, s>>>(a);
    paged_attn_merge_kernel<256><<<merge, 32, 0, s>>>(a);
  } else {
    if (f8) paged_attn_kernel<512, true><<<grid, 64, 0, s>>>(a);
    else paged_attn_kernel<512, false><<<grid, 64, 0, s>>>(a);
    paged_attn_merge_kernel<512><<<merge, 64, 0, s>>>(a);
  }
  return omni_launch_status();
}
