// Writing and reading a paged key-value cache on gfx950.
//
// Write: the new tokens' q and k rotated as rope_kv_append rotates them (each product rounded on its own), k and v put
// into their pages in bf16 or quantised to e4m3.  A quantised vector x of one (token, kv head) keeps one exponent e, the
// least with max |x| <= 448 * 2^e: x * 2^-e is exact, so a value is rounded once, to the nearest e4m3 (ties to even), and
// what is read back, code * 2^e, is exact in bf16 from e = -124 on (below, multiples of bf16's least number, 2^-133, at most
// half of it off).  (A scale max |x| / 448 would use up to one more binade of e4m3's range
// and cost a second rounding at the division and a third when read; e4m3's relative precision is the same in every
// binade above 2^-6, 14 below the largest.)  k is quantised from the rotated fp32 values, not from their bf16 rounding.
//
// Both kernels are one pass over their bytes, 16 (8 for e4m3) of one vector a thread: a step's launch is latency, a
// prompt's is HBM.  Measured, 8 prompts of 750-2400, 8 heads x 512, e4m3: write 102-105 us (4.6 TB/s), read 43-44 us (6.3).
// Pages go past the caches, which hold what the next kernels read: q, k and v.  The same prompts written and attended to 374 us,
// so 370; 16 rows of 1500 read back for 64 queries each 93, so 91.  All of it past the caches: one prompt of 1433 58, so 71.
#include "common.h"
#include "paged.h"

namespace omni {

// (re, im) -> (re*c - im*s, re*s + im*c), every operation rounded separately.
__device__ __forceinline__ void turn_pair(float& re, float& im, float c, float s) {
#pragma clang fp contract(off)
  const float a = re * c;
  const float b = im * s;
  const float d = re * s;
  const float e = im * c;
  re = a - b;
  im = d + e;
}

// The exponent of a vector whose largest finite |x| has the bits ``top``: 448 = 1.75 * 2^8.  Vectors below 2^-126 * 448
// keep e = -126, so that 2^e and 2^-e are normal numbers.
__device__ __forceinline__ int e4m3_exponent(uint32_t top) {
  const int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return top == 0 ? 0 : max(-126, e);
}

// x * down as e4m3; an infinity, which e4m3 does not have, as NaN.  At the last exponent, 120, values of 248 and more would
// round to 256 * 2^120, which bf16 does not have: they are held at 240.
__device__ __forceinline__ float to_e4m3_range(float x, float down, bool last) {
  const float y = x * down;
  if ((__float_as_uint(x) & 0x7fffffffu) == 0x7f800000u) return __uint_as_float(0x7fc00000u);
  return last && fabsf(y) > 240.f ? copysignf(240.f, y) : y;
}

struct PagedWrite {
  const uint16_t* qkv;  // [tokens, (heads + 2 kv) * D]
  int64_t qkv_stride;
  const float* cs;
  int64_t cs_rows;
  const int64_t* pos;
  const int64_t* slots;
  const int64_t* cache_pos;
  uint16_t* q_out;  // [tokens, heads, D]
  uint16_t* k_out;  // [tokens, kv, D] or nullptr
  int heads;
};

// One workgroup per token; a thread keeps the same 8 dimensions of every vector it takes, so the token's angles are read
// once and its cell is found once.  (Threads over all vectors of all tokens: those prompts written and read back 190 us, so
// 151.)
template <int D, bool kF8>
__global__ __launch_bounds__(256) void paged_write_kernel(PagedWrite w, PagedCache a) {
  constexpr int kLanes = D / 8;  // of one vector; a vector never spans two waves
  constexpr int kBatch = 3;      // vectors in flight
  const int stride = blockDim.x / kLanes;  // vectors at a time
  const int e0 = threadIdx.x % kLanes * 8, vectors = w.heads + 2 * a.kv;
  const int64_t n = blockIdx.x;
  const uint16_t* row = w.qkv + n * w.qkv_stride + e0;
  const int64_t p = w.pos[n];
  const int64_t cell0 = paged_cell(a, w.slots ? w.slots[n] : n, w.cache_pos ? w.cache_pos[n] : p, 0);
  const f32x4_t* angles = reinterpret_cast<const f32x4_t*>(w.cs + clamp64(p, 0, w.cs_rows - 1) * D + e0);
  const f32x4_t t0 = angles[0], t1 = angles[1];
  for (int v0 = threadIdx.x / kLanes; v0 < vectors; v0 += stride * kBatch) {
    u32x4_t raw[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (v0 + k * stride < vectors) raw[k] = *reinterpret_cast<const u32x4_t*>(row + (v0 + k * stride) * D);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int vec = v0 + k * stride;
      if (vec >= vectors) break;
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = bf16x8_elem(raw[k], e);
      u32x4_t bf = raw[k];
      if (vec < w.heads + a.kv) {
        turn_pair(x[0], x[1], t0[0], t0[1]);
        turn_pair(x[2], x[3], t0[2], t0[3]);
        turn_pair(x[4], x[5], t1[0], t1[1]);
        turn_pair(x[6], x[7], t1[2], t1[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) bf[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
      }
      if (vec < w.heads) {
        *reinterpret_cast<u32x4_t*>(w.q_out + (n * w.heads + vec) * D + e0) = bf;
        continue;
      }
      const bool is_k = vec < w.heads + a.kv;
      const int head = vec - w.heads - (is_k ? 0 : a.kv);
      if (is_k && w.k_out) *reinterpret_cast<u32x4_t*>(w.k_out + (n * a.kv + head) * D + e0) = bf;
      if (cell0 < 0) continue;
      const int64_t cell = cell0 + ((int64_t)head << a.page_log2);
      char* pages = is_k ? a.k : a.v;
      if constexpr (!kF8) {
        __builtin_nontemporal_store(bf, reinterpret_cast<u32x4_t*>(pages + (cell * D + e0) * 2));
      } else {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t u = __float_as_uint(x[e]) & 0x7fffffffu;
          top = max(top, u < 0x7f800000u ? u : 0u);
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, kWave));
        const int exponent = e4m3_exponent(top);
        const float down = __uint_as_float((uint32_t)(127 - exponent) << 23);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = to_e4m3_range(x[e], down, exponent == 120);
        u32x2_t codes;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int half = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
          codes[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], half, true);
        }
        __builtin_nontemporal_store(codes, reinterpret_cast<u32x2_t*>(pages + cell * D + e0));
        if (e0 == 0) (is_k ? a.k_scale : a.v_scale)[cell] = (uint8_t)(exponent + 127);
      }
    }
  }
}

struct PagedRead {
  const int64_t* slots;
  const int64_t* pos;
  uint16_t* k;  // [tokens, kv, D]
  uint16_t* v;
};

// One workgroup per token, as paged_write_kernel.
template <int D, bool kF8>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedRead r, PagedCache a) {
  constexpr int kLanes = D / 8, kBatch = 4;
  const int stride = blockDim.x / kLanes;
  const int e0 = threadIdx.x % kLanes * 8, vectors = 2 * a.kv;
  const int64_t n = blockIdx.x;
  const int64_t cell0 = paged_cell(a, r.slots[n], r.pos[n], 0);
  for (int v0 = threadIdx.x / kLanes; v0 < vectors; v0 += stride * kBatch) {
    u32x4_t out[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int vec = v0 + k * stride;
      const bool is_k = vec < a.kv;
      const int64_t cell = cell0 + ((int64_t)(vec - (is_k ? 0 : a.kv)) << a.page_log2);
      const char* pages = is_k ? a.k : a.v;
      out[k] = u32x4_t{0u, 0u, 0u, 0u};
      if (cell0 < 0 || vec >= vectors) continue;
      if constexpr (kF8) {
        out[k] = e4m3x8_to_bf16(__builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(pages + cell * D + e0)),
                                scale_of((is_k ? a.k_scale : a.v_scale)[cell]));
      } else {
        out[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(pages + (cell * D + e0) * 2));
      }
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int vec = v0 + k * stride, head = vec - (vec < a.kv ? 0 : a.kv);
      if (vec >= vectors) break;
      *reinterpret_cast<u32x4_t*>((vec < a.kv ? r.k : r.v) + (n * a.kv + head) * D + e0) = out[k];
    }
  }
}

}  // namespace omni

using namespace omni;

constexpr int64_t kPagedTokens = 0xffffff;  // a launch's threads, 256 to a token at most, are counted in 32 bits

// The instance of ``kernel`` for a head dim and cache type, with whole waves for a token's ``vectors``, four at most.
#define OMNI_PAGED_LAUNCH(kernel, head_dim, vectors, f8, grid, stream, ...)                         \
  do {                                                                                              \
    const int64_t lanes = (int64_t)(vectors) * (head_dim / 8);                                      \
    const int block = lanes >= 256 ? 256 : (int)((lanes + 63) / 64 * 64);                           \
    if (head_dim == 128) {                                                                          \
      if (f8) kernel<128, true><<<grid, block, 0, stream>>>(__VA_ARGS__);                           \
      else kernel<128, false><<<grid, block, 0, stream>>>(__VA_ARGS__);                             \
    } else if (head_dim == 256) {                                                                   \
      if (f8) kernel<256, true><<<grid, block, 0, stream>>>(__VA_ARGS__);                           \
      else kernel<256, false><<<grid, block, 0, stream>>>(__VA_ARGS__);                             \
    } else {                                                                                        \
      if (f8) kernel<512, true><<<grid, block, 0, stream>>>(__VA_ARGS__);                           \
      else kernel<512, false><<<grid, block, 0, stream>>>(__VA_ARGS__);                             \
    }                                                                                               \
  } while (0)

extern "C" int omni_rope_kv_paged(const void* qkv, int64_t qkv_row_stride, const float* cs, int64_t cs_rows,
                                  const int64_t* pos, const int64_t* slots, const int64_t* cache_pos, void* q_out,
                                  void* k_out, void* k_pages, void* v_pages, void* k_scale, void* v_scale,
                                  int32_t pages, int32_t page, const int32_t* table, int64_t table_stride,
                                  int64_t rows, int32_t width, int64_t n_tokens, int32_t heads, int32_t kv_heads,
                                  int32_t head_dim, int32_t cache_dtype, int32_t dtype, void* stream) {
  if (dtype != OMNI_BF16) return OMNI_ERR_DTYPE;
  if (n_tokens < 0 || heads <= 0 || kv_heads <= 0) return OMNI_ERR_INVALID;
  if (n_tokens == 0) return OMNI_OK;
  const int status = omni_check_pages(k_pages, v_pages, k_scale, v_scale, pages, page, kv_heads, head_dim, table,
                                      table_stride, rows, width, cache_dtype);
  if (status != OMNI_OK) return status;
  if (heads > 4096 || kv_heads > 4096 || n_tokens > kPagedTokens) return OMNI_ERR_SHAPE;
  if (k_pages == v_pages || (k_scale && k_scale == v_scale)) return OMNI_ERR_INVALID;  // two vectors for one place
  if (!qkv || !cs || !pos || !q_out || cs_rows <= 0) return OMNI_ERR_INVALID;
  if (((uintptr_t)qkv | (uintptr_t)cs | (uintptr_t)q_out | (uintptr_t)k_out) & 15u) return OMNI_ERR_INVALID;
  if (qkv_row_stride % 8 || qkv_row_stride < (heads + 2LL * kv_heads) * head_dim) return OMNI_ERR_INVALID;
  const PagedWrite w{(const uint16_t*)qkv, qkv_row_stride, cs, cs_rows, pos, slots, cache_pos, (uint16_t*)q_out,
                     (uint16_t*)k_out, heads};
  const PagedCache a =
      omni_paged_cache(k_pages, v_pages, k_scale, v_scale, pages, page, kv_heads, table, table_stride, rows, width);
  const dim3 grid((unsigned)n_tokens);
  OMNI_PAGED_LAUNCH(paged_write_kernel, head_dim, heads + 2 * kv_heads, cache_dtype == OMNI_E4M3, grid, (hipStream_t)stream, w, a);
  return omni_launch_status();
}

extern "C" int omni_paged_read(const void* k_pages, const void* v_pages, const void* k_scale, const void* v_scale,
                               int32_t pages, int32_t page, const int32_t* table, int64_t table_stride, int64_t rows,
                               int32_t width, const int64_t* slots, const int64_t* pos, int64_t n_tokens,
                               int32_t kv_heads, int32_t head_dim, int32_t cache_dtype, void* k_out, void* v_out,
                               void* stream) {
  if (n_tokens < 0 || kv_heads <= 0) return OMNI_ERR_INVALID;
  if (n_tokens == 0) return OMNI_OK;
  const int status = omni_check_pages(k_pages, v_pages, k_scale, v_scale, pages, page, kv_heads, head_dim, table,
                                      table_stride, rows, width, cache_dtype);
  if (status != OMNI_OK) return status;
  if (kv_heads > 4096 || n_tokens > kPagedTokens) return OMNI_ERR_SHAPE;
  if (!slots || !pos || !k_out || !v_out || (((uintptr_t)k_out | (uintptr_t)v_out) & 15u)) return OMNI_ERR_INVALID;
  const PagedRead r{slots, pos, (uint16_t*)k_out, (uint16_t*)v_out};
  const PagedCache a =
      omni_paged_cache(k_pages, v_pages, k_scale, v_scale, pages, page, kv_heads, table, table_stride, rows, width);
  const dim3 grid((unsigned)n_tokens);
  OMNI_PAGED_LAUNCH(paged_read_kernel, head_dim, 2 * kv_heads, cache_dtype == OMNI_E4M3, grid, (hipStream_t)stream, r, a);
  return omni_launch_status();
}
