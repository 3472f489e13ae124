// The paged key-value cache as the kernels see it (gfx950).
//
// Pages [pages, kv, page, D] (``page`` positions, a power of two from 16 to 256), found through ``table`` [rows, width]
// int32: position p of cache row r lives in page table[r, p / page] at offset p % page.  Elements are bf16, or e4m3 with
// one exponent byte b for each (page, kv head, offset) vector: the vector's values are code * 2^(b - 127).
#pragma once

#include "common.h"

namespace omni {

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

struct PagedCache {
  char* k;
  char* v;
  uint8_t* k_scale;  // [pages, kv, page], e4m3 only
  uint8_t* v_scale;
  const int32_t* table;
  int64_t table_stride;
  int64_t rows;       // of the table
  int64_t positions;  // width * page: what a row can hold
  int pages, kv, page_log2;
};

// Vector (page, kv head, offset) of position ``p`` of row ``r`` in the pages, or -1: no such cell.
__device__ __forceinline__ int64_t paged_cell(const PagedCache& a, int64_t r, int64_t p, int head) {
  if (r < 0 || r >= a.rows || p < 0 || p >= a.positions) return -1;
  const int page = a.table[r * a.table_stride + (p >> a.page_log2)];
  if (page < 0 || page >= a.pages) return -1;
  return (((int64_t)page * a.kv + head) << a.page_log2) + (p & ((1 << a.page_log2) - 1));
}

// 2^(b - 127) of an exponent byte.  (b = 0 would be 2^-127, which is no normal number; no vector is written with it.)
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Two e4m3 codes (the low or the high half of ``w``) times ``scale``, a power of two, as bf16: exact from
// 2^-124 on, below to the nearest multiple of bf16's least number, 2^-133 (the least code is 2^-9).
template <bool kHigh>
__device__ __forceinline__ uint32_t e4m3x2_to_bf16(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, kHigh));
}

// Eight e4m3 codes times ``scale`` as eight bf16.
__device__ __forceinline__ u32x4_t e4m3x8_to_bf16(u32x2_t w, float scale) {
  return u32x4_t{e4m3x2_to_bf16<false>(w[0], scale), e4m3x2_to_bf16<true>(w[0], scale),
                 e4m3x2_to_bf16<false>(w[1], scale), e4m3x2_to_bf16<true>(w[1], scale)};
}

}  // namespace omni

// The status of a call's pages and table, OMNI_OK if the kernels can take them.
static inline int omni_check_pages(const void* k_pages, const void* v_pages, const void* k_scale, const void* v_scale,
                                   int32_t pages, int32_t page, int32_t kv, int32_t head_dim, const void* table,
                                   int64_t table_stride, int64_t rows, int32_t width, int32_t cache_dtype) {
  if (cache_dtype != OMNI_BF16 && cache_dtype != OMNI_E4M3) return OMNI_ERR_DTYPE;
  if (pages < 0 || rows < 0 || width < 0 || kv <= 0) return OMNI_ERR_INVALID;
  if (head_dim != 128 && head_dim != 256 && head_dim != 512) return OMNI_ERR_SHAPE;
  if (page < 16 || page > 256 || (page & (page - 1)) != 0) return OMNI_ERR_SHAPE;
  if (!k_pages || !v_pages || !table || table_stride < width) return OMNI_ERR_INVALID;
  if (cache_dtype == OMNI_E4M3 && (!k_scale || !v_scale)) return OMNI_ERR_INVALID;
  if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15u) return OMNI_ERR_INVALID;
  if (((uintptr_t)k_scale | (uintptr_t)v_scale) & 7u) return OMNI_ERR_INVALID;  // read 8 positions at a time
  return OMNI_OK;
}

static inline omni::PagedCache omni_paged_cache(const void* k_pages, const void* v_pages, const void* k_scale,
                                                const void* v_scale, int32_t pages, int32_t page, int32_t kv,
                                                const int32_t* table, int64_t table_stride, int64_t rows,
                                                int32_t width) {
  return omni::PagedCache{(char*)k_pages, (char*)v_pages, (uint8_t*)k_scale, (uint8_t*)v_scale, table, table_stride,
                          rows, (int64_t)width * page, pages, kv, __builtin_ctz((unsigned)page)};
}
