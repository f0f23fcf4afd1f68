// What the paged key-value cache kernels share: the cache as a kernel sees it
// and the checks of a moe_paged_cache.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include "moe_common.cuh"

namespace moe {

constexpr int kMaxHeadDim = 256;

template <int DT> struct CacheType;
template <> struct CacheType<MOE_CACHE_F16> { using T = __half; };
template <> struct CacheType<MOE_CACHE_BF16> { using T = __nv_bfloat16; };
template <> struct CacheType<MOE_CACHE_E4M3> { using T = __nv_fp8_e4m3; };

inline int cache_elem_bytes(int dtype) { return dtype == MOE_CACHE_E4M3 ? 1 : 2; }

// Strides of axes of extent 1 become 0: nothing is ever added for them.
inline void normalise_strides(moe_paged_cache& c) {
  if (c.pages == 1) c.page_stride = 0;
  if (c.page_size == 1) c.token_stride = 0;
  if (c.kv_heads == 1) c.head_stride = 0;
}

// The cache as the kernels take it, or an error.
inline int take_cache(const moe_paged_cache* cache, moe_paged_cache& c) {
  MOE_REQUIRE(cache, MOE_ERR_INVALID, "null cache");
  c = *cache;
  normalise_strides(c);
  MOE_REQUIRE(c.dtype >= MOE_CACHE_F16 && c.dtype <= MOE_CACHE_E4M3, MOE_ERR_UNSUPPORTED,
              "cache type %d not supported", c.dtype);
  MOE_REQUIRE(c.k && c.v && (c.block_table || c.seqs == 0), MOE_ERR_INVALID, "null cache pointer");
  MOE_REQUIRE(c.pages > 0 && c.page_size > 0 && c.kv_heads > 0 && c.seqs >= 0 &&
                  c.table_width > 0 && c.table_stride >= 0,
              MOE_ERR_INVALID, "bad cache shape");
  MOE_REQUIRE((int64_t)c.table_width * c.page_size <= 0x7fff0000, MOE_ERR_UNSUPPORTED,
              "a sequence of %d pages of %d tokens is longer than 2^31 - 2^16 tokens",
              c.table_width, c.page_size);
  const int eb = cache_elem_bytes(c.dtype), ve = 16 / eb;
  MOE_REQUIRE(c.head_dim > 0 && c.head_dim <= kMaxHeadDim && c.head_dim % ve == 0,
              MOE_ERR_UNSUPPORTED, "head_dim %d: a multiple of %d up to %d is needed", c.head_dim,
              ve, kMaxHeadDim);
  MOE_REQUIRE(((uintptr_t)c.k | (uintptr_t)c.v) % 16 == 0 && c.page_stride % ve == 0 &&
                  c.token_stride % ve == 0 && c.head_stride % ve == 0,
              MOE_ERR_INVALID, "cache bases and strides must be multiples of 16 bytes");
  MOE_REQUIRE(c.page_stride >= 0 && c.token_stride >= 0 && c.head_stride >= 0, MOE_ERR_INVALID,
              "negative cache stride");
  // a tensor map holds no stride of 0 (pages and heads are counted in rows)
  MOE_REQUIRE(c.page_size == 1 || c.token_stride > 0, MOE_ERR_INVALID,
              "slots of a page share memory (token stride 0)");
  if (c.dtype == MOE_CACHE_E4M3)
    MOE_REQUIRE(c.k_scale > 0.f && c.v_scale > 0.f, MOE_ERR_INVALID, "cache scales must be > 0");
  else
    MOE_REQUIRE(c.k_scale == 1.f && c.v_scale == 1.f, MOE_ERR_INVALID,
                "only an e4m3 cache has scales");
  return MOE_OK;
}

// An append writes each row of head_dim elements by itself.
inline int check_cache_rows_apart(const moe_paged_cache& c) {
  const int64_t d = c.head_dim;
  MOE_REQUIRE((c.pages == 1 || c.page_stride >= d) && (c.page_size == 1 || c.token_stride >= d) &&
                  (c.kv_heads == 1 || c.head_stride >= d),
              MOE_ERR_INVALID, "rows of the cache share memory: strides (%lld, %lld, %lld)",
              (long long)c.page_stride, (long long)c.token_stride, (long long)c.head_stride);
  return MOE_OK;
}

}  // namespace moe
