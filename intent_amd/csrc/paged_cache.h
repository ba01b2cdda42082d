// A paged cache [page][HK][page size] of tokens' heads as the entries get it, and what all of them check of it.
#pragma once

#include "cache4.h"
#include "internal.h"

namespace intent {

// How the cache holds its rows: as the heads do, as E4M3FN codes with a scale for each token and head, or in
// 4 bits with a scale and a lowest value for each group of elements (cache4.h).
enum CacheFormat { kCacheSame = INTENT_CACHE_SAME, kCacheFp8 = INTENT_CACHE_FP8, kCacheInt4 = INTENT_CACHE_INT4 };

constexpr const char* cache_name(int format) {
  return format == kCacheFp8 ? ", fp8 cache" : format == kCacheInt4 ? ", int4 cache" : "";
}

// Of a token's head: elements of the cache's type, scales (or pairs of f16) beside them, and elements of the
// scales' tensor that make one.
struct RowSizes {
  int64_t row, params, each;
};
inline RowSizes row_sizes(int format, int64_t D) {
  if (format == kCacheInt4) return {D / 2, (D + kGroup4 - 1) / kGroup4, 2};
  return {D, format == kCacheFp8 ? 1 : 0, 1};
}

// Page strides in elements.
struct Cache {
  int format;
  const void* k;
  int64_t k_page_ld;
  const void* v;
  int64_t v_page_ld;
  const void* k_params;
  int64_t k_params_ld;
  const void* v_params;
  int64_t v_params_ld;
  int64_t pages, HK, page_size;
};

// Pointers, strides and alignment of a cache that holds something.
inline int check_cache(const Cache& c, int64_t D) {
  const RowSizes sizes = row_sizes(c.format, D);
  const int64_t rows = c.HK * c.page_size, step = c.format == kCacheSame ? 8 : 16;
  const bool one = c.pages == 1, bare = sizes.params == 0;
  INTENT_REQUIRE(c.k && c.v && (bare || (c.k_params && c.v_params)), INTENT_ERR_INVALID_ARGUMENT,
                 "null pointer argument");
  INTENT_REQUIRE(one || (c.k_page_ld >= rows * sizes.row && c.v_page_ld >= rows * sizes.row &&
                         (bare || (c.k_params_ld >= rows * sizes.params * sizes.each &&
                                   c.v_params_ld >= rows * sizes.params * sizes.each))),
                 INTENT_ERR_INVALID_ARGUMENT, "page stride smaller than the page");
  INTENT_REQUIRE(aligned16(c.k) && aligned16(c.v) && (one || (c.k_page_ld % step == 0 && c.v_page_ld % step == 0)) &&
                     (bare || (aligned4(c.k_params) && aligned4(c.v_params) &&
                               (one || (c.k_params_ld % sizes.each == 0 && c.v_params_ld % sizes.each == 0)))),
                 INTENT_ERR_ALIGNMENT, "the cache must be 16-byte aligned with page strides of whole 16 bytes");
  return INTENT_OK;
}

}  // namespace intent
