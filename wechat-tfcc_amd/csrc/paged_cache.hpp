// The paged cache of keys and values as kernels see it, and the checks of a call that names one.
#pragma once

#include "common.hpp"

namespace tfcc_rocm {

constexpr unsigned kCacheMostSize = 256;

// Quotients by a number that a launch fixes, without a division: n / d = (n * factor) >> shift for n < 2^31, with shift =
// 31 + ceil(log2 d) and factor = 2^shift / d rounded up.  factor * d exceeds 2^shift by less than d <= 2^(shift - 31), so
// n times the excess stays below 2^shift and the quotient is exact.
struct Divisor {
  unsigned d, factor, shift;
  __host__ static Divisor of(unsigned d) {
    unsigned log = 0;
    while ((1ull << log) < d) ++log;
    return {d, (unsigned)(((1ull << (31 + log)) + d - 1) / d), 31 + log};
  }
  __host__ __device__ unsigned quotient(unsigned n) const { return (unsigned)(((unsigned long long)n * factor) >> shift); }
};

struct CacheView {
  const void *keys, *values;
  const float *key_scales, *value_scales;
  unsigned long long page, head, row;
  unsigned long long scale_page, scale_head, scale_row;
  unsigned pages, heads, size;
  Divisor page_size;
};

inline CacheView view_of(const tfcc_rocm_paged_cache& c) {
  return {c.keys, c.values, c.key_scales, c.value_scales, c.page_stride, c.head_stride, c.row_stride, c.scale_page_stride,
          c.scale_head_stride, c.scale_row_stride, c.pages, c.heads, c.size, Divisor::of(c.page_size)};
}

inline int check_cache(const tfcc_rocm_paged_cache& c, const char* what) {
  TFCC_REQUIRE(c.type == TFCC_ROCM_F32 || c.type == TFCC_ROCM_S8, "%s: a cache of type %d", what, c.type);
  const bool s8 = c.type == TFCC_ROCM_S8;
  const unsigned unit = s8 ? 8 : 4, bytes = s8 ? 8 : 16;
  TFCC_REQUIRE(c.keys && c.values && (!s8 || (c.key_scales && c.value_scales)), "%s: null cache", what);
  TFCC_REQUIRE(c.size > 0 && c.size <= kCacheMostSize && c.size % unit == 0, "%s: heads of %u values (a multiple of %u up to %u)", what,
               c.size, unit, kCacheMostSize);
  TFCC_REQUIRE(c.heads > 0 && c.heads <= 65535, "%s: %u cache heads", what, c.heads);
  TFCC_REQUIRE(c.page_size > 0 && c.page_size <= (1u << 24), "%s: pages of %u rows", what, c.page_size);
  TFCC_REQUIRE(c.pages > 0 && c.pages <= 0x7fffffffu, "%s: %u pages", what, c.pages);
  TFCC_REQUIRE((c.page_stride | c.head_stride | c.row_stride) % unit == 0, "%s: cache strides that are not multiples of %u", what, unit);
  TFCC_REQUIRE((reinterpret_cast<uintptr_t>(c.keys) | reinterpret_cast<uintptr_t>(c.values)) % bytes == 0, "%s: cache memory off %u bytes", what, bytes);
  return TFCC_ROCM_OK;
}

}  // namespace tfcc_rocm
