// Keys and values into a paged cache, and sequences back out of it.  Bound: HBM (a few launches' latency for single tokens).
//
// Write: a row is one head of one token.  Its lanes hold four values each (a power of two of lanes, 16 to 64, several rows to a
// wavefront), so the row is read once: the largest absolute value is joined over its lanes, and
//   scale = amax * (1 / 127) (float32),  n = x / scale rounded to nearest, ties to even.
// The quotient is not formed: n is taken from x * (1 / scale), which can miss only next to a border, and the remainder x - n * scale,
// which a fused multiply-add gives exactly there (|x| <= 127.5 scale, so it is a multiple of the smaller last place of x and scale
// and at most about scale / 2: 24 bits hold it), moves it to the neighbour or, on a tie, to the even one.  So every
// integer is that of the true quotient, at eight operations instead of a 64-bit division.
// What is read and written once, the rows on their way in and out, passes the caches by, so that the int8 rows stay in the last level for
// those who read them next (16 prompts of up to 2048 tokens of 8 x 128, written and read back, 274 MB each way: 75 + 73 us without, 81 + 49, 3.4 and 5.6 TB/s, with).
// The amax is formed on the bits of |x|, which order infinities and NaNs above all numbers: a row with one gets a scale that is not
// finite, integers 0, and reads back as NaN.
#include "paged_cache.hpp"

namespace tfcc_rocm {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // needs no more than a float's alignment

struct WriteArgs {
  CacheView cache;
  const float *keys, *values;
  unsigned long long key_token, key_head, value_token, value_head;
  const void* slots;
  int wide_slots;
  unsigned tokens, rows;  // rows = tokens * heads
  Divisor heads;
};

constexpr unsigned kCacheThreads = 256;

// largest of the LANES lanes of a row, as bits
template <int LANES>
__device__ __forceinline__ unsigned row_max(unsigned u) {
#pragma unroll
  for (int m = LANES / 2; m > 0; m /= 2) {
    const unsigned o = (unsigned)__shfl_xor((int)u, m, 64);
    u = u > o ? u : o;
  }
  return u;
}

__device__ __forceinline__ int nearest(float x, float scale, float inverse) {
  float n = rintf(x * inverse);
  const float left = fmaf(-n, scale, x), half = 0.5f * scale;
  const bool odd = ((int)n & 1) != 0;
  if (left > half || (left == half && odd)) n += 1.0f;
  else if (left < -half || (left == -half && odd)) n -= 1.0f;
  return (int)fminf(fmaxf(n, -127.0f), 127.0f);
}

template <bool S8, int LANES>
__global__ __launch_bounds__(kCacheThreads) void cache_write_kernel(WriteArgs p) {
  const unsigned row = blockIdx.x * (kCacheThreads / LANES) + threadIdx.x / LANES, d = (threadIdx.x % LANES) * 4;
  if (row >= p.rows) return;
  const unsigned token = p.heads.quotient(row), head = row - token * p.heads.d;
  const long long slot = p.wide_slots ? static_cast<const long long*>(p.slots)[token] : static_cast<const int*>(p.slots)[token];
  if (slot < 0 || slot >= (long long)p.cache.pages * p.cache.page_size.d) return;
  // (a division of 64 bits takes as long as a sixth of all the rest)
  const unsigned long long page = slot < 0x80000000ll ? p.cache.page_size.quotient((unsigned)slot) : (unsigned long long)slot / p.cache.page_size.d;
  const unsigned inside = (unsigned)(slot - page * p.cache.page_size.d);
  const bool value = blockIdx.y != 0;
  const float* in = value ? p.values + token * p.value_token + head * p.value_head : p.keys + token * p.key_token + head * p.key_head;
  const unsigned long long at = page * p.cache.page + head * p.cache.head + inside * p.cache.row;
  const bool mine = d < p.cache.size;
  f32x4 x = {0, 0, 0, 0};
  if (mine) x = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(in + d));
  if constexpr (!S8) {
    float* out = static_cast<float*>(const_cast<void*>(value ? p.cache.values : p.cache.keys)) + at;
    if (mine) *reinterpret_cast<f32x4*>(out + d) = x;
  } else {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned u = __float_as_uint(x[i]) & 0x7fffffffu;
      top = top > u ? top : u;
    }
    top = row_max<LANES>(top);
    const float scale = __uint_as_float(top) * (1.0f / 127.0f);
    int n[4] = {0, 0, 0, 0};
    if (top < 0x7f800000u && scale > 0.0f) {
      // a subnormal scale has no finite reciprocal: both are lifted by 2^64, which changes no quotient
      const float lift = scale < 1e-30f ? 18446744073709551616.0f : 1.0f, s = scale * lift, inverse = 1.0f / s;
#pragma unroll
      for (int i = 0; i < 4; ++i) n[i] = nearest(x[i] * lift, s, inverse);
    }
    int8_t* out = static_cast<int8_t*>(const_cast<void*>(value ? p.cache.values : p.cache.keys)) + at;
    if (mine)
      *reinterpret_cast<unsigned*>(out + d) = ((unsigned)n[0] & 255u) | ((unsigned)n[1] & 255u) << 8 | ((unsigned)n[2] & 255u) << 16 | (unsigned)n[3] << 24;
    if (d == 0)
      const_cast<float*>(value ? p.cache.value_scales : p.cache.key_scales)[page * p.cache.scale_page + head * p.cache.scale_head + inside * p.cache.scale_row] = scale;
  }
}

struct ReadArgs {
  CacheView cache;
  const int* table;
  unsigned long long table_stride;
  unsigned table_width, batch;
  const int* starts;
  unsigned tokens;
  float *keys, *values;
};

constexpr unsigned kReadTokens = 4;  // of a workgroup

// LANES lanes of four values to a row, as above; a workgroup finds its tokens' slots once for all their heads.
template <bool S8, int LANES>
__global__ __launch_bounds__(kCacheThreads) void cache_read_kernel(ReadArgs p) {
  __shared__ unsigned pages[kReadTokens], insides[kReadTokens];
  constexpr unsigned kOutside = 0xffffffffu, kBehind = 0xfffffffeu;
  const unsigned first = blockIdx.x * kReadTokens;
  if (threadIdx.x < kReadTokens) {
    const int token = (int)(first + threadIdx.x);
    unsigned page = kBehind, inside = 0;
    if (token < (int)p.tokens && token < p.starts[p.batch] && token >= p.starts[0]) {
      unsigned lo = 0, hi = p.batch;  // starts[lo] <= token < starts[hi]
      while (hi - lo > 1) {
        const unsigned mid = (lo + hi) / 2;
        if (p.starts[mid] <= token) lo = mid;
        else hi = mid;
      }
      const unsigned at = (unsigned)(token - p.starts[lo]), index = p.cache.page_size.quotient(at);
      inside = at - index * p.cache.page_size.d;
      page = kOutside;
      if (index < p.table_width) {
        const int named = p.table[lo * p.table_stride + index];
        if (named >= 0 && (unsigned)named < p.cache.pages) page = (unsigned)named;
      }
    }
    pages[threadIdx.x] = page;
    insides[threadIdx.x] = inside;
  }
  __syncthreads();
  const bool value = blockIdx.y != 0;
  const unsigned d = (threadIdx.x % LANES) * 4;
  if (d >= p.cache.size) return;
  float* const out = value ? p.values : p.keys;
  const void* const held = value ? p.cache.values : p.cache.keys;
  const float* const scales = value ? p.cache.value_scales : p.cache.key_scales;
  constexpr unsigned step = kCacheThreads / LANES;
  for (unsigned t = 0; t < kReadTokens; ++t) {
    const unsigned page = pages[t], inside = insides[t];
    if (page == kBehind) continue;
    for (unsigned head = threadIdx.x / LANES; head < p.cache.heads; head += step) {
      f32x4 x = {0, 0, 0, 0};
      if (page != kOutside) {
        const unsigned long long at = page * p.cache.page + head * p.cache.head + inside * p.cache.row + d;
        if constexpr (S8) {
          const unsigned n = *reinterpret_cast<const unsigned*>(static_cast<const int8_t*>(held) + at);
          const float scale = scales[page * p.cache.scale_page + head * p.cache.scale_head + inside * p.cache.scale_row];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(n >> (8 * i)) * scale;
        } else {
          x = *reinterpret_cast<const f32x4*>(static_cast<const float*>(held) + at);
        }
      }
      __builtin_nontemporal_store(x, reinterpret_cast<f32x4_any*>(out + ((unsigned long long)(first + t) * p.cache.heads + head) * p.cache.size + d));
    }
  }
}

}  // namespace
}  // namespace tfcc_rocm

using namespace tfcc_rocm;

extern "C" {

int tfcc_rocm_cache_write(void* stream, const tfcc_rocm_paged_cache* cache, const float* keys, uint64_t key_token_stride,
                          uint64_t key_head_stride, const float* values, uint64_t value_token_stride,
                          uint64_t value_head_stride, unsigned tokens, const void* slots, int slot_type) {
  TFCC_REQUIRE(cache != nullptr, "cache_write: null cache");
  if (int e = check_cache(*cache, "cache_write")) return e;
  TFCC_REQUIRE(slot_type == TFCC_ROCM_S32 || slot_type == TFCC_ROCM_S64, "cache_write: slot type %d", slot_type);
  if (tokens == 0) return TFCC_ROCM_OK;
  // memory that several rows share can be read, but not written
  TFCC_REQUIRE((cache->pages == 1 || cache->page_stride > 0) && (cache->heads == 1 || cache->head_stride > 0) && (cache->page_size == 1 || cache->row_stride > 0),
               "cache_write: a cache stride of 0");
  TFCC_REQUIRE(cache->type != TFCC_ROCM_S8 || ((cache->pages == 1 || cache->scale_page_stride > 0) && (cache->heads == 1 || cache->scale_head_stride > 0) &&
                                               (cache->page_size == 1 || cache->scale_row_stride > 0)),
               "cache_write: a cache scale stride of 0");
  // threads of a launch: whole workgroups
  const unsigned lanes = cache->size <= 64 ? 16 : cache->size <= 128 ? 32 : 64;
  TFCC_REQUIRE((uint64_t)tokens * cache->heads * lanes <= 0xffffffffu - (kCacheThreads - 1), "cache_write: %u tokens of %u heads", tokens, cache->heads);
  TFCC_REQUIRE(keys && values && slots, "cache_write: null argument");
  WriteArgs a{view_of(*cache), keys, values, key_token_stride, key_head_stride, value_token_stride, value_head_stride, slots,
              slot_type == TFCC_ROCM_S64, tokens, tokens * cache->heads, Divisor::of(cache->heads)};
  const hipStream_t s = as_stream(stream);
  const bool s8 = cache->type == TFCC_ROCM_S8;
  const auto start = [&](auto kernel) {
    const unsigned rows = kCacheThreads / lanes;
    hipLaunchKernelGGL(kernel, dim3((a.rows + rows - 1) / rows, 2), dim3(kCacheThreads), 0, s, a);
  };
  if (lanes == 16) start(s8 ? cache_write_kernel<true, 16> : cache_write_kernel<false, 16>);
  else if (lanes == 32) start(s8 ? cache_write_kernel<true, 32> : cache_write_kernel<false, 32>);
  else start(s8 ? cache_write_kernel<true, 64> : cache_write_kernel<false, 64>);
  return check_launch("cache_write");
}

int tfcc_rocm_cache_read(void* stream, const tfcc_rocm_paged_cache* cache, const int32_t* table, uint64_t table_stride,
                         unsigned table_width, unsigned batch, const int32_t* starts, unsigned tokens, float* keys,
                         float* values) {
  TFCC_REQUIRE(cache != nullptr, "cache_read: null cache");
  if (int e = check_cache(*cache, "cache_read")) return e;
  if (tokens == 0 || batch == 0) return TFCC_ROCM_OK;
  TFCC_REQUIRE((uint64_t)tokens * (kCacheThreads / kReadTokens) <= 0xffffffffu - (kCacheThreads - 1) && batch <= 0x7fffffffu,  // threads of a launch, as above
               "cache_read: %u tokens of %u sequences", tokens, batch);
  TFCC_REQUIRE(table && starts && keys && values, "cache_read: null argument");
  ReadArgs a{view_of(*cache), table, table_stride, table_width, batch, starts, tokens, keys, values};
  const hipStream_t s = as_stream(stream);
  const bool s8 = cache->type == TFCC_ROCM_S8;
  const auto start = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((tokens + kReadTokens - 1) / kReadTokens, 2), dim3(kCacheThreads), 0, s, a);
  };
  if (cache->size <= 64) start(s8 ? cache_read_kernel<true, 16> : cache_read_kernel<false, 16>);
  else if (cache->size <= 128) start(s8 ? cache_read_kernel<true, 32> : cache_read_kernel<false, 32>);
  else start(s8 ? cache_read_kernel<true, 64> : cache_read_kernel<false, 64>);
  return check_launch("cache_read");
}

}  // extern "C"
