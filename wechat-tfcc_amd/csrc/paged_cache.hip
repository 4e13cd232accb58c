// Keys and values into a paged cache, and sequences back out of it.  Bound: HBM (a few launches' latency for single tokens).
//
// Write: a row is one head of one token.  Its lanes hold four values each (a power of two of lanes, 16 to 64, several rows to a
// wavefront), so the row is read once: the largest absolute value is joined over its lanes, and
//   scale = amax * (1 / 127) (float32),  n = x / scale rounded to nearest, ties to even
// (1 / 7 for integers of 4 bits, which lie two to a byte).
// The quotient is not formed: n is taken from x * (1 / scale), which can miss only next to a border, and the remainder x - n * scale,
// which a fused multiply-add gives exactly there (|x| <= 127.5 scale, so it is a multiple of the smaller last place of x and scale
// and at most about scale / 2: 24 bits hold it), tells: below scale / 2 n is right, and where one of a lane's four is not, all are taken again and moved
// to the neighbour or, on a tie, to the even one.  So every integer is that of the true quotient, at four operations a value (with the
// moves formed for every value, the join of the largest through LDS and keys and values in workgroups of their own the kernel was bound by its operations).
// 16 x 2048 tokens of 8 x 128, 268 MB in: 67 us, 4.5 TB/s, for 4 bits, 69 us, 4.9 TB/s, for 8 (104 and 101 so), 80 us, 6.7 TB/s, as float32.
// What is read and written once, the rows on their way in and out, passes the caches by, so that the integers stay in the last level for
// those who read them next.
// The amax is formed on the bits of |x|, which order infinities and NaNs above all numbers: a row with one gets a scale that is not
// finite, integers 0, and reads back as NaN.
#include "paged_cache.hpp"

namespace tfcc_rocm {
namespace {

// What a cache holds of a value: the type's code.  Integers go from -kLargest to kLargest.
template <int TYPE>
constexpr int kLargest = TYPE == TFCC_ROCM_S8 ? 127 : 7;

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
constexpr float kAlign = 12582912.0f;  // 1.5 x 2^23: the last place of a sum with it is 1


// largest of the LANES lanes of a row, as bits
template <int LANES>
__device__ __forceinline__ unsigned row_max(unsigned u) {
  // sixteen lanes turn among themselves without LDS
  const auto turned = [&](auto by) {
    const unsigned o = (unsigned)__builtin_amdgcn_update_dpp(0, (int)u, 0x120 + decltype(by)::value, 0xf, 0xf, true);
    u = u > o ? u : o;
  };
  turned(std::integral_constant<int, 8>{});
  turned(std::integral_constant<int, 4>{});
  turned(std::integral_constant<int, 2>{});
  turned(std::integral_constant<int, 1>{});
#pragma unroll
  for (int m = LANES / 2; m > 8; m /= 2) {
    const unsigned o = (unsigned)__shfl_xor((int)u, m, 64);
    u = u > o ? u : o;
  }
  return u;
}

template <int LARGEST>
__device__ __forceinline__ int nearest(float x, float scale, float inverse) {
  float n = rintf(x * inverse);
  const float left = fmaf(-n, scale, x), half = 0.5f * scale;
  const bool odd = ((int)n & 1) != 0;
  if (left > half || (left == half && odd)) n += 1.0f;
  else if (left < -half || (left == -half && odd)) n -= 1.0f;
  return (int)fminf(fmaxf(n, -(float)LARGEST), (float)LARGEST);
}

template <int TYPE, int LANES>
__global__ __launch_bounds__(kCacheThreads) void cache_write_kernel(WriteArgs p) {
  const unsigned row = blockIdx.x * (kCacheThreads / LANES) + threadIdx.x / LANES, d = (threadIdx.x % LANES) * 4;
  if (row >= p.rows) return;
  const unsigned token = p.heads.quotient(row), head = row - token * p.heads.d;
  const bool mine = d < p.cache.size;
  f32x4 both[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  if (mine) {
    both[0] = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(p.keys + token * p.key_token + head * p.key_head + d));
    both[1] = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(p.values + token * p.value_token + head * p.value_head + d));
  }
  const long long slot = p.wide_slots ? static_cast<const long long*>(p.slots)[token] : static_cast<const int*>(p.slots)[token];
  if (slot < 0 || slot >= (long long)p.cache.pages * p.cache.page_size.d) return;
  // (a division of 64 bits takes its time)
  const unsigned long long page = slot < 0x80000000ll ? p.cache.page_size.quotient((unsigned)slot) : (unsigned long long)slot / p.cache.page_size.d;
  const unsigned inside = (unsigned)(slot - page * p.cache.page_size.d);
  const unsigned long long at = page * p.cache.page + head * p.cache.head + inside * p.cache.row;
#pragma unroll
  for (int value = 0; value < 2; ++value) {
    const f32x4 x = both[value];
    if constexpr (TYPE == TFCC_ROCM_F32) {
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
      const float scale = __uint_as_float(top) * (1.0f / kLargest<TYPE>);
      unsigned bits[4] = {0, 0, 0, 0};  // the integers, right in their lowest bits
      if (top < 0x7f800000u && scale > 0.0f) {
        // the sum leaves the integer in its low bits; v_rcp_f32 is off by a unit in the last place, which only the remainder's test has to know
        const float inverse = __builtin_amdgcn_rcpf(scale), half = 0.5f * scale;
        float over = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float sum = fmaf(x[i], inverse, kAlign);
          bits[i] = __float_as_uint(sum);
          over = fmaxf(over, fabsf(fmaf(kAlign - sum, scale, x[i])));
        }
        if (!(over < half) || scale < 1e-30f) {
          // a subnormal scale has no finite reciprocal: both are lifted by 2^64, which changes no quotient
          const float lift = scale < 1e-30f ? 18446744073709551616.0f : 1.0f, s = scale * lift, inverse = 1.0f / s;
#pragma unroll
          for (int i = 0; i < 4; ++i) bits[i] = (unsigned)nearest<kLargest<TYPE>>(x[i] * lift, s, inverse);
        }
      }
      int8_t* out = static_cast<int8_t*>(const_cast<void*>(value ? p.cache.values : p.cache.keys)) + at;
      if constexpr (TYPE == TFCC_ROCM_S8) {
        const unsigned low = __builtin_amdgcn_perm(bits[1], bits[0], 0x0c0c0400u), high = __builtin_amdgcn_perm(bits[3], bits[2], 0x04000c0cu);
        if (mine) *reinterpret_cast<unsigned*>(out + d) = low | high;
      } else {
        const unsigned pair = (bits[0] & 15u) | (bits[1] & 15u) << 4 | (bits[2] & 15u) << 8 | (bits[3] & 15u) << 12;
        if (mine) *reinterpret_cast<uint16_t*>(out + d / 2) = (uint16_t)pair;
      }
      if (d == 0)
        const_cast<float*>(value ? p.cache.value_scales : p.cache.key_scales)[page * p.cache.scale_page + head * p.cache.scale_head + inside * p.cache.scale_row] = scale;
    }
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

// LANES lanes of four values to a row, as above; a workgroup finds its tokens' slots once for all their heads (16 sequences of up to 2048 tokens of
// 8 x 128: from 4 bits 44 us, 5.9 TB/s, from 8 bits 49 us, 5.6 TB/s).
template <int TYPE, int LANES>
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
        const unsigned long long at = page * p.cache.page + head * p.cache.head + inside * p.cache.row;
        if constexpr (TYPE == TFCC_ROCM_F32) {
          x = *reinterpret_cast<const f32x4*>(static_cast<const float*>(held) + at + d);
        } else {
          const float scale = scales[page * p.cache.scale_page + head * p.cache.scale_head + inside * p.cache.scale_row];
          if constexpr (TYPE == TFCC_ROCM_S8) {
            const unsigned n = *reinterpret_cast<const unsigned*>(static_cast<const int8_t*>(held) + at + d);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(n >> (8 * i)) * scale;
          } else {
            const int n = *reinterpret_cast<const uint16_t*>(static_cast<const int8_t*>(held) + at + d / 2);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = (float)(n << (28 - 4 * i) >> 28) * scale;
          }
        }
      }
      __builtin_nontemporal_store(x, reinterpret_cast<f32x4_any*>(out + ((unsigned long long)(first + t) * p.cache.heads + head) * p.cache.size + d));
    }
  }
}

// Runs of rows to other places of the cache.  Bound: HBM, a launch for a few pages.  What a run moves of keys or values, [heads][rows][chunks] of
// UNIT bytes, is gone over as one range, cut into pieces for several workgroups: a thread has all its loads under way before it stores the first.  Pieces
// behind those move the scales, 4 bytes to a unit.  (1500 whole pages of 64 rows of 8 x 128 in 4 bits, 209 MB moved: 45 us, 4.6 TB/s, and 34 where the last-level
// cache holds them; 500 of 32 rows in float32, 262 MB: 41 us, 6.4 TB/s; four half pages 3.8 us.)
// From so many runs on a page whose rows are one piece has its scales moved by the same workgroup: fewer of them outweigh that the scales wait for the rows (pages of 16 rows of
// 8 x 128 in 4 bits, 3000 runs: 19.9 us, apart 24.9; 300: 4.5 and 4.6; 100: 3.7 and 3.3).
constexpr unsigned kManyRuns = 256;
constexpr unsigned kCopyEach = 4, kCopyUnits = kCacheThreads * kCopyEach;
struct CopyArgs {
  void* rows_of[2];
  float* scales_of[2];
  unsigned long long page, head, row, scale_page, scale_head, scale_row;  // in bytes
  const void *sources, *destinations;
  const int* rows;
  int wide_slots;
  unsigned pages, units, scale_units, row_pieces;
  int together;  // a run's one piece of rows moves its scales as well
  Divisor page_size, chunks, pieces;
};

template <class Unit>
__device__ __forceinline__ void copy_piece(unsigned piece, unsigned units, const Divisor& chunks, const Divisor& page_size, unsigned rows, char* memory,
                                           unsigned long long from, unsigned long long to, unsigned long long head_stride, unsigned long long row_stride) {
  Unit held[kCopyEach];
  unsigned long long at[kCopyEach];
  bool mine[kCopyEach];
#pragma unroll
  for (unsigned i = 0; i < kCopyEach; ++i) {
    const unsigned unit = piece * kCopyUnits + i * kCacheThreads + threadIdx.x;
    const unsigned line = chunks.quotient(unit), chunk = unit - line * chunks.d, head = page_size.quotient(line), row = line - head * page_size.d;
    mine[i] = unit < units && row < rows;
    at[i] = head * head_stride + row * row_stride + chunk * (unsigned long long)sizeof(Unit);
    if (mine[i]) held[i] = *reinterpret_cast<const Unit*>(memory + from + at[i]);
  }
#pragma unroll
  for (unsigned i = 0; i < kCopyEach; ++i)
    if (mine[i]) *reinterpret_cast<Unit*>(memory + to + at[i]) = held[i];
}

template <unsigned UNIT>
__global__ __launch_bounds__(kCacheThreads) void cache_copy_kernel(CopyArgs p) {
  const unsigned run = p.pieces.quotient(blockIdx.x), piece = blockIdx.x - run * p.pieces.d;
  const auto slot_of = [&](const void* slots) { return p.wide_slots ? static_cast<const long long*>(slots)[run] : static_cast<const int*>(slots)[run]; };
  const long long source = slot_of(p.sources), destination = slot_of(p.destinations), slots = (long long)p.pages * p.page_size.d;
  if (source < 0 || source >= slots || destination < 0 || destination >= slots) return;
  const auto page_of = [&](long long slot) {
    return slot < 0x80000000ll ? p.page_size.quotient((unsigned)slot) : (unsigned long long)slot / p.page_size.d;
  };
  const unsigned long long from_page = page_of(source), to_page = page_of(destination);
  const unsigned from_row = (unsigned)(source - from_page * p.page_size.d), to_row = (unsigned)(destination - to_page * p.page_size.d);
  unsigned rows = p.page_size.d - (from_row > to_row ? from_row : to_row);
  if (p.rows != nullptr) {
    const int wanted = p.rows[run];
    if (wanted <= 0) return;
    rows = (unsigned)wanted < rows ? (unsigned)wanted : rows;
  }
  if (piece < p.row_pieces) {
    typedef unsigned unit __attribute__((ext_vector_type(UNIT / 4)));
    copy_piece<unit>(piece, p.units, p.chunks, p.page_size, rows, static_cast<char*>(p.rows_of[blockIdx.y]), from_page * p.page + from_row * p.row,
                     to_page * p.page + to_row * p.row, p.head, p.row);
  }
  if (piece >= p.row_pieces || p.together) {
    const Divisor one = {1, 1u << 31, 31};
    copy_piece<unsigned>(p.together ? 0 : piece - p.row_pieces, p.scale_units, one, p.page_size, rows, reinterpret_cast<char*>(p.scales_of[blockIdx.y]),
                         from_page * p.scale_page + from_row * p.scale_row, to_page * p.scale_page + to_row * p.scale_row, p.scale_head, p.scale_row);
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
  if (int e = check_written(*cache, "cache_write")) return e;
  // threads of a launch: whole workgroups
  const unsigned lanes = cache->size <= 64 ? 16 : cache->size <= 128 ? 32 : 64;
  TFCC_REQUIRE((uint64_t)tokens * cache->heads * lanes <= 0xffffffffu - (kCacheThreads - 1), "cache_write: %u tokens of %u heads", tokens, cache->heads);
  TFCC_REQUIRE(keys && values && slots, "cache_write: null argument");
  WriteArgs a{view_of(*cache), keys, values, key_token_stride, key_head_stride, value_token_stride, value_head_stride, slots,
              slot_type == TFCC_ROCM_S64, tokens, tokens * cache->heads, Divisor::of(cache->heads)};
  const hipStream_t s = as_stream(stream);
  const auto start = [&](auto s4, auto s8, auto f32) {
    const unsigned rows = kCacheThreads / lanes;
    hipLaunchKernelGGL((cache->type == TFCC_ROCM_S4 ? s4 : cache->type == TFCC_ROCM_S8 ? s8 : f32), dim3((a.rows + rows - 1) / rows), dim3(kCacheThreads), 0, s, a);
  };
  if (lanes == 16) start(cache_write_kernel<TFCC_ROCM_S4, 16>, cache_write_kernel<TFCC_ROCM_S8, 16>, cache_write_kernel<TFCC_ROCM_F32, 16>);
  else if (lanes == 32) start(cache_write_kernel<TFCC_ROCM_S4, 32>, cache_write_kernel<TFCC_ROCM_S8, 32>, cache_write_kernel<TFCC_ROCM_F32, 32>);
  else start(cache_write_kernel<TFCC_ROCM_S4, 64>, cache_write_kernel<TFCC_ROCM_S8, 64>, cache_write_kernel<TFCC_ROCM_F32, 64>);
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
  const auto start = [&](auto s4, auto s8, auto f32) {
    hipLaunchKernelGGL((cache->type == TFCC_ROCM_S4 ? s4 : cache->type == TFCC_ROCM_S8 ? s8 : f32), dim3((tokens + kReadTokens - 1) / kReadTokens, 2), dim3(kCacheThreads), 0, s, a);
  };
  if (cache->size <= 64) start(cache_read_kernel<TFCC_ROCM_S4, 16>, cache_read_kernel<TFCC_ROCM_S8, 16>, cache_read_kernel<TFCC_ROCM_F32, 16>);
  else if (cache->size <= 128) start(cache_read_kernel<TFCC_ROCM_S4, 32>, cache_read_kernel<TFCC_ROCM_S8, 32>, cache_read_kernel<TFCC_ROCM_F32, 32>);
  else start(cache_read_kernel<TFCC_ROCM_S4, 64>, cache_read_kernel<TFCC_ROCM_S8, 64>, cache_read_kernel<TFCC_ROCM_F32, 64>);
  return check_launch("cache_read");
}

int tfcc_rocm_cache_copy(void* stream, const tfcc_rocm_paged_cache* cache, const void* sources, const void* destinations, int slot_type,
                         const int32_t* rows, unsigned runs) {
  TFCC_REQUIRE(cache != nullptr, "cache_copy: null cache");
  const tfcc_rocm_paged_cache& c = *cache;
  if (int e = check_cache(c, "cache_copy")) return e;
  TFCC_REQUIRE(slot_type == TFCC_ROCM_S32 || slot_type == TFCC_ROCM_S64, "cache_copy: slot type %d", slot_type);
  if (runs == 0) return TFCC_ROCM_OK;
  if (int e = check_written(c, "cache_copy")) return e;
  CopyArgs a{};
  const unsigned element = element_bytes(c), bytes = row_bytes(c);
  const bool wide = (bytes | c.page_stride * element | c.head_stride * element | c.row_stride * element | reinterpret_cast<uintptr_t>(c.keys) |
                     reinterpret_cast<uintptr_t>(c.values)) % 16 == 0;
  const unsigned unit = wide ? 16 : 8;
  a.rows_of[0] = c.keys;
  a.rows_of[1] = c.values;
  a.scales_of[0] = c.key_scales;
  a.scales_of[1] = c.value_scales;
  a.page = c.page_stride * element;
  a.head = c.head_stride * element;
  a.row = c.row_stride * element;
  a.scale_page = c.scale_page_stride * 4;
  a.scale_head = c.scale_head_stride * 4;
  a.scale_row = c.scale_row_stride * 4;
  a.sources = sources;
  a.destinations = destinations;
  a.rows = rows;
  a.wide_slots = slot_type == TFCC_ROCM_S64;
  a.pages = c.pages;
  a.page_size = Divisor::of(c.page_size);
  a.chunks = Divisor::of(bytes / unit);
  const uint64_t units = (uint64_t)c.heads * c.page_size * (bytes / unit), scales = has_scales(c) ? (uint64_t)c.heads * c.page_size : 0;
  const uint64_t row_pieces = (units + kCopyUnits - 1) / kCopyUnits, scale_pieces = (scales + kCopyUnits - 1) / kCopyUnits;
  a.together = runs >= kManyRuns && row_pieces == 1 && scale_pieces == 1;
  const uint64_t pieces = row_pieces + (a.together ? 0 : scale_pieces);
  TFCC_REQUIRE(units <= 0x7fffffffu - kCopyUnits && (row_pieces + scale_pieces) * runs <= 0x7fffffffu / kCacheThreads, "cache_copy: %u runs of up to %llu bytes", runs,
               (unsigned long long)units * unit);
  TFCC_REQUIRE(sources && destinations, "cache_copy: null argument");
  a.units = (unsigned)units;
  a.scale_units = (unsigned)scales;
  a.row_pieces = (unsigned)row_pieces;
  a.pieces = Divisor::of((unsigned)pieces);
  hipLaunchKernelGGL((wide ? cache_copy_kernel<16> : cache_copy_kernel<8>), dim3((unsigned)pieces * runs, 2), dim3(kCacheThreads), 0, as_stream(stream), a);
  return check_launch("cache_copy");
}

}  // extern "C"
