// One token for each row of logits: temperature, top-k, top-p, min-p and a given random number.
//
// Weights exp((x - max) / temperature) are formed in 64 bits and summed as integers of 2^-shift of the largest one.  Sums of integers
// do not depend on their order, so a row's token does not either, however the row is shared out; and a token is decided at borders
// between sums of up to a million weights, where float32 sums would choose a neighbour now and then.
// The kept tokens are the first of the order of falling logits, so each filter is a border in that order: a key (the logit's bits,
// ordered) and how many of the tokens with just that key, by position.  Borders are found eight bits of the key at a time, from
// the highest: 256 counts and sums of weights, then on in the one that holds the border.
#include "common.hpp"

namespace tfcc_rocm {
namespace {

typedef unsigned long long u64;

struct SampleArgs {
  const float* logits;
  u64 row_stride;
  unsigned rows, length;
  int shift;
  const float* random;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  long long* tokens;
  float* probabilities;
};

constexpr unsigned kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr unsigned kNoToken = 0x007fffffu;  // the key of -infinity; that of a NaN is below

// Order of logits as unsigned integers; both zeros are one.
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);
  return x != x ? 0u : (u & 0x80000000u ? ~u : u | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// exp(x) * 2^shift for x <= 0: 2^n 2^f with |f| <= 1/2 and the Taylor polynomial of e^(f ln 2) to the 11th power, whose rest is below
// 6e-15 of it.  Where x is a NaN - infinity less infinity - it is the largest weight.
__device__ __forceinline__ double weight_of(double x, int shift) {
  double t = x * 1.4426950408889634074;
  t = t > -1000.0 ? t : (t <= -1000.0 ? -1000.0 : 0.0);
  const double n = rint(t), f = (t - n) * 0.69314718055994530942;
  double e = 2.50521083854417188e-8;
  e = fma(e, f, 2.75573192239858907e-7);
  e = fma(e, f, 2.75573192239858907e-6);
  e = fma(e, f, 2.48015873015873016e-5);
  e = fma(e, f, 1.98412698412698413e-4);
  e = fma(e, f, 1.38888888888888889e-3);
  e = fma(e, f, 8.33333333333333333e-3);
  e = fma(e, f, 4.16666666666666667e-2);
  e = fma(e, f, 1.66666666666666667e-1);
  e = fma(e, f, 0.5);
  e = fma(e, f, 1.0);
  e = fma(e, f, 1.0);
  return ldexp(e, (int)n + shift);
}
// to the nearest integer, below 2^52
__device__ __forceinline__ u64 integer_of(double w) { return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull; }

struct Row {
  float top;
  double slope;  // 1 / temperature
  int shift;
  __device__ double weight(float x) const { return weight_of(((double)x - (double)top) * slope, shift); }
};

__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
  for (int m = 32; m > 0; m /= 2) v += (u64)__shfl_xor((long long)v, m, 64);
  return v;
}

struct Shared {
  unsigned counts[256];
  u64 weights[256];
  u64 totals[kSampleWaves];
  unsigned tops[kSampleWaves];
  unsigned digit, key, position;
  unsigned found;
  u64 above, ties, sum;
};

// Which of 256 bins, from the highest, holds the border: the first at which the running sum of counts (or weights) from `start` on
// reaches `target`.  `above`: what the bins before it hold.  One wavefront.
template <class T>
__device__ void find_bin(const T* bins, u64 start, u64 target, unsigned* bin, u64* above) {
  const unsigned lane = threadIdx.x & 63;
  u64 v[4], mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = bins[255 - (4 * lane + i)];
    mine += v[i];
  }
  u64 upto = mine;
#pragma unroll
  for (int m = 1; m < 64; m *= 2) {
    const u64 o = (u64)__shfl_up((long long)upto, m, 64);
    if (lane >= (unsigned)m) upto += o;
  }
  upto += start;
  const u64 reached = __ballot(upto >= target);
  const unsigned at = reached == 0 ? 63u : (unsigned)__builtin_ctzll(reached);
  if (lane == at) {
    u64 before = upto - mine;
    unsigned b = 4 * lane;
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (before + v[i] < target && b == 4 * lane + i) {
        before += v[i];
        ++b;
      }
    *bin = 255 - b;
    *above = before;
  }
}

// A border of one row: tokens with a larger key, and `ties` of those with this one, are kept.
struct Border {
  unsigned key;
  u64 ties;
};

template <bool WEIGHTS>
__device__ Border find_border(const float* x, unsigned length, const Row& row, u64 target, Shared& s, u64& kept_weight) {
  unsigned prefix = 0, mask = 0;
  u64 count_above = 0, weight_above = 0;
  for (int bits = 24; bits >= 0; bits -= 8) {
    for (unsigned i = threadIdx.x; i < 256; i += kSampleThreads) {
      s.counts[i] = 0;
      s.weights[i] = 0;
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < length; i += kSampleThreads) {
      const float v = x[i];
      const unsigned key = key_of(v);
      if ((key & mask) == prefix) {
        const unsigned b = (key >> bits) & 255;
        atomicAdd(&s.counts[b], 1u);
        if (key > kNoToken) atomicAdd(&s.weights[b], integer_of(row.weight(v)));
      }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
      if (WEIGHTS) find_bin(s.weights, weight_above, target, &s.digit, &s.above);
      else find_bin(s.counts, count_above, target, &s.digit, &s.above);
    }
    __syncthreads();
    const unsigned digit = s.digit;
    u64 counts = 0, weights = 0;
    for (unsigned i = digit + 1 + (threadIdx.x & 63); i < 256; i += 64) {
      counts += s.counts[i];
      weights += s.weights[i];
    }
    count_above += wave_sum64(counts);
    weight_above += wave_sum64(weights);
    prefix |= digit << bits;
    mask |= 255u << bits;
    if (bits == 0) {
      const u64 there = s.counts[digit], weight = there == 0 ? 0 : s.weights[digit] / there;
      u64 ties = there;
      if (!WEIGHTS) ties = target - count_above < there ? target - count_above : there;
      else if (weight > 0 && target > weight_above) {
        const u64 needs = (target - weight_above + weight - 1) / weight;
        ties = needs < there ? needs : there;
      }
      if (ties == 0) ties = 1;
      kept_weight = weight_above + ties * weight;
      __syncthreads();
      return {prefix, ties};
    }
    __syncthreads();
  }
  return {0, 0};
}

// One workgroup to a row.
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(SampleArgs p) {
  __shared__ Shared s;
  const unsigned r = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  const float* x = p.logits + r * p.row_stride;
  unsigned top = 0;
  for (unsigned i = threadIdx.x; i < p.length; i += kSampleThreads) {
    const unsigned k = key_of(x[i]);
    top = top > k ? top : k;
  }
#pragma unroll
  for (int m = 32; m > 0; m /= 2) {
    const unsigned o = (unsigned)__shfl_xor((int)top, m, 64);
    top = top > o ? top : o;
  }
  if (lane == 0) s.tops[wave] = top;
  if (threadIdx.x == 0) s.position = 0xffffffffu;
  __syncthreads();
  for (unsigned w = 0; w < kSampleWaves; ++w) top = top > s.tops[w] ? top : s.tops[w];
  if (top <= kNoToken) {
    if (threadIdx.x == 0) {
      p.tokens[r] = -1;
      if (p.probabilities) p.probabilities[r] = 0.0f;
    }
    return;
  }
  const float temperature = p.temperature ? p.temperature[r] : 1.0f;
  if (!(temperature > 0.0f)) {
    for (unsigned i = threadIdx.x; i < p.length; i += kSampleThreads)
      if (key_of(x[i]) == top) {
        atomicMin(&s.position, i);
        break;
      }
    __syncthreads();
    if (threadIdx.x == 0) {
      p.tokens[r] = s.position;
      if (p.probabilities) p.probabilities[r] = 1.0f;
    }
    return;
  }
  const Row row{value_of(top), 1.0 / (double)temperature, p.shift};
  Border border{kNoToken + 1, ~0ull};
  u64 total = 0;
  const int k = p.top_k ? p.top_k[r] : 0;
  if (k > 0 && (unsigned)k < p.length) {
    border = find_border<false>(x, p.length, row, (u64)k, s, total);
  } else {
    u64 mine = 0;
    for (unsigned i = threadIdx.x; i < p.length; i += kSampleThreads)
      if (key_of(x[i]) > kNoToken) mine += integer_of(row.weight(x[i]));
    mine = wave_sum64(mine);
    if (lane == 0) s.totals[wave] = mine;
    __syncthreads();
    for (unsigned w = 0; w < kSampleWaves; ++w) total += s.totals[w];
    __syncthreads();
  }
  const float top_p = p.top_p ? p.top_p[r] : 1.0f;
  if (top_p < 1.0f) {
    u64 target = top_p > 0.0f ? (u64)ceil((double)top_p * (double)total) : 0;
    if (target < 1) target = 1;
    border = find_border<true>(x, p.length, row, target, s, total);
  }
  if (border.key <= kNoToken) border = {kNoToken + 1, ~0ull};
  const float min_p = p.min_p ? p.min_p[r] : 0.0f;
  const double least = ldexp(fmin((double)min_p, 1.0), p.shift);  // of a kept weight
  // Each wavefront takes a run of positions.  Of the tokens with the border's key, the first `ties` count.
  const unsigned run = (p.length + kSampleThreads - 1) / kSampleThreads * 64, first = wave * run;
  const unsigned behind = first + run < p.length ? first + run : p.length;
  u64 ties = 0;
  for (unsigned i = first + lane; i < behind; i += 64) ties += key_of(x[i]) == border.key ? 1 : 0;
  ties = wave_sum64(ties);
  if (lane == 0) s.totals[wave] = ties;
  __syncthreads();
  u64 seen = 0;
  for (unsigned w = 0; w < wave; ++w) seen += s.totals[w];
  __syncthreads();
  const u64 seen0 = seen;
  const auto kept = [&](unsigned i, u64& seen) -> u64 {  // a token's weight, 0 if it is not kept; all lanes of a wavefront together
    const float v = i < behind ? x[i] : NAN;
    const unsigned key = key_of(v);
    const u64 same = __ballot(key == border.key);
    const u64 before = seen + __popcll(same & ((1ull << lane) - 1));
    seen += __popcll(same);
    if (key < border.key || (key == border.key && before >= border.ties)) return 0;
    const double w = row.weight(v);
    return w >= least ? integer_of(w) : 0;
  };
  u64 mine = 0;
  for (unsigned base = first; base < first + run; base += 64) mine += kept(base + lane, seen);
  mine = wave_sum64(mine);
  if (lane == 0) s.totals[wave] = mine;
  __syncthreads();
  u64 before = 0, sum = 0;
  for (unsigned w = 0; w < kSampleWaves; ++w) {
    if (w < wave) before += s.totals[w];
    sum += s.totals[w];
  }
  const float random = p.random[r];
  u64 target = random > 0.0f ? (u64)((double)random * (double)sum) : 0;
  if (target >= sum) target = sum - 1;
  if (target < before || target >= before + mine) return;  // the token is another wavefront's
  seen = seen0;
  for (unsigned base = first; base < first + run; base += 64) {
    const u64 w = kept(base + lane, seen);
    u64 upto = w;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const u64 o = (u64)__shfl_up((long long)upto, m, 64);
      if (lane >= (unsigned)m) upto += o;
    }
    upto += before;
    const u64 past = __ballot(upto > target);
    if (past != 0) {
      if (lane == (unsigned)__builtin_ctzll(past)) {
        p.tokens[r] = base + lane;
        if (p.probabilities) p.probabilities[r] = (float)(row.weight(x[base + lane]) / (double)sum);
      }
      return;
    }
    before = (u64)__shfl((long long)upto, 63, 64);
  }
}

int shift_for(unsigned length) {
  int log = 0;
  while ((1ull << log) < length) ++log;
  return 63 - log < 51 ? 63 - log : 51;
}

}  // namespace
}  // namespace tfcc_rocm

using namespace tfcc_rocm;

extern "C" {

size_t tfcc_rocm_sample_workspace(unsigned rows, unsigned length) { return 0; }

int tfcc_rocm_sample_f32(void* stream, const tfcc_rocm_sample_desc* desc) {
  TFCC_REQUIRE(desc != nullptr, "sample: null descriptor");
  const tfcc_rocm_sample_desc& d = *desc;
  TFCC_REQUIRE(d.length > 0 && d.length <= (1u << 20), "sample: rows of %u logits (1 to 2^20)", d.length);
  TFCC_REQUIRE(d.rows <= 0x7fffffffu, "sample: %u rows", d.rows);
  if (d.rows == 0) return TFCC_ROCM_OK;
  TFCC_REQUIRE(d.logits && d.random && d.tokens, "sample: null argument");
  SampleArgs a{d.logits, d.row_stride, d.rows, d.length, shift_for(d.length), d.random, d.temperature, d.top_k, d.top_p, d.min_p,
               reinterpret_cast<long long*>(d.tokens), d.probabilities};
  hipLaunchKernelGGL(sample_kernel, dim3(d.rows), dim3(kSampleThreads), 0, as_stream(stream), a);
  return check_launch("sample");
}

}  // extern "C"
