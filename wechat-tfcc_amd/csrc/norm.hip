// Root-mean-square norm with the residual's addition, as float32 or as 8-bit integers with a scale for each row, and rows of integers
// back to float32.  Bound: HBM; for few rows the latency of a launch.  8192 rows of 4096 with a residual: as float32 100 us, 5.4 TB/s, as integers 84 us,
// 5.2 TB/s, and back to float32 28 us, 5.9 TB/s; one row 3.9, 5.5 and 4.1 us.
//
// One pass: a row's threads keep h and the weights in registers while the sum of squares (and the largest |t|, t = h * weight) is joined, then round their
// products.  The integers of a row do not depend on its root: n = 127 t / max |t|.  A product of two float32 is exact in 64 bits, so t and the largest are,
// and n is that of the true quotient: t * (127 / max) is off by 2^-51 of itself, and where that may matter, next to a border, 127 t is compared with
// (n +- 1/2) max in exact sums of two doubles.  64-bit operations run at the rate of 32-bit ones here, and a value takes a dozen of them: the norm stays
// bound by HBM.
#include "common.hpp"
#include "paged_cache.hpp"

namespace tfcc_rocm {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));  // needs no more than a float's alignment
typedef unsigned u32_any __attribute__((aligned(1)));

constexpr unsigned kNormMost = 16384;  // values of a row that registers hold
// Up to so many rows a thread takes four values: with a workgroup for each CU or less a row's own time counts (float32, 4096 wide: 16 rows 4.0 us,
// with sixteen values to a thread 4.5; 256 rows 5.1 and 5.6).  More rows fill the CUs either way, and fewer wavefronts join faster.
// The integers of a row of 4096 are not faster so (16 rows: 5.9 us, with sixteen values to a thread 5.5).
constexpr unsigned kFewRows = 256;

struct NormArgs {
  const float *x, *residual, *weight;
  float *sum, *out;
  uint8_t* steps;
  float* scales;
  int32_t* sums;
  unsigned long long x_row, residual_row, sum_row, out_row, steps_row;
  unsigned rows, width;
  double eps;
};

// The value of lane i ^ MASK of a double, as butterfly_pair does it for a float.
template <int MASK>
__device__ __forceinline__ void butterfly_pair64(double v, double& a, double& b) {
  float lo_a, lo_b, hi_a, hi_b;
  butterfly_pair<MASK>(__int_as_float(__double2loint(v)), lo_a, lo_b);
  butterfly_pair<MASK>(__int_as_float(__double2hiint(v)), hi_a, hi_b);
  a = __hiloint2double(__float_as_int(hi_a), __float_as_int(lo_a));
  b = __hiloint2double(__float_as_int(hi_b), __float_as_int(lo_b));
}
// Of LANES neighbours, 16 or more.
template <unsigned LANES, class Join>
__device__ __forceinline__ double wave_join64(double v, Join join) {
  double a, b;
  if constexpr (LANES > 32) { butterfly_pair64<32>(v, a, b); v = join(a, b); }
  if constexpr (LANES > 16) { butterfly_pair64<16>(v, a, b); v = join(a, b); }
  butterfly_pair64<8>(v, a, b); v = join(a, b);
  butterfly_pair64<4>(v, a, b); v = join(a, b);
  butterfly_pair64<2>(v, a, b); v = join(a, b);
  butterfly_pair64<1>(v, a, b); v = join(a, b);
  return v;
}

constexpr double kInfinity = __builtin_inf();
struct RowTotals {
  double squares;
  double top;  // the largest |t|; infinity where one is not finite.  (The squares say nothing of it: the root is the same whether integers are asked for or not.)
};
__device__ __forceinline__ double add64(double a, double b) { return a + b; }
__device__ __forceinline__ double max64(double a, double b) { return fmax(a, b); }

// Sum and maximum over the threads of a row, THREADS of them (16, 32 or a multiple of 64); shared: two rows of THREADS / 64.
template <unsigned THREADS, bool STEPS>
__device__ __forceinline__ RowTotals row_totals(double squares, double top, double (*shared)[16]) {
  constexpr unsigned lanes = THREADS < 64 ? THREADS : 64;
  squares = wave_join64<lanes>(squares, add64);
  if constexpr (STEPS) top = wave_join64<lanes>(top, max64);
  if constexpr (THREADS > 64) {
    constexpr unsigned waves = THREADS / 64;
    const unsigned wave = threadIdx.x / 64;
    if (threadIdx.x % 64 == 0) {
      shared[0][wave] = squares;
      if constexpr (STEPS) shared[1][wave] = top;
    }
    __syncthreads();
    squares = shared[0][0];
    if constexpr (STEPS) top = shared[1][0];
#pragma unroll
    for (unsigned w = 1; w < waves; ++w) {
      squares += shared[0][w];
      if constexpr (STEPS) top = max64(top, shared[1][w]);
    }
  }
  return {squares, top};
}
template <unsigned THREADS>
__device__ __forceinline__ int row_count(int count, int* shared) {
#pragma unroll
  for (int m = THREADS < 64 ? THREADS / 2 : 32; m > 0; m /= 2) count += __shfl_xor(count, m, 64);
  if constexpr (THREADS > 64) {
    if (threadIdx.x % 64 == 0) shared[threadIdx.x / 64] = count;
    __syncthreads();
    count = 0;
#pragma unroll
    for (unsigned w = 0; w < THREADS / 64; ++w) count += shared[w];
  }
  return count;
}

// 127 t / top to the nearest, ties to even; factor = 127 / top.
__device__ __forceinline__ int step_of(double t, double top, double factor) {
  const double u = t * factor;
  double n = rint(u);
  const double off = u - n;
  if (fabs(off) > 0.499999999) {  // a border: u is off by 2^-44 at most
    const double other = off > 0.0 ? n + 1.0 : n - 1.0, border = 0.5 * (n + other);
    // 127 t - border top, exactly but for the last sum, whose sign is right
    const double p = 127.0 * t, p_rest = fma(127.0, t, -p), s = border * top, s_rest = fma(border, top, -s);
    const double left = (p - s) + (p_rest - s_rest);
    const bool odd = ((int)n & 1) != 0;
    if (left == 0.0 ? odd : (left > 0.0) == (off > 0.0)) n = other;
  }
  return (int)n;
}

struct RowFactors {
  double root;    // 1 / sqrt(mean + eps)
  double factor;  // 127 / largest |t|; 0: all steps are 128
  float scale;
};
__device__ __forceinline__ RowFactors factors_of(const NormArgs& p, const RowTotals& totals) {
  RowFactors f;
  const bool odd = totals.top == kInfinity;
  f.root = 1.0 / sqrt(totals.squares / p.width + p.eps);
  f.factor = totals.top > 0.0 && !odd ? 127.0 / totals.top : 0.0;
  f.scale = odd ? __uint_as_float(0x7fc00000u) : (totals.top > 0.0 ? (float)(totals.top * f.root / 127.0) : 0.0f);
  return f;
}

// A row to THREADS threads, HELD times four values of it to a thread: 4 HELD THREADS values at most, and the fewest that hold a row: short ones share a
// wavefront (60000 rows of 64: float32 11.9 us, 5.2 TB/s, 8 bits 13.4; with a wavefront to a row and sixteen values to a thread 29.5 and 47.6), and a value that is not there
// costs as much as one that is (16384 of 256: 12.7 and 15.3 us, with places for 1024 13.9 and 19.3).  The form with integers is held to the registers
// of 8 wavefronts to a SIMD (3000 rows of 9537: 85 us, without 108); the plain one would spill there (110 us, without 95).
template <unsigned THREADS, unsigned HELD, bool STEPS>
__global__ __launch_bounds__(THREADS < 256 ? 256 : THREADS, STEPS && HELD > 1 ? 8 : 4) void rms_norm_kernel(NormArgs p) {
  constexpr unsigned ROWS = THREADS < 256 ? 256 / THREADS : 1;
  static_assert(THREADS <= 64 || ROWS == 1);
  __shared__ double shared[2][16];
  __shared__ int shared_count[16];
  const unsigned long long row = (unsigned long long)blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x / THREADS : 0);
  if (row >= p.rows) return;  // whole wavefronts, or their halves and quarters that rows have
  const unsigned me = threadIdx.x % THREADS;
  const float* const x = p.x + row * p.x_row;
  const float* const residual = p.residual != nullptr ? p.residual + row * p.residual_row : nullptr;
  f32x4 h[HELD], w[HELD];
#pragma unroll
  for (unsigned i = 0; i < HELD; ++i) {
    const unsigned at = 4 * (me + THREADS * i);
    h[i] = w[i] = f32x4{0, 0, 0, 0};
    if (at + 4 <= p.width) {
      h[i] = *reinterpret_cast<const f32x4_any*>(x + at);
      w[i] = *reinterpret_cast<const f32x4_any*>(p.weight + at);
      if (residual != nullptr) h[i] += *reinterpret_cast<const f32x4_any*>(residual + at);
    } else {
#pragma unroll
      for (unsigned j = 0; j < 3; ++j)
        if (at + j < p.width) {
          h[i][j] = x[at + j];
          w[i][j] = p.weight[at + j];
          if (residual != nullptr) h[i][j] += residual[at + j];
        }
    }
  }
  const auto product = [&](unsigned i, unsigned j) { return (double)h[i][j] * (double)w[i][j]; };
  double squares = 0.0, top = 0.0, rest = 0.0;
#pragma unroll
  for (unsigned i = 0; i < HELD; ++i) {
    const unsigned at = 4 * (me + THREADS * i);
    if (p.sum != nullptr) {
      float* const sum = p.sum + row * p.sum_row;
      if (at + 4 <= p.width) {
        *reinterpret_cast<f32x4_any*>(sum + at) = h[i];
      } else {
#pragma unroll
        for (unsigned j = 0; j < 3; ++j)
          if (at + j < p.width) sum[at + j] = h[i][j];
      }
    }
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) {
      const double v = h[i][j];
      squares = fma(v, v, squares);
      if constexpr (STEPS) {
        const double t = product(i, j);
        top = max64(top, fabs(t));
        rest = fma(t, 0.0, rest);  // 0, or NaN where t is not finite
      }
    }
  }
  if constexpr (STEPS) top = rest == 0.0 ? top : kInfinity;
  const RowTotals totals = row_totals<THREADS, STEPS>(squares, top, shared);
  const RowFactors f = factors_of(p, totals);
  int count = 0;
#pragma unroll
  for (unsigned i = 0; i < HELD; ++i) {
    const unsigned at = 4 * (me + THREADS * i);
    if (at >= p.width) break;
    const unsigned some = p.width - at < 4 ? p.width - at : 4;
    if (p.out != nullptr) {
      f32x4 y;
#pragma unroll
      for (unsigned j = 0; j < 4; ++j) y[j] = (float)(product(i, j) * f.root);
      float* const out = p.out + row * p.out_row + at;
      if (some == 4) {
        *reinterpret_cast<f32x4_any*>(out) = y;
      } else {
#pragma unroll
        for (unsigned j = 0; j < 3; ++j)
          if (j < some) out[j] = y[j];
      }
    }
    if constexpr (STEPS) {
      unsigned word = 0;
#pragma unroll
      for (unsigned j = 0; j < 4; ++j) {
        const int q = 128 + (f.factor > 0.0 ? step_of(product(i, j), totals.top, f.factor) : 0);
        count += j < some ? q : 0;
        word |= (unsigned)q << (8 * j);
      }
      uint8_t* const steps = p.steps + row * p.steps_row + at;
      if (some == 4) {
        *reinterpret_cast<u32_any*>(steps) = word;
      } else {
#pragma unroll
        for (unsigned j = 0; j < 3; ++j)
          if (j < some) steps[j] = (uint8_t)(word >> (8 * j));
      }
    }
  }
  if constexpr (STEPS) {
    if (p.sums != nullptr) count = row_count<THREADS>(count, shared_count);
    if (me == 0) {
      p.scales[row] = f.scale;
      if (p.sums != nullptr) p.sums[row] = count;
    }
  }
}

// Rows of more values than registers hold: read twice, the second time from the caches.  A thread goes over the same values both times.
template <bool STEPS>
__global__ __launch_bounds__(1024) void rms_norm_wide_kernel(NormArgs p) {
  __shared__ double shared[2][16];
  __shared__ int shared_count[16];
  const unsigned long long row = blockIdx.x;
  const float* const x = p.x + row * p.x_row;
  const float* const residual = p.residual != nullptr ? p.residual + row * p.residual_row : nullptr;
  float* const sum = p.sum != nullptr ? p.sum + row * p.sum_row : nullptr;
  double squares = 0.0, top = 0.0, rest = 0.0;
  for (unsigned at = threadIdx.x; at < p.width; at += 1024) {
    float h = x[at];
    if (residual != nullptr) h += residual[at];
    const double t = (double)h * (double)p.weight[at];
    squares = fma((double)h, (double)h, squares);
    if constexpr (STEPS) {
      top = max64(top, fabs(t));
      rest = fma(t, 0.0, rest);
    }
  }
  if constexpr (STEPS) top = rest == 0.0 ? top : kInfinity;
  const RowTotals totals = row_totals<1024, STEPS>(squares, top, shared);
  const RowFactors f = factors_of(p, totals);
  int count = 0;
  for (unsigned at = threadIdx.x; at < p.width; at += 1024) {
    float h = x[at];
    if (residual != nullptr) h += residual[at];
    if (sum != nullptr) sum[at] = h;  // (x or the residual may lie there: this thread is done with it)
    const double t = (double)h * (double)p.weight[at];
    if (p.out != nullptr) p.out[row * p.out_row + at] = (float)(t * f.root);
    if constexpr (STEPS) {
      const int q = 128 + (f.factor > 0.0 ? step_of(t, totals.top, f.factor) : 0);
      count += q;
      p.steps[row * p.steps_row + at] = (uint8_t)q;
    }
  }
  if constexpr (STEPS) {
    if (p.sums != nullptr) count = row_count<1024>(count, shared_count);
    if (threadIdx.x == 0) {
      p.scales[row] = f.scale;
      if (p.sums != nullptr) p.sums[row] = count;
    }
  }
}

struct RowsArgs {
  const void* in;
  const float *scales, *columns;
  float* out;
  Divisor width;
  unsigned total;
  int offset;
};

__device__ __forceinline__ float less_offset(int v, int offset) { return (float)((long long)v - offset); }

// Four values to a thread, kRowsEach times.
constexpr unsigned kRowsThreads = 256, kRowsEach = 4;
template <class T>
__global__ __launch_bounds__(kRowsThreads) void dequantize_rows_kernel(RowsArgs p) {
  typedef T four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  const T* const in = static_cast<const T*>(p.in);
  four v[kRowsEach];
  const unsigned first = blockIdx.x * (kRowsThreads * kRowsEach) + threadIdx.x;
#pragma unroll
  for (unsigned i = 0; i < kRowsEach; ++i) {
    const unsigned at = 4 * (first + kRowsThreads * i);
    v[i] = four{};
    if (at + 4 <= p.total) {
      v[i] = *reinterpret_cast<const four*>(in + at);
    } else {
#pragma unroll
      for (unsigned j = 0; j < 3; ++j)
        if (at + j < p.total) v[i][j] = in[at + j];
    }
  }
#pragma unroll
  for (unsigned i = 0; i < kRowsEach; ++i) {
    const unsigned at = 4 * (first + kRowsThreads * i);
    if (at >= p.total) return;
    unsigned row = p.width.quotient(at), column = at - row * p.width.d;
    float scale = p.scales[row];
    f32x4 y;
#pragma unroll
    for (unsigned j = 0; j < 4; ++j) {
      if (column == p.width.d && at + j < p.total) {
        column = 0;
        scale = p.scales[++row];
      }
      y[j] = less_offset(v[i][j], p.offset) * scale;
      if (p.columns != nullptr && at + j < p.total) y[j] *= p.columns[column];
      ++column;
    }
    if (at + 4 <= p.total) {
      *reinterpret_cast<f32x4_any*>(p.out + at) = y;
    } else {
#pragma unroll
      for (unsigned j = 0; j < 3; ++j)
        if (at + j < p.total) p.out[at + j] = y[j];
    }
  }
}

}  // namespace
}  // namespace tfcc_rocm

using namespace tfcc_rocm;

extern "C" {

int tfcc_rocm_rms_norm_f32(void* stream, const tfcc_rocm_rms_norm_desc* desc) {
  TFCC_REQUIRE(desc != nullptr, "rms_norm: null descriptor");
  const tfcc_rocm_rms_norm_desc& d = *desc;
  TFCC_REQUIRE(d.width > 0 && d.width <= 0x7fffff00u / 255, "rms_norm: rows of %u values", d.width);  // sums of steps are 32-bit
  TFCC_REQUIRE(d.eps >= 0.0f && d.eps <= 3.4028234e38f, "rms_norm: eps %g", d.eps);
  TFCC_REQUIRE(d.rows <= (d.width <= 1024 ? (1u << 26) - 4 : (1u << 24) - 1) && (d.width <= 4096 || d.rows <= 0xffffffffu / 1024), "rms_norm: %u rows", d.rows);
  TFCC_REQUIRE(d.out != nullptr || d.steps != nullptr || d.rows == 0, "rms_norm: no result");
  TFCC_REQUIRE((d.steps != nullptr) == (d.scales != nullptr) && (d.steps != nullptr || d.sums == nullptr), "rms_norm: steps and scales go together");
  TFCC_REQUIRE((d.sum != d.x || d.sum_row_stride == d.x_row_stride || d.sum == nullptr) && (d.sum != d.residual || d.sum_row_stride == d.residual_row_stride || d.sum == nullptr) &&
                   (d.out != d.x || d.out_row_stride == d.x_row_stride || d.out == nullptr),
               "rms_norm: in place with other strides");
  TFCC_REQUIRE(d.out == nullptr || (d.out != d.sum && d.out != d.residual), "rms_norm: the result over the sum or the residual");
  TFCC_REQUIRE(d.rows <= 1 || ((d.sum == nullptr || d.sum_row_stride >= d.width) && (d.out == nullptr || d.out_row_stride >= d.width) &&
                               (d.steps == nullptr || d.steps_row_stride >= d.width)),
               "rms_norm: results whose rows share memory");
  if (d.rows == 0) return TFCC_ROCM_OK;
  TFCC_REQUIRE(d.x && d.weight, "rms_norm: null argument");
  const NormArgs a{d.x, d.residual, d.weight, d.sum, d.out, d.steps, d.scales, d.sums, d.x_row_stride, d.residual_row_stride, d.sum_row_stride,
                   d.out_row_stride, d.steps_row_stride, d.rows, d.width, (double)d.eps};
  const hipStream_t s = as_stream(stream);
  const auto start = [&](auto plain, auto quantized, unsigned threads, unsigned each) {
    hipLaunchKernelGGL((d.steps != nullptr ? quantized : plain), dim3((d.rows + each - 1) / each), dim3(threads), 0, s, a);
  };
  const bool few = d.rows <= kFewRows;
  if (d.width <= 64) start(rms_norm_kernel<16, 1, false>, rms_norm_kernel<16, 1, true>, 256, 16);
  else if (d.width <= 128) start(rms_norm_kernel<32, 1, false>, rms_norm_kernel<32, 1, true>, 256, 8);
  else if (d.width <= 1024 && few) start(rms_norm_kernel<256, 1, false>, rms_norm_kernel<256, 1, true>, 256, 1);
  else if (d.width <= 256) start(rms_norm_kernel<64, 1, false>, rms_norm_kernel<64, 1, true>, 256, 4);
  else if (d.width <= 512) start(rms_norm_kernel<64, 2, false>, rms_norm_kernel<64, 2, true>, 256, 4);
  else if (d.width <= 1024) start(rms_norm_kernel<64, 4, false>, rms_norm_kernel<64, 4, true>, 256, 4);
  else if (d.width <= 4096 && few && d.steps == nullptr) start(rms_norm_kernel<1024, 1, false>, nullptr, 1024, 1);
  else if (d.width <= 2048) start(rms_norm_kernel<256, 2, false>, rms_norm_kernel<256, 2, true>, 256, 1);
  else if (d.width <= 4096) start(rms_norm_kernel<256, 4, false>, rms_norm_kernel<256, 4, true>, 256, 1);
  else if (d.width <= 8192) start(rms_norm_kernel<512, 4, false>, rms_norm_kernel<512, 4, true>, 512, 1);
  else if (d.width <= kNormMost) start(rms_norm_kernel<1024, 4, false>, rms_norm_kernel<1024, 4, true>, 1024, 1);
  else start(rms_norm_wide_kernel<false>, rms_norm_wide_kernel<true>, 1024, 1);
  return check_launch("rms_norm");
}

int tfcc_rocm_dequantize_rows(void* stream, const void* in, int in_type, unsigned rows, unsigned width, int32_t offset, const float* scales,
                              const float* column_scales, float* out) {
  TFCC_REQUIRE(in_type == TFCC_ROCM_S32 || in_type == TFCC_ROCM_S8 || in_type == TFCC_ROCM_U8, "dequantize_rows: type %d", in_type);
  TFCC_REQUIRE((uint64_t)rows * width <= 0x7fffffffu, "dequantize_rows: %u rows of %u values", rows, width);
  if (rows == 0 || width == 0) return TFCC_ROCM_OK;
  TFCC_REQUIRE(in && scales && out, "dequantize_rows: null argument");
  const RowsArgs a{in, scales, column_scales, out, Divisor::of(width), rows * width, offset};
  constexpr unsigned each = 4 * kRowsThreads * kRowsEach;
  const dim3 grid((a.total + each - 1) / each), block(kRowsThreads);
  const hipStream_t s = as_stream(stream);
  if (in_type == TFCC_ROCM_S32) hipLaunchKernelGGL(dequantize_rows_kernel<int32_t>, grid, block, 0, s, a);
  else if (in_type == TFCC_ROCM_S8) hipLaunchKernelGGL(dequantize_rows_kernel<int8_t>, grid, block, 0, s, a);
  else hipLaunchKernelGGL(dequantize_rows_kernel<uint8_t>, grid, block, 0, s, a);
  return check_launch("dequantize_rows");
}

}  // extern "C"
