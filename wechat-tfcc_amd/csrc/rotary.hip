// Rotary positions.  A pair (a, b) of a head's values turns by position * frequency:
//   a' = (a cos - b sin) * magnitude,  b' = (b cos + a sin) * magnitude.
// Bound: HBM, 8 bytes for each value (4096 tokens of 32 + 8 heads of 128, 168 MB: 28 us, 6.0 TB/s with what the last-level cache holds of it; one token:
// 2.4 us).  The angles are those of a token, not of a head: a workgroup takes one token, forms the
// sines and cosines of its part / 2 pairs once in LDS and runs over its share of the heads.  The angle is a product in 64 bits,
// reduced to a fraction of a turn there: position 10^6 at one radian a position loses 2^-33 of a radian, where float32 would be
// off by 0.06.  The fraction and its sine and cosine are float32: it is off by 2^-26 of a turn at most, 0.8 of a unit in the last place of what it turns
// (4096 tokens at far positions: 5.9e-8 from 64 bits, with angles rounded to nothing less than that 4.2e-8).
#include <math.h>

#include "common.hpp"

namespace tfcc_rocm {
namespace {

struct RotaryArgs {
  const float* in[2];
  float* out[2];
  unsigned long long in_token[2], in_head[2], out_token[2], out_head[2];
  unsigned heads[2];
  unsigned size, part;
  const void* positions;
  const double* frequencies;
  float magnitude;
  int wide_positions, copy_rest[2];
};

constexpr unsigned kRotaryThreads = 256;
constexpr unsigned kRotaryMost = 1024;  // values of a head

// VEC values at a time: of one half and its partners in the other, or VEC / 2 neighbouring pairs.
template <bool INTERLEAVED, int VEC>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryArgs p) {
  __shared__ __align__(16) float cosines[kRotaryMost / 2];
  __shared__ __align__(16) float sines[kRotaryMost / 2];
  const unsigned token = blockIdx.x;
  const long long position = p.wide_positions ? static_cast<const long long*>(p.positions)[token] : static_cast<const int*>(p.positions)[token];
  const unsigned half = p.part / 2;
  for (unsigned i = threadIdx.x; i < half; i += kRotaryThreads) {
    // 1 / (2 pi) in two parts, and the first product's rounding kept: 2^31 positions make 3 x 10^8 turns
    const double angle = (double)position * p.frequencies[i], whole = angle * 0.15915494309189535;
    const double turns = (whole - rint(whole)) + fma(angle, 0.15915494309189535, -whole) + angle * -9.839338337591243e-18;
    float s, c;
    sincospif(2.0f * (float)turns, &s, &c);
    cosines[i] = c * p.magnitude;
    sines[i] = s * p.magnitude;
  }
  __syncthreads();
  // loads and stores of several floats need no more than a float's alignment
  typedef float vec __attribute__((ext_vector_type(VEC), aligned(4)));
  constexpr int REST = VEC == 4 ? 4 : 1;
  typedef float rest_vec __attribute__((ext_vector_type(REST), aligned(4)));
  const unsigned rest = (p.size - p.part) / REST;
  for (int which = 0; which < 2; ++which) {
    if (p.in[which] == nullptr) break;
    const float* in = p.in[which] + token * p.in_token[which];
    float* out = p.out[which] + token * p.out_token[which];
    const unsigned each = (INTERLEAVED ? p.part : half) / VEC, per_head = each + (p.copy_rest[which] ? rest : 0);
    const unsigned total = per_head * p.heads[which];
    for (unsigned at = blockIdx.y * kRotaryThreads + threadIdx.x; at < total; at += gridDim.y * kRotaryThreads) {
      const unsigned head = at / per_head, v = at - head * per_head;
      const float* x = in + head * p.in_head[which];
      float* y = out + head * p.out_head[which];
      if (v >= each) {
        const unsigned d = p.part + (v - each) * REST;
        *reinterpret_cast<rest_vec*>(y + d) = *reinterpret_cast<const rest_vec*>(x + d);
      } else if constexpr (INTERLEAVED) {
        const unsigned d = v * VEC;
        const vec a = *reinterpret_cast<const vec*>(x + d);
        vec r;
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const float c = cosines[d / 2 + i], s = sines[d / 2 + i];
          r[2 * i] = a[2 * i] * c - a[2 * i + 1] * s;
          r[2 * i + 1] = a[2 * i + 1] * c + a[2 * i] * s;
        }
        *reinterpret_cast<vec*>(y + d) = r;
      } else {
        const unsigned d = v * VEC;
        const vec a = *reinterpret_cast<const vec*>(x + d), b = *reinterpret_cast<const vec*>(x + d + half);
        const vec c = *reinterpret_cast<const vec*>(cosines + d), s = *reinterpret_cast<const vec*>(sines + d);
        *reinterpret_cast<vec*>(y + d) = a * c - b * s;
        *reinterpret_cast<vec*>(y + d + half) = b * c + a * s;
      }
    }
  }
}

}  // namespace
}  // namespace tfcc_rocm

using namespace tfcc_rocm;

extern "C" {

int tfcc_rocm_rotary_frequencies(unsigned part, double base, int scaling, double factor, unsigned original_length, double low,
                                 double high, double* frequencies, float* magnitude) {
  TFCC_REQUIRE(frequencies != nullptr, "rotary_frequencies: null argument");
  TFCC_REQUIRE(part >= 2 && part % 2 == 0 && part <= kRotaryMost, "rotary_frequencies: part %u is not even from 2 to %u", part, kRotaryMost);
  TFCC_REQUIRE(base > 0 && std::isfinite(base), "rotary_frequencies: base %g", base);
  TFCC_REQUIRE(scaling >= TFCC_ROCM_ROTARY_PLAIN && scaling <= TFCC_ROCM_ROTARY_INDEX, "rotary_frequencies: scaling %d", scaling);
  TFCC_REQUIRE(scaling == TFCC_ROCM_ROTARY_PLAIN || (factor > 0 && std::isfinite(factor)), "rotary_frequencies: factor %g", factor);
  const bool ramp = scaling == TFCC_ROCM_ROTARY_TURNS || scaling == TFCC_ROCM_ROTARY_INDEX;
  TFCC_REQUIRE(!ramp || (original_length > 0 && low > 0 && high > low && std::isfinite(high)),
               "rotary_frequencies: original_length %u, turns from %g to %g", original_length, low, high);
  TFCC_REQUIRE(scaling != TFCC_ROCM_ROTARY_BASE || part > 2, "rotary_frequencies: a single pair has no base to change");
  TFCC_REQUIRE(scaling != TFCC_ROCM_ROTARY_INDEX || base > 1, "rotary_frequencies: base %g has no falling frequencies", base);
  const double pi2 = 6.283185307179586477;
  if (scaling == TFCC_ROCM_ROTARY_BASE) base *= pow(factor, part / (part - 2.0));
  double first = 0, last = 0;  // of the falling ramp over indices
  if (scaling == TFCC_ROCM_ROTARY_INDEX) {
    const auto index_of = [&](double turns) { return part * log(original_length / (turns * pi2)) / (2 * log(base)); };
    first = fmax(0.0, floor(index_of(high)));
    last = ceil(index_of(low));  // behind the last pair where that makes more than `low` turns
    if (last <= first) last = first + 0.001;
  }
  for (unsigned i = 0; i < part / 2; ++i) {
    const double f = pow(base, -2.0 * i / part);
    double r = 1.0;
    if (scaling == TFCC_ROCM_ROTARY_LINEAR) r = 0.0;
    if (scaling == TFCC_ROCM_ROTARY_TURNS) r = fmin(1.0, fmax(0.0, (original_length * f / pi2 - low) / (high - low)));
    if (scaling == TFCC_ROCM_ROTARY_INDEX) r = 1.0 - fmin(1.0, fmax(0.0, (i - first) / (last - first)));
    frequencies[i] = r == 1.0 ? f : f * (r + (1.0 - r) / factor);
  }
  if (magnitude != nullptr) *magnitude = scaling == TFCC_ROCM_ROTARY_INDEX && factor > 1 ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
  return TFCC_ROCM_OK;
}

int tfcc_rocm_rotary_f32(void* stream, const tfcc_rocm_rotary_desc* desc) {
  TFCC_REQUIRE(desc != nullptr, "rotary: null descriptor");
  const tfcc_rocm_rotary_desc& d = *desc;
  TFCC_REQUIRE(d.size > 0 && d.size <= kRotaryMost, "rotary: heads of %u values (1 to %u)", d.size, kRotaryMost);
  TFCC_REQUIRE(d.part >= 2 && d.part % 2 == 0 && d.part <= d.size, "rotary: part %u of heads of %u values", d.part, d.size);
  TFCC_REQUIRE(d.position_type == TFCC_ROCM_S32 || d.position_type == TFCC_ROCM_S64, "rotary: position type %d", d.position_type);
  TFCC_REQUIRE((uint64_t)d.tokens * kRotaryThreads <= 0xffffffffu, "rotary: %u tokens", d.tokens);  // of a launch
  TFCC_REQUIRE(d.in[1] != nullptr || d.out[1] == nullptr, "rotary: a second result without a second input");
  if (d.tokens == 0) return TFCC_ROCM_OK;
  TFCC_REQUIRE(d.in[0] && d.out[0] && d.positions && d.frequencies, "rotary: null argument");
  RotaryArgs a{};
  unsigned heads = 0;
  for (int i = 0; i < 2 && d.in[i] != nullptr; ++i) {
    TFCC_REQUIRE(d.out[i] != nullptr, "rotary: null argument");
    TFCC_REQUIRE(d.heads[i] > 0 && d.heads[i] <= 65536, "rotary: %u heads", d.heads[i]);
    TFCC_REQUIRE(d.in[i] != d.out[i] || (d.in_token_stride[i] == d.out_token_stride[i] && d.in_head_stride[i] == d.out_head_stride[i]),
                 "rotary: in place with other strides");
    a.in[i] = d.in[i];
    a.out[i] = d.out[i];
    a.in_token[i] = d.in_token_stride[i];
    a.in_head[i] = d.in_head_stride[i];
    a.out_token[i] = d.out_token_stride[i];
    a.out_head[i] = d.out_head_stride[i];
    a.heads[i] = d.heads[i];
    a.copy_rest[i] = d.in[i] != d.out[i] && d.part < d.size;
    heads += d.heads[i];
  }
  a.size = d.size;
  a.part = d.part;
  a.positions = d.positions;
  a.frequencies = d.frequencies;
  a.magnitude = d.magnitude;
  a.wide_positions = d.position_type == TFCC_ROCM_S64;
  // four values at a time where halves and heads hold a multiple of four
  const bool wide = d.size % 4 == 0 && d.part % (d.interleaved ? 4 : 8) == 0;
  // few tokens: a token's heads are shared by two workgroups, which each form its angles (32 + 8 heads of 128, 16 tokens: 2.7 us, with one 3.0, with
  // four 2.7; 256: 3.35, 3.7 and 3.4; 1024: 7.1 either way, with four 7.4)
  const unsigned steps = (heads * d.size / (wide ? 8 : 2) + kRotaryThreads - 1) / kRotaryThreads;
  const unsigned share = steps > 1 && d.tokens < 512 ? 2 : 1;
  const dim3 grid(d.tokens, share), block(kRotaryThreads);
  const hipStream_t s = as_stream(stream);
  if (d.interleaved) {
    if (wide) hipLaunchKernelGGL((rotary_kernel<true, 4>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((rotary_kernel<true, 2>), grid, block, 0, s, a);
  } else if (wide) {
    hipLaunchKernelGGL((rotary_kernel<false, 4>), grid, block, 0, s, a);
  } else {
    hipLaunchKernelGGL((rotary_kernel<false, 1>), grid, block, 0, s, a);
  }
  return check_launch("rotary");
}

}  // extern "C"
