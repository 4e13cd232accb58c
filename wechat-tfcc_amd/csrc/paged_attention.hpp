// Attention of new tokens over a paged cache: out = softmax(c q k^T) v for the chunk of each sequence, one pass over the keys with
// the running maximum and sum of each row.
//
// The query heads of a token that share a cache head are rows of one product: row r of a sequence is token r / group, head r % group, and
// a tile holds 16 rows, or 128 or 256 of chunks of many tokens.  Both products run transposed on the matrix cores, with a row in each column:
//   S^T = K Q^T   (16 keys x 16 rows): lane l holds row l % 16 and keys 4 (l / 16) + i, i < 4
//   O^T = V^T P^T (16 values x 16 rows)
// so a row's maximum, sum and scale sit in the lanes that hold its scores, and the scores are where the second product wants its
// right operand: a contraction may run over the keys in any order, so lane group g contracts the keys that it holds.  Nothing is
// exchanged between lanes but two steps of the row maximum.  V is loaded as it lies, row by row; which column of the
// product stands for which value of a head is free as well and follows the loads.
//
// An int8 cache keeps float32 accuracy: an int8 is exact in fp16, a float32 is the sum of two but for 2^-23 of it, so each product is two
// fp16 matrix operations.  Queries are scaled by a power of two for each row.  What meets the values is a weight times a value's scale, and
// what has to stay in fp16's range is that product, not the weight: a row's weights are 2^(score - frame), and the frame moves where
// score + log2(scale) exceeds it by 15, to 8 below.  Between moves nothing is rescaled, and what fp16 cannot hold is 2^-32 of
// the largest product or less.  The sum of the weights is kept in the same frame.  Integers of 4 bits are those of 8 but for the way they are unpacked: the
// bytes on their way halve, the operations do not.  A float32 cache goes through the fp32 matrix operations, and
// chunks of many tokens over one through three fp16 operations of pieces, which take two fifths of the time.
//
// The keys of a tile are dealt to the wavefronts of a workgroup in turns, and in pieces to several workgroups where there are few tiles; each
// wavefront keeps frame, sum and output of its own, joined in LDS, the pieces by a second launch.  A frame of -infinity: no key was seen.
#pragma once

#include <type_traits>

#include "lds_dma.hpp"
#include "paged_attention_plan.hpp"
#include "paged_cache.hpp"
#include "score_tanh.hpp"

namespace tfcc_rocm {

struct AttentionArgs {
  CacheView cache;
  const float* q;
  float* out;
  unsigned long long q_token, q_head, out_token, out_head;
  unsigned tokens, batch;
  const int *starts, *lengths, *table;
  unsigned long long table_stride;
  unsigned table_width, max_length;
  float scale;  // times log2 e
  int causal;
  unsigned window;
  Divisor group, cache_heads, pieces;
  float *partial, *statistics;  // [splits][tokens][heads][size], [splits][tokens][heads][2]
  unsigned splits, split_keys;
  int longest_first;  // 0: sequences in the batch's order, else by length / 2^(longest_first - 1)
  // of shaped scores: a cap in the units of log2 and its inverse (0: none), a slope for each query head, a prefix of each sequence
  float cap, cap_inverse;
  const float* slopes;
  const int* prefixes;
};

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned long long u64;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// What a workgroup works on; the same in all its lanes but for the row's members.
struct Tile {
  bool any;
  unsigned sequence;
  int first, count;      // of the chunk's tokens
  int row0;              // of the tile within the chunk's rows
  int length;            // keys that are there
  int low, high;         // keys that some row sees
  int all_low, all_high; // keys that every row sees
  int row_token, row_head;  // of this lane's row; token < 0: no such row
  int row_low, row_high;
  int row_position;         // for shaped scores
};

// The value of the lane that a data-parallel move names, 0 where there is none.
template <int CONTROL, int ROWS>
__device__ __forceinline__ unsigned moved(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, ROWS, 0xf, false);
}
// Sums of the lanes up to each: 1, 2, 4 and 8 lanes along the rows of 16, then on from row to row and from half to half.
__device__ __forceinline__ unsigned wave_scan(unsigned v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}

// The chunks' tiles are counted off along the batch, 64 sequences at a time; with longest_first (a shift and 1) those
// 64 are taken by falling length, in 16 buckets: workgroups begin in their order, and where there are more than run at once, a long one that begins late is what the others
// have to wait for (64 sequences of 1024 to 4096, 8 heads of 128: 4 bits 48 us, in the batch's order 56, int8 80 and 85; 12 chunks of 500 over up to 3000, 4 bits: 313 and 364).
template <bool SHAPED>
__device__ __forceinline__ Tile find_tile(const AttentionArgs& p, unsigned tile, unsigned rows_of_tile, unsigned row) {
  const unsigned lane = threadIdx.x & 63;
  Tile t;
  t.any = false;
  unsigned before = 0;
  int length = 0;
#pragma unroll 1
  for (unsigned base = 0; base < p.batch; base += 64) {
    const unsigned b = base + lane;
    int first = 0, count = 0, held = 0;
    if (b < p.batch) {
      first = p.starts[b];
      int next = p.starts[b + 1];
      held = p.lengths[b];
      next = next > (int)p.tokens ? (int)p.tokens : next;
      count = first >= 0 && next > first ? next - first : 0;
    }
    unsigned mine = ((unsigned)count * p.group.d + rows_of_tile - 1) / rows_of_tile, upto = wave_scan(mine) + before;
    unsigned long long past = __ballot(upto > tile);
    if (past != 0) {
      unsigned from = b;
      if (p.longest_first != 0) {
        const unsigned there = p.batch - base < 64 ? p.batch - base : 64;
        const int bucket = lane >= there ? -1 : held <= 0 ? 0 : (held >> (p.longest_first - 1)) < 15 ? held >> (p.longest_first - 1) : 15;
        unsigned rank = lane, longer = 0;  // lanes behind the batch stay where they are
#pragma unroll
        for (int i = 15; i >= 0; --i) {
          const unsigned long long equal = __ballot(bucket == i);
          const unsigned before_me = __builtin_amdgcn_mbcnt_hi((unsigned)(equal >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)equal, longer));
          rank = bucket == i ? before_me : rank;
          longer += (unsigned)__builtin_popcountll(equal);
        }
        const auto sent = [&](int v) { return __builtin_amdgcn_ds_permute((int)(4 * rank), v); };
        first = sent(first);
        count = sent(count);
        held = sent(held);
        mine = (unsigned)sent((int)mine);
        from = (unsigned)sent((int)b);
        upto = wave_scan(mine) + before;
        past = __ballot(upto > tile);
      }
      const int at = __builtin_ctzll(past);
      t.any = true;
      t.sequence = (unsigned)__builtin_amdgcn_readlane((int)from, at);
      t.first = __builtin_amdgcn_readlane(first, at);
      t.count = __builtin_amdgcn_readlane(count, at);
      length = __builtin_amdgcn_readlane(held, at);
      unsigned within = tile - (unsigned)__builtin_amdgcn_readlane((int)(upto - mine), at);
      // of a chunk the last rows, which see most
      if (p.longest_first != 0) within = (unsigned)__builtin_amdgcn_readlane((int)mine, at) - 1 - within;
      t.row0 = (int)(within * rows_of_tile);
      break;
    }
    before = (unsigned)__builtin_amdgcn_readlane((int)upto, 63);
  }
  if (!t.any) return t;
  length = length < 0 ? 0 : length;
  const int position0 = length - t.count;  // of the chunk's first token
  t.length = length < (int)p.max_length ? length : (int)p.max_length;
  const int rows = t.count * (int)p.group.d;
  const int last_row = t.row0 + (int)rows_of_tile < rows ? t.row0 + (int)rows_of_tile - 1 : rows - 1;
  const int token0 = (int)p.group.quotient((unsigned)t.row0), token1 = (int)p.group.quotient((unsigned)last_row);
  int prefix = 0;
  if constexpr (SHAPED)
    if (p.prefixes != nullptr) prefix = p.prefixes[__builtin_amdgcn_readfirstlane((int)t.sequence)];
  const auto sight = [&](int token, int& low, int& high) {
    low = 0;
    high = t.length;
    if (p.causal) {
      const int position = position0 + token, upto = SHAPED && position + 1 < prefix ? prefix : position + 1;
      high = upto < t.length ? upto : t.length;
      if (p.window > 0 && (long long)position + 1 > (long long)p.window) low = position + 1 - (int)p.window;
    }
  };
  sight(token0, t.low, t.all_high);
  sight(token1, t.all_low, t.high);
  const int r = t.row0 + (int)row;
  t.row_token = -1;
  t.row_head = 0;
  t.row_low = 0;
  t.row_high = 0;
  t.row_position = 0;
  if (r < rows) {
    t.row_token = (int)p.group.quotient((unsigned)r);
    t.row_head = r - t.row_token * (int)p.group.d;
    sight(t.row_token, t.row_low, t.row_high);
    t.row_position = position0 + t.row_token;
  }
  return t;
}

__device__ __forceinline__ float across_groups_max(float v) {
  float a, b;
  butterfly_pair<16>(v, a, b);
  v = fmaxf(a, b);
  butterfly_pair<32>(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float across_groups_sum(float v) {
  float a, b;
  butterfly_pair<16>(v, a, b);
  v = a + b;
  butterfly_pair<32>(v, a, b);
  return a + b;
}

// The largest of neighbouring lanes, LANES of them.
template <int LANES>
__device__ __forceinline__ unsigned lanes_max(unsigned v) {
  const auto larger = [](unsigned a, unsigned b) { return a > b ? a : b; };
  v = larger(v, moved<0xb1, 0xf>(v));  // lanes 1, 2, then those of a half row from its other end, then 8 apart
  v = larger(v, moved<0x4e, 0xf>(v));
  if constexpr (LANES >= 8) v = larger(v, moved<0x141, 0xf>(v));
  if constexpr (LANES >= 16) v = larger(v, moved<0x128, 0xf>(v));
  if constexpr (LANES >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = larger(r[0], r[1]);
  }
  if constexpr (LANES >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = larger(r[0], r[1]);
  }
  return v;
}
// The frame that goes out with a sum: scores of NaN raise none, but a row that has one is not a row without keys.
__device__ __forceinline__ float frame_out(float frame, float sum) { return sum != sum && frame == -INFINITY ? 0.0f : frame; }
// 2^e for e in [-126, 127]; infinity for 128
__device__ __forceinline__ float power(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
// e with |v| < 2^e, from -100 to 128, so that 2^(14 - e) and its inverse are normal numbers
__device__ __forceinline__ int bound_of(float v) {
  const int e = (int)((__float_as_uint(v) >> 23) & 255) - 126;
  return e < -100 ? -100 : (e > 128 ? 128 : e);
}

// A row's scores with a cap and a bias that depends on distance.  In the units of log2, as all scores here.
//
// tanh (score_tanh.hpp) has two forms, and most scores are far below their cap: where those of a whole wavefront are, the second is passed over.  A score as
// it comes (`raw`) takes the factor of its row and the cap's inverse in one, and leaves in units of `unit`, the cap where nothing is added to it: a
// cap costs nine operations, a bias two (int8, 32 sequences of up to 6000 with a window of 4096, 8 heads of 256, at the rate of HBM: 97 us with a cap, 92 without; 4 chunks of 1024
// over 4096 in 4 bits: 380 us plain, 500 with a cap, 417 with slopes).
// The bias is slope * distance.  A row's softmax does not change with what all its scores have in common, so a position behind the last key
// that the row may see counts as that key's, and one before the first as the first's: differences are whole numbers, exact up to 2^24.
struct ScoreShape {
  float cap = 0.0f, slope = 0.0f, factor = 1.0f, unit = 1.0f;
  int position = 0;
  bool biased = false;

  // factor_of_row: of the scores as they come
  __device__ __forceinline__ void start(const AttentionArgs& p, const Tile& t, unsigned head, float factor_of_row) {
    cap = p.cap;
    biased = p.slopes != nullptr;
    factor_of_row = fminf(factor_of_row, 3.4028234e38f);  // a score of 0 stays one where the factor overflows
    factor = cap > 0.0f ? fminf(factor_of_row * p.cap_inverse, 3.4028234e38f) : biased ? factor_of_row : 1.0f;
    unit = biased ? 1.0f : cap > 0.0f ? cap : factor_of_row;
    if (biased && t.row_token >= 0) {
      slope = p.slopes[head * p.group.d + t.row_head] * 1.44269504088896341f;
      if (fabsf(slope) == INFINITY) slope = copysignf(3.4028234e38f, slope);  // times a distance of 0 it stays 0
      position = t.row_position < t.row_high - 1 ? t.row_position : t.row_high - 1;
      position = position > 0 ? position : 0;
    }
  }
  // key: of s[0]; AWAY(i): that of s[i] less it
  template <int N, class Away>
  __device__ __forceinline__ void apply(float (&s)[N], int key, Away away) const {
    if (cap > 0.0f) {
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        s[i] *= factor;
        most = fmaxf(most, fabsf(s[i]));
      }
      const bool large = __any(!(most < kTanhNear));
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float x = s[i];
        float r = tanh_near(x);
        if (large) {
          const float far = tanh_far(x, [](float v) { return __builtin_amdgcn_exp2f(v); }, [](float v) { return __builtin_amdgcn_rcpf(v); });
          r = fabsf(x) < kTanhNear ? r : far;
        }
        s[i] = r;
      }
    }
    if (biased) {
      const float first = (float)(key - position), times = cap > 0.0f ? cap : factor;
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] = fmaf(-slope, fabsf(first + (float)away(i)), s[i] * times);
    }
  }
};

// two of the bytes of a and b as fp16, exactly: 0x6400 + u is 1024 + u, and u = byte ^ 0x80 is the int8 + 128
template <unsigned A, unsigned B>
__device__ __forceinline__ f16x2 two_int8(unsigned a, unsigned b) {
  const unsigned u = __builtin_amdgcn_perm(b, a, A | 0x0c00u | (4 + B) << 16 | 0x0c000000u) ^ 0x64806480u;
  const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
  return __builtin_bit_cast(f16x2, u) - bias;
}

union Half8 {
  f16x8 v;
  f16x2 p[4];
};

// Eight int8 that lie side by side.
__device__ __forceinline__ f16x8 eight_int8(unsigned lo, unsigned hi) {
  Half8 h;
  h.p[0] = two_int8<0, 1>(lo, lo);
  h.p[1] = two_int8<2, 3>(lo, lo);
  h.p[2] = two_int8<0, 1>(hi, hi);
  h.p[3] = two_int8<2, 3>(hi, hi);
  return h.v;
}
// Byte B of eight words.
template <unsigned B>
__device__ __forceinline__ f16x8 eight_of(const unsigned (&w)[8]) {
  Half8 h;
#pragma unroll
  for (int i = 0; i < 4; ++i) h.p[i] = two_int8<B, B>(w[2 * i], w[2 * i + 1]);
  return h.v;
}

// The integers of 4 bits of a word as fp16, exactly: out[i] holds those of its bits 4 i and 16 + 4 i, i < 4.  As above with u the int4 + 8, whose highest bit is
// the other one; where it lies four bits up, 0x6400 + 16 u is 1024 + 16 u, a sixteenth of which is 64 + u.  (Two operations for two integers: the mask, the bit and
// the bias are one.)
__device__ __forceinline__ void eight_int4(unsigned w, f16x2 (&out)[4]) {
  const unsigned low = 0x000f000fu, low_bias = 0x64086408u, high = 0x00f000f0u, high_bias = 0x64806480u;
  const f16x2 less = {(_Float16)1032.0f, (_Float16)1032.0f}, sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f}, less_high = {(_Float16)-72.0f, (_Float16)-72.0f};
  const unsigned v = w >> 8;
  out[0] = __builtin_bit_cast(f16x2, (w & low) ^ low_bias) - less;
  out[1] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (w & high) ^ high_bias), sixteenth, less_high);
  out[2] = __builtin_bit_cast(f16x2, (v & low) ^ low_bias) - less;
  out[3] = __builtin_elementwise_fma(__builtin_bit_cast(f16x2, (v & high) ^ high_bias), sixteenth, less_high);
}
// The eight of a word: in the order 0, 4, 1, 5, 2, 6, 3, 7, which the other factor of a product follows.
__device__ __forceinline__ f16x8 word_int4(unsigned w) {
  Half8 h;
  eight_int4(w, h.p);
  return h.v;
}
// Integer 4 HIGH + e of eight words in out[e], e < 4.
template <int HIGH>
__device__ __forceinline__ void four_of_int4(const unsigned (&w)[8], f16x8 (&out)[4]) {
  Half8 h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f16x2 pair[4];
    eight_int4(__builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], HIGH ? 0x07060302u : 0x05040100u), pair);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e].p[i] = pair[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = h[e].v;
}

// float32 as the sum of two fp16, both to the nearest: the second is 2^-11 of the value at most and the error 2^-23, or half of fp16's smallest number, 2^-25
__device__ __forceinline__ void split_two(float a, float b, f16x2& hi, f16x2& lo) {
  hi = __builtin_convertvector(f32x2{a, b}, f16x2);
  // a - hi, which is exact: one operation that takes half a register as fp16 (of a conversion and a difference the compiler makes two)
  float rest_a, rest_b;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(rest_a) : "v"(hi), "v"(a));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rest_b) : "v"(hi), "v"(b));
  lo = __builtin_convertvector(f32x2{rest_a, rest_b}, f16x2);
}

// Powers of two for a row of queries whose largest value is `top`: `up` brings it to 2^13 .. 2^14 under the sign of the scale (0 for a scale of 0),
// `scale` undoes that and is the positive factor of the scores.
struct QueryScale {
  float up, scale;
};
__device__ __forceinline__ QueryScale query_scale(float top, float scale) {
  const int e = bound_of(top);
  const float up = power(14 - e);
  return {scale > 0.0f ? up : scale < 0.0f ? -up : 0.0f * scale, scale != 0.0f ? fmaxf(power(e - 14) * fabsf(scale), 1.17549435e-38f) : 1.0f};
}
// The factor from one frame to a higher one is the square of this.  Sums of weights are multiplied by it twice: where the scales of the values
// span more than float32's exponents, a sum of 2^90 in the lower frame may be all there is in the higher, and the square itself underflows.
__device__ __forceinline__ float half_step(float from, float to) { return __builtin_amdgcn_exp2f(0.5f * (from - to)); }
// log2 of a value's scale for the frame.  A row of zeros, whose scale is 0, counts like one of 2^-90: its weight is summed and may not overflow.
__device__ __forceinline__ float frame_log(float value_scale) { return fmaxf(__builtin_amdgcn_logf(fabsf(value_scale)), -90.0f); }

// Joins the wavefronts' outputs and writes them: to `out` where the keys are in one piece, else to the piece's part of the workspace.
// o[] of a lane is its row's value `place(n)`; four neighbours in n are four neighbours in memory.
template <int DPAD, int WAVES>
struct Joining {
  static constexpr int LD = DPAD + 4;
  alignas(16) float outputs[WAVES][kAttentionRows][LD];
  float maxima[WAVES][kAttentionRows], sums[WAVES][kAttentionRows];
};
template <int DPAD, int WAVES, class Place>
__device__ __forceinline__ void join_and_store(Joining<DPAD, WAVES>& s, const AttentionArgs& p, const Tile& t, unsigned head, unsigned split, float m, float l, const float* o, Place place) {
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x / 64, row = lane % 16;
  constexpr int N = DPAD / 4;  // of a lane: 16 rows of DPAD values over 64 lanes
  if (lane < 16) {
    s.maxima[wave][row] = m;
    s.sums[wave][row] = l;
  }
#pragma unroll
  for (int n = 0; n < N; n += 4) {
    const f32x4 v = {o[n], o[n + 1], o[n + 2], o[n + 3]};
    *reinterpret_cast<f32x4*>(&s.outputs[wave][row][place(n)]) = v;
  }
  __syncthreads();
  const unsigned size = p.cache.size, heads = p.cache.heads * p.group.d;
  const int rows = t.count * (int)p.group.d;
  for (unsigned at = threadIdx.x; at < kAttentionRows * (DPAD / 4); at += (WAVES * 64)) {
    const unsigned r = at / (DPAD / 4), d = at % (DPAD / 4) * 4;
    const int in_chunk = t.row0 + (int)r;
    if (in_chunk >= rows || d >= size) continue;
    float top = s.maxima[0][r];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) top = fmaxf(top, s.maxima[w][r]);
    float total = 0;
    f32x4 sum = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (s.maxima[w][r] == -INFINITY) continue;  // a wavefront that saw no key of this row
      const float h = half_step(s.maxima[w][r], top);
      total += s.sums[w][r] * h * h;
      sum += h * h * *reinterpret_cast<const f32x4*>(&s.outputs[w][r][d]);
    }
    const unsigned token = p.group.quotient((unsigned)in_chunk), inner = (unsigned)in_chunk - token * p.group.d;
    const unsigned long long global = t.first + token, query_head = head * p.group.d + inner;
    if (p.splits == 1) {
      const f32x4 none = {0, 0, 0, 0};
      *reinterpret_cast<f32x4*>(p.out + global * p.out_token + query_head * p.out_head + d) = top == -INFINITY ? none : sum / total;
    } else {
      const unsigned long long place_of = ((unsigned long long)split * p.tokens + global) * heads + query_head;
      *reinterpret_cast<f32x4*>(p.partial + place_of * size + d) = sum;
      if (d == 0) {
        p.statistics[place_of * 2] = top;
        p.statistics[place_of * 2 + 1] = total;
      }
    }
  }
}

// The workgroup's tile, cache head and piece of the keys; false: nothing to do here.  A piece without keys still says so to the
// launch that joins the pieces.
template <bool SHAPED>
__device__ __forceinline__ bool take_work(const AttentionArgs& p, unsigned rows_of_tile, unsigned row, Tile& t, unsigned& head, unsigned& split, int& begin, int& end) {
  // cache heads first, then pieces, then tiles
  const unsigned outer = p.cache_heads.quotient(blockIdx.x), tile = p.pieces.quotient(outer);
  head = blockIdx.x - outer * p.cache_heads.d;
  split = outer - tile * p.pieces.d;
  t = find_tile<SHAPED>(p, tile, rows_of_tile, row);
  if (!t.any) return false;
  const long long from = (t.low & ~31) + (long long)split * p.split_keys, upto = from + p.split_keys;
  end = upto < t.high ? (int)upto : t.high;
  begin = from < end ? (int)from : end;
  if (begin >= end && p.splits > 1) {
    if (t.row_token >= 0) {  // several lanes write the same for a row
      const unsigned long long at = ((unsigned long long)split * p.tokens + t.first + t.row_token) * p.cache.heads * p.group.d + head * p.group.d + t.row_head;
      p.statistics[at * 2] = -INFINITY;
      p.statistics[at * 2 + 1] = 0.0f;
    }
    return false;
  }
  return true;
}

// 16 bytes of each lane's own address to LDS, lane i's to m0 + 16 i.
__device__ __forceinline__ void dma16_global(const void* from, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(to), "v"(from) : "memory", "m0");
}

__device__ __forceinline__ void dma4_global(const void* from, unsigned to) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off" : : "s"(to), "v"(from) : "memory", "m0");
}

// The page that holds a key, in two halves: what the table says of it, and, when that is wanted, whether there is such a page (-1: none).
// What is loaded in one step is looked at in the next: a step does not wait for the table.
// (Constant memory as far as a launch goes, so that entries come through the scalar cache: among the vector loads, which return in their order,
// one would have to wait for all the rows that are on their way.)
struct PageEntry {
  int named;
  bool listed;
};
typedef const __attribute__((address_space(4))) int* ConstantInts;
__device__ __forceinline__ PageEntry entry_of(const AttentionArgs& p, const int* table, unsigned index) {  // a table that has a column
  const bool listed = index < p.table_width;
  return {((ConstantInts)table)[listed ? index : 0], listed};
}
__device__ __forceinline__ int page_of(const AttentionArgs& p, const PageEntry& e) {
  return e.listed && (unsigned)e.named < p.cache.pages ? e.named : -1;
}
// The page that holds a key; -1: none.
__device__ __forceinline__ int page_of(const AttentionArgs& p, const int* table, unsigned index) {
  if (index >= p.table_width) return -1;
  const int page = table[index];
  return page >= 0 && (unsigned)page < p.cache.pages ? page : -1;
}

// How rows of 64 BLOCKS integers go to lanes: PER of them to a byte, BYTES in a row, N to a lane as values, and as keys RUN (of 16 bytes, or 8 where a row has
// 32) side by side in each 4 RUN of them.
template <int TYPE, int BLOCKS>
struct ScaledLayout {
  static constexpr int PER = TYPE == TFCC_ROCM_S4 ? 2 : 1, BYTES = 64 * BLOCKS / PER, N = 4 * BLOCKS, RUN = BYTES < 64 ? 8 * PER : 16 * PER, KS = 2 * BLOCKS,
                       KEY_WORDS = BYTES / 16, VALUE_WORDS = BYTES < 64 ? 1 : BYTES / 64;
};

// A tile's rows over a cache of integers: queries and running results of one wavefront.
template <int TYPE, int BLOCKS, bool SHAPED>
struct ScaledRows : ScaledLayout<TYPE, BLOCKS> {
  using Layout = ScaledLayout<TYPE, BLOCKS>;
  using Layout::KEY_WORDS;
  using Layout::KS;
  using Layout::N;
  using Layout::RUN;
  using Layout::VALUE_WORDS;
  f16x8 q_hi[KS], q_lo[KS];                  // the lane's values of the head, eight side by side in each, in the order in which integers come out of words, as two fp16 under a power of two
  f32x4 o[N];                                // value N (4 g + i) + n in [n][i]
  float row_scale, frame = -INFINITY, l = 0.0f;
  ScoreShape shape;

  __device__ __forceinline__ void start(const AttentionArgs& p, const Tile& t, unsigned head, unsigned g) {
    f32x4 x[2 * KS];
    float top = 0.0f;
    const float* q = p.q + (unsigned long long)(t.first + (t.row_token < 0 ? 0 : t.row_token)) * p.q_token + (head * p.group.d + t.row_head) * p.q_head;
#pragma unroll
    for (int b = 0; b < 2 * KS; ++b) {
      const unsigned d = 4 * RUN * (4 * b / RUN) + RUN * g + 4 * b % RUN;
      f32x4 v = {0, 0, 0, 0};
      if (t.row_token >= 0 && d < p.cache.size) v = *reinterpret_cast<const f32x4*>(q + d);
      x[b] = v;
    }
#pragma unroll
    for (int b = 0; b < 2 * KS; ++b)
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(x[b][j]));
    const QueryScale scale = query_scale(across_groups_max(top), p.scale);
    const float up = scale.up;
    row_scale = scale.scale;
#pragma unroll
    for (int b = 0; b < KS; ++b) {
      Half8 hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (TYPE == TFCC_ROCM_S4) split_two(x[2 * b][j] * up, x[2 * b + 1][j] * up, hi.p[j], lo.p[j]);
        else split_two(x[2 * b + j / 2][j % 2 * 2] * up, x[2 * b + j / 2][j % 2 * 2 + 1] * up, hi.p[j], lo.p[j]);
      }
      q_hi[b] = hi.v;
      q_lo[b] = lo.v;
    }
#pragma unroll
    for (int n = 0; n < N; ++n) o[n] = f32x4{0, 0, 0, 0};
    if constexpr (SHAPED) {
      shape.start(p, t, head, row_scale);
      row_scale = shape.unit;
    }
  }

  // k: the lane's words of key 16 h + c in [h]; key_scale: of keys 16 h + 4 g + i, and so s[4 h + i], scores but for row_scale
  __device__ __forceinline__ void score(const unsigned (&k)[2][KEY_WORDS], const f32x4 (&key_scale)[2], float (&s)[8]) const {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 acc = {0, 0, 0, 0};
      constexpr int EACH = RUN / 8;  // products of a lane's run
#pragma unroll
      for (int b = 0; b < KS; b += EACH) {
        f16x8 part[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
          if constexpr (TYPE == TFCC_ROCM_S4) part[i] = word_int4(k[h][b + i]);
          else part[i] = eight_int8(k[h][2 * (b + i)], k[h][2 * (b + i) + 1]);
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(part[i], q_lo[b + i], acc, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < EACH; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(part[i], q_hi[b + i], acc, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * h + i] = acc[i] * key_scale[h][i];
    }
  }

  // SHAPED: the scores as they are meant, of keys kb + 16 h + 4 g + i
  __device__ __forceinline__ void form(int kb, unsigned g, float (&s)[8]) const {
    if constexpr (SHAPED) shape.apply(s, kb + 4 * (int)g, [](int i) { return 16 * (i / 4) + i % 4; });
  }

  // `missing`: a bit for each of the lane's eight keys that no page holds
  __device__ __forceinline__ static void hide(const Tile& t, int kb, unsigned g, unsigned missing, float (&s)[8], f32x4 (&value_scale)[2]) {
    if (__any(missing != 0) || kb < t.all_low || kb + 32 > t.all_high) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = kb + 16 * (i / 4) + 4 * (int)g + i % 4;
        const bool seen = (missing >> i & 1) == 0 && key >= t.row_low && key < t.row_high;
        s[i] = seen ? s[i] : -INFINITY;
        value_scale[i / 4][i % 4] = seen ? value_scale[i / 4][i % 4] : 0.0f;
      }
    }
  }

  // v: words from value N c of key 16 h + 4 g + i in [4 h + i]
  __device__ __forceinline__ void add(float (&s)[8], const f32x4 (&value_scale)[2], const unsigned (&v)[8][VALUE_WORDS]) {
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fmaf(s[i], row_scale, frame_log(value_scale[i / 4][i % 4])));
    top = across_groups_max(top);
    if (__any(top - frame > 15.0f)) {
      const float next = top - frame > 15.0f ? top - 8.0f : frame, h = next == frame ? 1.0f : half_step(frame, next), f = h * h;
      frame = next;
      l = l * h * h;
#pragma unroll
      for (int i = 0; i < N; ++i) o[i] *= f;
    }
    const float zero = frame == -INFINITY ? 0.0f : frame;
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = __builtin_amdgcn_exp2f(fmaf(s[i], row_scale, -zero));
      l += e;
      w[i] = e * value_scale[i / 4][i % 4];
    }
    Half8 w_hi, w_lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) split_two(w[2 * i], w[2 * i + 1], w_hi.p[i], w_lo.p[i]);
#pragma unroll
    for (int b = 0; b < VALUE_WORDS; ++b) {
      unsigned word[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) word[i] = v[i][b];
#pragma unroll
      for (int half = 0; half < N / VALUE_WORDS / 4; ++half) {
        const int at = N / VALUE_WORDS * b + 4 * half;
        f16x8 part[4];
        if constexpr (TYPE == TFCC_ROCM_S4) {
          if (half == 0) four_of_int4<0>(word, part);
          else four_of_int4<1>(word, part);
        } else {
          part[0] = eight_of<0>(word);
          part[1] = eight_of<1>(word);
          part[2] = eight_of<2>(word);
          part[3] = eight_of<3>(word);
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) o[at + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(part[n], w_lo.v, o[at + n], 0, 0, 0);
#pragma unroll
        for (int n = 0; n < 4; ++n) o[at + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(part[n], w_hi.v, o[at + n], 0, 0, 0);
      }
    }
  }

  template <int WAVES>
  __device__ __forceinline__ void finish(Joining<64 * BLOCKS, WAVES>& joining, const AttentionArgs& p, const Tile& t, unsigned head, unsigned split, unsigned g) {
    l = across_groups_sum(l);
    float list[4 * N];  // neighbours in the list are neighbours in the head
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int n = 0; n < N; ++n) list[i * N + n] = o[n][i];
    join_and_store(joining, p, t, head, split, frame_out(frame, l), l, list, [&](int at) { return N * (4 * (int)g + at / N) + at % N; });
  }
};

// Integers with pages of 16 rows and more that can be read 16 bytes at a time.  A wavefront takes 32 keys in a step, two halves
// of 16; WITHIN: pages of a multiple of 16 rows, so that a half lies in one, or of 32 for a whole step (4 bits), else (0) a half in up to two, and so where
// rows are no multiples of 16 bytes (-1, 4 bits), which come four bytes to a lane.  8 bits, 32 sequences of up to 4096, 186 MB: 46 us, 4.1 TB/s, pages of 24 rows 49.
// Bound: HBM, which wants more on its way than registers can take: a wavefront copies the rows of its next steps straight into LDS, a ring of kStages of its own
// (no barriers), and reads a step from there when it is due.  4 bits: by the vector unit besides, which is active 42 to 45 % of the time, the matrix cores 16 % (64 sequences of 1024 to 4096,
// 8 heads of 128, 197 MB: 48 to 51 us, 3.9 to 4.1 TB/s; 32 of 16384, 571 MB: 117 to 130 us, 4.4 to 4.9 TB/s).
template <int TYPE, int BLOCKS, int WAVES, bool NARROW>
struct ScaledRing {
  static constexpr int kRow = ScaledLayout<TYPE, BLOCKS>::BYTES, kHalf = 16 * kRow, kRows = 4 * kHalf, kBytes = kRows + 256;  // keys and values, scales
  static constexpr int kStages = TYPE == TFCC_ROCM_S4 || kRow >= 128 ? 2 : 4;
  static constexpr int kCopies = (NARROW ? kRow / 4 : kRow < 64 ? 2 : 4 * (kRow / 64)) + 1;
  union {
    alignas(16) unsigned char ring[WAVES][kStages][kBytes];
    Joining<64 * BLOCKS, WAVES> joining;
  };
};
template <int TYPE, int BLOCKS, int WAVES, int WITHIN, bool SHAPED>
__global__ __launch_bounds__(WAVES * 64, TYPE == TFCC_ROCM_S4 ? (BLOCKS == 1 ? 4 : BLOCKS == 2 ? 3 : 2) : 1) void attention_scaled_kernel(AttentionArgs p) {
  constexpr bool WHOLE = WITHIN > 0;
  constexpr bool NARROW = WITHIN < 0;
  typedef ScaledRing<TYPE, BLOCKS, WAVES, NARROW> Ring;
  typedef ScaledLayout<TYPE, BLOCKS> Layout;
  constexpr int STEP = 32 * WAVES, CHUNKS = Layout::BYTES / 16 /* of 16 bytes in a row */;
  // Rows of 32 bytes: one copy brings both halves' keys, or values.
  constexpr bool BOTH = CHUNKS == 2;
  constexpr int LINES = BOTH ? 1 : CHUNKS / 4 /* copies of a half */, PER_COPY = 16 / LINES /* rows of it */, FOURS = PER_COPY / 4;
  __shared__ Ring shared;
  Tile t;
  unsigned head, split;
  int begin, end;
  if (!take_work<SHAPED>(p, kAttentionRows, threadIdx.x % 16, t, head, split, begin, end)) return;
  const unsigned lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  const unsigned wave = (unsigned)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64));
  const unsigned size = p.cache.size / Layout::PER /* of a row, in bytes */, row_bytes = (unsigned)p.cache.row;
  const int8_t* const keys = static_cast<const int8_t*>(p.cache.keys) + head * p.cache.head;
  const int8_t* const values = static_cast<const int8_t*>(p.cache.values) + head * p.cache.head;
  const float* const scales = (lane < 32 ? p.cache.key_scales : p.cache.value_scales) + head * p.cache.scale_head + c;
  const int* const table = p.table + (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)t.sequence) * p.table_stride;
  int kb = __builtin_amdgcn_readfirstlane(begin + 32 * (int)wave);
  end = __builtin_amdgcn_readfirstlane(end);

  const auto exchange = [](unsigned row) { return BOTH ? row / 8 : CHUNKS == 4 ? row / 4 % 4 : row % CHUNKS; };
  // A copy brings PER_COPY whole rows, CHUNKS lanes to a row: lanes side by side ask for memory side by side (with a lane for each row the copies
  // take four times as long).  A lane puts its 16 bytes at its own place in LDS; which of the row's chunks that is, and which row, is free
  // and chosen so that what is read together lies in different banks.  Keys are read 16 rows at a time, a chunk of each: chunks are
  // exchanged within a row by its number.  Values are read a few bytes of rows 4 g + i at a time: those rows lie side by side.
  unsigned key_at[LINES], value_at[LINES];
  const unsigned slot = lane / CHUNKS % 16, chunk = lane % CHUNKS;
  const auto key_row = [&](int b) { return b * PER_COPY + slot; };
  const auto value_row = [&](int b) { return (b * FOURS + slot % FOURS) * 4 + slot / FOURS; };
#pragma unroll
  for (int b = 0; b < LINES; ++b) {
    const unsigned from = (chunk ^ exchange(key_row(b))) * 16;
    key_at[b] = key_row(b) * row_bytes + (from < size ? from : 0);
    value_at[b] = value_row(b) * row_bytes + (chunk * 16 < size ? chunk * 16 : 0);
  }
  if (BOTH && WITHIN == 32 && lane >= 32) {
    key_at[0] += 16 * row_bytes;
    value_at[0] += 16 * row_bytes;
  }
  const unsigned half_bytes = (WITHIN == 32 ? 31 : 15) * row_bytes + size;  // from a half's first row on, or a step's
  unsigned char* const ring = shared.ring[wave][0];
  const unsigned ring_at = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char*)ring;

  // of each half: the page of its first key and, where that may be another one, of its last
  constexpr int PAGES = WHOLE ? 1 : 2;
  PageEntry entries[2][PAGES] = {};
  const auto ask_pages = [&](int at) {
#pragma unroll
    for (int h = 0; h < (WITHIN == 32 ? 1 : 2); ++h)
#pragma unroll
      for (int n = 0; n < PAGES; ++n) entries[h][n] = entry_of(p, table, p.cache.page_size.quotient((unsigned)at + 16 * h + 15 * n));
  };
  const auto inside_page = [&](unsigned key) { return key - p.cache.page_size.quotient(key) * p.cache.page_size.d; };
  // the row of a half that the second page begins with
  const auto cut_of = [&](unsigned key) { return p.cache.page_size.d - inside_page(key); };
  const auto copy = [&](unsigned stage, int at, const int (&page)[2][PAGES]) {
    const unsigned to = (unsigned)__builtin_amdgcn_readfirstlane((int)(ring_at + stage * Ring::kBytes));
    if constexpr (NARROW) {
      // 4 bytes to a lane, which go where the above puts them: lane l of copy n has word l % WORDS of place n * ROWS + l / WORDS
      constexpr int WORDS = Ring::kRow / 4, ROWS = 64 / WORDS;
      const unsigned word = lane % WORDS;
      const float* scale_of[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned key = (unsigned)at + 16 * h, inside = inside_page(key), cut = cut_of(key);
        const unsigned long long first = page[h][0] < 0 ? 0 : (unsigned)page[h][0], next = page[h][PAGES - 1] < 0 ? 0 : (unsigned)page[h][PAGES - 1];
        const long long base = (long long)(first * p.cache.page + inside * p.cache.row), other = (long long)(next * p.cache.page) - cut * (long long)p.cache.row;
        scale_of[h] = c >= cut ? scales + next * p.cache.scale_page - cut : scales + first * p.cache.scale_page + inside;
#pragma unroll 1  // (unrolled, their addresses take registers that a step does not have)
        for (int n = 0; n < 16 / ROWS; ++n) {
          const unsigned row = n * ROWS + lane / WORDS, from = ((word / 4 ^ exchange(row)) * 4 + word % 4) * 4;
          dma4_global(keys + (row >= cut ? other : base) + (row * row_bytes + (from < size ? from : 0)), to + h * Ring::kHalf + n * 256);
        }
#pragma unroll 1
        for (int n = 0; n < 16 / ROWS; ++n) {
          const unsigned place = n * ROWS + lane / WORDS, row = (place / PER_COPY * FOURS + place % PER_COPY % FOURS) * 4 + place % PER_COPY / FOURS, from = word * 4;
          dma4_global(values + (row >= cut ? other : base) + (row * row_bytes + (from < size ? from : 0)), to + (2 + h) * Ring::kHalf + n * 256);
        }
      }
      dma4_global((lane & 16) ? scale_of[1] : scale_of[0], to + Ring::kRows);
      return;
    }
    if constexpr (WITHIN == 32) {
      const unsigned inside = inside_page((unsigned)at);
      const unsigned long long held = page[0][0] < 0 ? 0 : (unsigned)page[0][0], base = held * p.cache.page + inside * p.cache.row;
      const lds_dma_v4i k = make_rsrc(keys + base, half_bytes), v = make_rsrc(values + base, half_bytes);
#pragma unroll
      for (int h = 0; h < (BOTH ? 1 : 2); ++h)
#pragma unroll
        for (int b = 0; b < LINES; ++b) {
          if (h == 0) dma16(k, to + b * 1024, key_at[b]);
          else dma16s(k, to + (LINES + b) * 1024, key_at[b], 16 * row_bytes);
        }
#pragma unroll
      for (int h = 0; h < (BOTH ? 1 : 2); ++h)
#pragma unroll
        for (int b = 0; b < LINES; ++b) {
          if (h == 0) dma16(v, to + 2 * Ring::kHalf + b * 1024, value_at[b]);
          else dma16s(v, to + 2 * Ring::kHalf + (LINES + b) * 1024, value_at[b], 16 * row_bytes);
        }
      const float* const scale = scales + held * p.cache.scale_page + inside + (lane & 16);
      dma4_global(scale, to + Ring::kRows);
      return;
    }
    const float* scale_at[2];
    unsigned long long row_at[2];  // BOTH: of the lane's row of keys, and of values, in the first half and in the second
    unsigned long long value_row_at[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned key = (unsigned)at + 16 * h, inside = inside_page(key);
      const unsigned long long held = page[h][0] < 0 ? 0 : (unsigned)page[h][0], base = held * p.cache.page + inside * p.cache.row;
      scale_at[h] = scales + held * p.cache.scale_page + inside;
      if constexpr (BOTH && WHOLE) {
        row_at[h] = value_row_at[h] = base;
      } else if constexpr (WHOLE) {
        const lds_dma_v4i k = make_rsrc(keys + base, half_bytes), v = make_rsrc(values + base, half_bytes);
#pragma unroll
        for (int b = 0; b < LINES; ++b) dma16(k, to + (h * LINES + b) * 1024, key_at[b]);
#pragma unroll
        for (int b = 0; b < LINES; ++b) dma16(v, to + ((2 + h) * LINES + b) * 1024, value_at[b]);
      } else {
        const unsigned long long next = page[h][PAGES - 1] < 0 ? 0 : (unsigned)page[h][PAGES - 1];
        const long long cut = cut_of(key), other = (long long)(next * p.cache.page) - cut * (long long)p.cache.row;
        if (c >= cut) scale_at[h] = scales + next * p.cache.scale_page - cut;
        row_at[h] = key_row(0) >= cut ? other : (long long)base;
        value_row_at[h] = value_row(0) >= cut ? other : (long long)base;
        if constexpr (BOTH) continue;
#pragma unroll
        for (int b = 0; b < LINES; ++b) dma16_global(keys + (key_row(b) >= cut ? other : (long long)base) + key_at[b], to + (h * LINES + b) * 1024);
#pragma unroll
        for (int b = 0; b < LINES; ++b) dma16_global(values + (value_row(b) >= cut ? other : (long long)base) + value_at[b], to + ((2 + h) * LINES + b) * 1024);
      }
    }
    if constexpr (BOTH) {
      dma16_global(keys + (lane < 32 ? row_at[0] : row_at[1]) + key_at[0], to);
      dma16_global(values + (lane < 32 ? value_row_at[0] : value_row_at[1]) + value_at[0], to + 2 * Ring::kHalf);
    }
    const float* const scale = (lane & 16) ? scale_at[1] : scale_at[0];
    dma4_global(scale, to + Ring::kRows);
  };
  unsigned gone = 0;  // four bits a stage: of each half, what would be on its first and on its last page is nowhere
  if (kb < end) ask_pages(kb);
  int ahead = kb;  // the first step that no copy is under way for
  const auto send = [&](unsigned stage) {
    if (ahead < end) {
      int pages[2][PAGES];
      unsigned none = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          if (n < PAGES) pages[h][n] = WITHIN == 32 && h > 0 ? pages[0][n] : page_of(p, entries[h][n]);
          none |= pages[h][n < PAGES ? n : 0] < 0 ? 1u << (2 * h + n) : 0u;
        }
      copy(stage, ahead, pages);
      gone = (gone & ~(15u << (4 * stage))) | none << (4 * stage);
      ahead += STEP;
      if (ahead < end) ask_pages(ahead);
    }
  };
  // Loads come back in their order: queries behind the copies wait for all stages to be filled, before them the copies wait for the queries.  4 bits, whose stages
  // take longer to work on than to fill: the queries first (64 sequences of up to 4096: 49.3 us, behind the copies 49.8); 8 bits: behind (32 of up to 4096: 46.2 us, before
  // them 46.7, 32 of up to 2000 25.6 and 26.6).
  constexpr bool QUERIES_FIRST = TYPE == TFCC_ROCM_S4;
  ScaledRows<TYPE, BLOCKS, SHAPED> rows;
  if constexpr (QUERIES_FIRST) rows.start(p, t, head, g);
#pragma unroll 1
  for (unsigned stage = 0; stage < Ring::kStages; ++stage) send(stage);
  if constexpr (!QUERIES_FIRST) rows.start(p, t, head, g);

  unsigned stage = 0;
#pragma unroll 1
  for (; kb < end; kb += STEP) {
    // the copies of the stages behind this one may still be under way
    if (kb + (Ring::kStages - 1) * STEP < end) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((Ring::kStages - 1) * Ring::kCopies) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    const unsigned char* const from = ring + stage * Ring::kBytes;
    unsigned k[2][Layout::KEY_WORDS], v[8][Layout::VALUE_WORDS];
    f32x4 key_scale[2], value_scale[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned char* const row = from + h * Ring::kHalf + c * Ring::kRow;
      if constexpr (BOTH) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(row + (g ^ 2 * exchange(c)) * 8);
        k[h][0] = w[0];
        k[h][1] = w[1];
      } else {
#pragma unroll
        for (int b = 0; b < LINES; ++b) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(row + ((4 * b + g) ^ exchange(c)) * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) k[h][4 * b + i] = w[i];
        }
      }
      key_scale[h] = *reinterpret_cast<const f32x4*>(from + Ring::kRows + (16 * h + 4 * g) * 4);
      value_scale[h] = *reinterpret_cast<const f32x4*>(from + Ring::kRows + 128 + (16 * h + 4 * g) * 4);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const unsigned char* const at = from + (2 + i / 4) * Ring::kHalf + (g / FOURS) * 1024 + ((i % 4) * FOURS + g % FOURS) * Ring::kRow + Ring::kRow / 16 * c;
      if constexpr (BOTH) {
        v[i][0] = *reinterpret_cast<const unsigned short*>(at);
      } else if constexpr (LINES == 1) {
        v[i][0] = *reinterpret_cast<const unsigned*>(at);
      } else if constexpr (LINES == 2) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(at);
        v[i][0] = w[0];
        v[i][1] = w[1];
      } else {
        const u32x4 w = *reinterpret_cast<const u32x4*>(at);
#pragma unroll
        for (int b = 0; b < 4; ++b) v[i][b] = w[b];
      }
    }
    const unsigned none = gone >> (4 * stage) & 15;
    unsigned missing = (none & 1 ? 15u : 0u) | (none & 4 ? 240u : 0u);
    if (!WHOLE && none != 0) {
      missing = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const unsigned h = i / 4, behind = 4 * g + i % 4 >= cut_of((unsigned)kb + 16 * h) ? 1 : 0;
        missing |= (none >> (2 * h + behind) & 1) << i;
      }
    }
    // Read: the stage may be written again.  (By the builtin, which the compiler counts with: it would else wait for the reads once more, and
    // with them for the page entries that send() has asked for.)
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    send(stage);
    stage = stage + 1 == Ring::kStages ? 0 : stage + 1;
    float s[8];
    rows.score(k, key_scale, s);
    rows.form(kb, g, s);
    rows.hide(t, kb, g, missing, s, value_scale);
    rows.add(s, value_scale, v);
  }
  __syncthreads();  // the ring is done with
  rows.template finish<WAVES>(shared.joining, p, t, head, split, g);
}

// Chunks of many tokens, int8 as above: a workgroup takes 128 rows, a wavefront 32 of them, and all go over the same keys, 32 in a step.  Bound: the waits of steps whose wavefronts
// take turns with matrix cores and vector unit; neither is full (4 chunks of 1024 over 4096, 32 heads over 8 of 128: int8 377 us, matrix operations and LDS
// reads alone 283; 4 bits 380; matrix cores active 34 to 35 % of the time, the vector unit 37 to 41 %, 1.5 wavefronts to a SIMD where two fit, of whose cycles 30 to 39 % are waits; with a cap 57 % of the
// vector unit; float32 589, with tiles of 16 rows on the fp32 matrix operations 1930).  So the keys and values of a step are turned into fp16 once for all wavefronts, in the
// order in which the matrix cores take them, into one of two LDS buffers while the other is worked on; the next step's rows
// are on their way to registers meanwhile.  Products of 32 x 32 as above, with
//   S^T: lane l holds row l % 32 and keys 8 a + 4 (l / 32) + i in [4 a + i]
//   O^T: likewise values place(8 a + 4 (l / 32) + i, n) of the head in tile n
constexpr int kTileKeys = 32;

// Which value of a head is row L of tile n of the second product: a word of four values goes to four tiles, or to two rows of two where
// 64 values are left; float32: two neighbours go to two tiles.
template <int BLOCKS, bool SCALED>
__device__ __forceinline__ constexpr unsigned value_of(unsigned L, unsigned n) {
  if (!SCALED) return n / 2 * 64 + 2 * L + n % 2;
  return n / 4 * 4 + 4 <= 2 * BLOCKS ? n / 4 * 128 + 4 * L + n % 4 : n / 4 * 128 + 4 * (L % 16) + 2 * (L / 16) + n % 4;
}

// A row of a float32 cache is two fp16 pieces under a power of two of its own, which is its scale as an int8 row's is: what is said above of
// int8 holds, with a third operation for the product of the first factor's large piece with the second's small one.  The two
// small ones' product, 2^-22 of the whole at most and 2^-25 in the mean, is left out: with the pieces' own 2^-23 each a term is right to 2^-21, where the
// fp32 operations, at five times their cost, round to 2^-24 (6 chunks of 517 with a window: 4.3 to 4.9e-7 from 64 bits, elementary float32 operations 4.3 to 4.4e-7).  Infinities and NaN have no such pieces: where a row sees one, the workgroup takes its rows
// once more by the fp32 operations (an infinity in the first page of every sequence: 4 chunks of 1024 over 4096 2530 us, with tiles of 16 rows 2060).  Weights and scores have float32's exponents to stay in, so numbers from 2^80 on go that way too, and what undoes a value row's power of
// two is taken 2^kLift times, which the results are freed of: these scales lie between 2^-78 and 2^102.  A weight that brings the largest scale to
// the frame's 2^8 is 2^-94, those 2^-30 below it are normal numbers, and one that brings the smallest to 2^15 is 2^93, of which 2^34 can be summed.
constexpr unsigned kFar = 0x67800000u;  // 2^80
constexpr int kLift = 36;

// Rows of a tile, 16 of them, over a float32 cache: the keys of steps kb, kb + STEP, ... below end, 16 in each.  The next step's keys are loaded into the registers
// of this one's as soon as the scores are formed, its values once the weights have met them.  PAGES that the keys of a step may lie in: 1 (of a
// multiple of 16 rows), 2 (16 rows at least) or any number, 0.  `missing`: a bit for each of the lane's four keys that no page holds.
// look: sees each step's rows as they were loaded; done: takes value 64 b + 4 (4 g + i) + j of the row in o[b][j][i], its frame and the lane's share of its sum.
// (Handed out through references, they cost heads of more than 128 values 5 to 8 %.)
template <int BLOCKS, int STEP, int PAGES, bool SHAPED, class Look, class Done>
__device__ __forceinline__ void stream_rows(const AttentionArgs& p, const Tile& t, unsigned head, int kb, int end, const int* table, Look look, Done done) {
  constexpr int DPAD = 64 * BLOCKS;
  const unsigned lane = threadIdx.x & 63, g = lane / 16, c = lane % 16;
  const unsigned size = p.cache.size;
  const float* const keys = static_cast<const float*>(p.cache.keys) + head * p.cache.head;
  const float* const values = static_cast<const float*>(p.cache.values) + head * p.cache.head;

  kb = __builtin_amdgcn_readfirstlane(kb);
  end = __builtin_amdgcn_readfirstlane(end);
  f32x4 k[4 * BLOCKS], v[4][BLOCKS];
  unsigned missing = 0;
  const auto inside_page = [&](unsigned key) { return key - p.cache.page_size.quotient(key) * p.cache.page_size.d; };
  const auto locate = [&](int key, unsigned long long& row) {
    const int page = page_of(p, table, p.cache.page_size.quotient((unsigned)key));
    row = page < 0 ? 0 : page * p.cache.page + inside_page((unsigned)key) * p.cache.row;
    return page >= 0;
  };
  PageEntry entries[PAGES == 2 ? 2 : 1] = {};
  const auto ask_pages = [&](int at) {
#pragma unroll
    for (int n = 0; n < PAGES; ++n) entries[n] = entry_of(p, table, p.cache.page_size.quotient((unsigned)at + 15 * n));
  };
  struct Held {
    int page[2];
  };
  const auto pages_of = [&] {
    Held held = {};
#pragma unroll
    for (int n = 0; n < PAGES; ++n) held.page[n] = page_of(p, entries[n]);
    return held;
  };
  // where row r of the step at `at` lies, and whether it is anywhere
  const auto place = [&](int at, unsigned r, const Held& held, unsigned long long& row) {
    if constexpr (PAGES == 0) return locate(at + (int)r, row);
    const unsigned inside = inside_page((unsigned)at), cut = p.cache.page_size.d - inside;
    const bool behind = PAGES == 2 && r >= cut;
    const int page = behind ? held.page[1] : held.page[0];
    row = (page < 0 ? 0ull : (unsigned)page) * p.cache.page + (behind ? r - cut : inside + r) * p.cache.row;
    return page >= 0;
  };
  const auto load_keys = [&](int at, const Held& held) {
    unsigned long long row;
    place(at, c, held, row);
#pragma unroll
    for (int b = 0; b < 4 * BLOCKS; ++b) k[b] = *reinterpret_cast<const f32x4*>(keys + row + (16 * b + 4 * g < size ? 16 * b + 4 * g : 0));
  };
  const auto load_values = [&](int at, const Held& held) {
    missing = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      unsigned long long row;
      missing |= place(at, 4 * g + i, held, row) ? 0u : 1u << i;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) v[i][b] = *reinterpret_cast<const f32x4*>(values + row + (64 * b + 4 * c < size ? 64 * b + 4 * c : 0));
    }
  };
  if (kb < end) {
    ask_pages(kb);
    const Held held = pages_of();
    load_keys(kb, held);
    load_values(kb, held);
    if (kb + STEP < end) ask_pages(kb + STEP);
  }
  // value 16 b + 4 g + j of the row's query in q[b][j]
  f32x4 q[4 * BLOCKS];
  {
    const float* x = p.q + (unsigned long long)(t.first + (t.row_token < 0 ? 0 : t.row_token)) * p.q_token + (head * p.group.d + t.row_head) * p.q_head;
#pragma unroll
    for (int b = 0; b < 4 * BLOCKS; ++b) {
      const unsigned d = 16 * b + 4 * g;
      f32x4 v = {0, 0, 0, 0};
      if (t.row_token >= 0 && d < size) v = *reinterpret_cast<const f32x4*>(x + d) * p.scale;
      q[b] = v;
    }
  }
  f32x4 o[BLOCKS][4];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[b][j] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;
  ScoreShape shape;
  if constexpr (SHAPED) shape.start(p, t, head, 1.0f);

  if constexpr (BLOCKS == 1) {
    for (; kb < end; kb += STEP) {
#define STEP_FOLLOWS kb + STEP < end
#include "paged_attention_step.hpp"
    }
  } else {
    // The last step, which asks for nothing, apart from the others: as one of them, the loads of the next keys and of their values would each be under a condition, and a way with one and without the
    // other, which the compiler has to count with, makes the first wait for a key one for all values on their way as well (random calls, geometric means of the time apart over that in one loop: heads of 193 to
    // 256 0.95, of 129 to 192 0.97 to 1.00, of 65 to 128 0.98, over fewer than 256 keys 1.006; of up to 64, whose loads are few, 1.01, which stay with one).
#pragma unroll 1
    for (; kb + STEP < end; kb += STEP) {
#define STEP_FOLLOWS true
#include "paged_attention_step.hpp"
    }
    if (kb < end) {
#define STEP_FOLLOWS false
#include "paged_attention_step.hpp"
    }
  }
  done(o, m, l);
}

// The wavefront's 32 rows of a tile over a float32 cache by the fp32 matrix operations, 16 at a time.  Only rows that see a number of kFar or above are
// written: the others keep what they have, whatever lies beside them.
template <int BLOCKS, bool SHAPED>
__device__ __forceinline__ void stream_far_rows(const AttentionArgs& p, const Tile& t, unsigned head, unsigned split, int begin, int end, const int* table) {
  const unsigned lane = threadIdx.x & 63, g = lane / 16, size = p.cache.size;
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {
    Tile u = t;
    const int row = 16 * half + (int)(lane % 16);
    u.row_token = __shfl(t.row_token, row, 64);
    u.row_head = __shfl(t.row_head, row, 64);
    u.row_low = __shfl(t.row_low, row, 64);
    u.row_high = __shfl(t.row_high, row, 64);
    u.row_position = __shfl(t.row_position, row, 64);
    const u64 there = __ballot(u.row_token >= 0) & 0xffff;  // the first ones
    if (there == 0) return;
    // what these rows see of the piece, from one of its steps on
    const int low = __builtin_amdgcn_readfirstlane(u.row_low), high = __builtin_amdgcn_readlane(u.row_high, 63 - __builtin_clzll(there));
    const int from = low > begin ? begin + (low - begin) / 16 * 16 : begin, upto = high < end ? high : end;
    bool far = false;
    const auto look = [&](int kb, const f32x4 (&k)[4 * BLOCKS], const f32x4 (&v)[4][BLOCKS], unsigned missing) {
      const auto size_of = [](const f32x4& x) {
        unsigned most = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const unsigned bits = __float_as_uint(x[j]) & 0x7fffffffu;
          most = bits > most ? bits : most;
        }
        return most;
      };
      // a bit for each key of the step: lanes c, c + 16, ... have key c, the 16 of group g value rows 4 g + i
      unsigned most = 0;
#pragma unroll
      for (int b = 0; b < 4 * BLOCKS; ++b) most = size_of(k[b]) > most ? size_of(k[b]) : most;
      const u64 key_lanes = __ballot(most >= kFar);
      unsigned keys = (unsigned)(key_lanes | key_lanes >> 16 | key_lanes >> 32 | key_lanes >> 48) & 0xffffu;
      unsigned none = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        most = 0;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) most = size_of(v[i][b]) > most ? size_of(v[i][b]) : most;
        const u64 value_lanes = __ballot(most >= kFar), none_lanes = __ballot((missing >> i & 1) != 0);
#pragma unroll
        for (int group = 0; group < 4; ++group) {
          keys |= (value_lanes >> (16 * group) & 0xffff) != 0 ? 1u << (4 * group + i) : 0u;
          none |= (unsigned)(none_lanes >> (16 * group) & 1) << (4 * group + i);
        }
      }
      const int first = u.row_low > kb ? u.row_low - kb : 0, behind = u.row_high - kb < 16 ? u.row_high - kb : 16;
      if (first < behind) far |= (keys & ~none & ((1u << behind) - 1) >> first << first) != 0;
    };
    const auto write = [&](const f32x4 (&o)[BLOCKS][4], float m, float l) {
      l = across_groups_sum(l);
      m = frame_out(m, l);
      if (u.row_token < 0 || !far) return;
      const unsigned long long token = u.first + u.row_token, query_head = head * p.group.d + u.row_head;
      float* to = p.out + token * p.out_token + query_head * p.out_head;
      const f32x4 zeros = {0, 0, 0, 0};
      float divisor = l;
      if (p.splits > 1) {
        const unsigned long long place = ((unsigned long long)split * p.tokens + token) * p.cache.heads * p.group.d + query_head;
        to = p.partial + place * size;
        divisor = 1.0f;
        if (g == 0) {
          p.statistics[place * 2] = m;
          p.statistics[place * 2 + 1] = l;
        }
      }
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned d = 64 * b + 4 * (4 * g + i);
          if (d < size) *reinterpret_cast<f32x4*>(to + d) = m == -INFINITY ? zeros : f32x4{o[b][0][i], o[b][1][i], o[b][2][i], o[b][3][i]} / divisor;
        }
    };
    stream_rows<BLOCKS, 16, 2, SHAPED>(p, u, head, from, upto, table, look, write);
  }
}

// The same as a function of its own that finds the work once more: what it wants takes no registers from the kernel's steps (4 chunks of 1024 over 4096, 32 heads
// over 8 of 128: 667 us, and 679 with the above in the kernel; 12 heads of 64: 30 chunks of up to 500 over up to 800 115 and 119, with biases and prefixes 129 and 134).
template <int BLOCKS, int WAVES, bool SHAPED>
__device__ __attribute__((noinline)) void stream_far_rows_apart(const AttentionArgs& p) {
  Tile t;
  unsigned head, split;
  int begin, end;
  if (!take_work<SHAPED>(p, WAVES * 32, threadIdx.x / 64 * 32 + threadIdx.x % 32, t, head, split, begin, end)) return;
  stream_far_rows<BLOCKS, SHAPED>(p, t, head, split, begin, end, p.table + (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)t.sequence) * p.table_stride);
}

// WAVES: 4, and 8 where a thread's part of a step's rows would else take the registers (float32, heads of 128: four wavefronts spill).
template <int TYPE, int BLOCKS, int WAVES, bool WHOLE, bool SHAPED>
__global__ __launch_bounds__(WAVES * 64, WAVES == 4 && BLOCKS > 2 ? 1 : 2) void attention_tile_kernel(AttentionArgs p) {
  constexpr bool S8 = TYPE != TFCC_ROCM_F32 /* integers with scales */, S4 = TYPE == TFCC_ROCM_S4;
  static_assert(!S4 || BLOCKS == 2);
  constexpr int KS = 4 * BLOCKS, N = 2 * BLOCKS, PIECES = S8 ? 1 : 2;  // products over a head, tiles of 32 of its values
  static_assert(S8 ? WAVES == 4 : BLOCKS * 4 == WAVES);
  struct Stage {
    u32x4 keys[PIECES][KS][64];       // lane l: key l % 32, values 16 s + 8 (l / 32) + j; float32: exchange() within the half
    u32x4 values[PIECES][N][2][64];   // lane l: value_of(l % 32, n), keys 16 m + 8 (j / 4) + 4 (l / 32) + j % 4
    float key_scale[kTileKeys], value_scale[kTileKeys], value_log[kTileKeys];
    unsigned gone[WAVES / 2];         // keys that no page holds: a bit for each; what each of the first wavefronts knows of it
  };
  __shared__ Stage stages[2];
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x / 64, half = lane / 32;
  Tile t;
  unsigned head, split;
  int begin, end;
  if (!take_work<SHAPED>(p, WAVES * 32, wave * 32 + lane % 32, t, head, split, begin, end)) return;
  const unsigned size = p.cache.size;
  using Element = std::conditional_t<S8, int8_t, float>;
  const Element* const keys = static_cast<const Element*>(p.cache.keys) + head * p.cache.head;
  const Element* const values = static_cast<const Element*>(p.cache.values) + head * p.cache.head;
  const int* const table = p.table + (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)t.sequence) * p.table_stride;
  begin = __builtin_amdgcn_readfirstlane(begin);
  end = __builtin_amdgcn_readfirstlane(end);
  // what this wavefront's rows see; rows that are there come first
  const int there = __builtin_popcountll(__ballot(t.row_token >= 0) & 0xffffffffull), last = there > 0 ? there - 1 : 0;
  const int low = __builtin_amdgcn_readfirstlane(t.row_low), high = there > 0 ? __builtin_amdgcn_readlane(t.row_high, last) : 0;
  const int all_low = __builtin_amdgcn_readlane(t.row_low, last), all_high = __builtin_amdgcn_readfirstlane(t.row_high);

  // A step's rows: threads of the first half fetch keys, 16 bytes of key (thread % 32) at a time, float32: SIDE threads side by side those of one
  // key; those of the second values, four values of eight keys at a time, float32: two; the first wavefront the scales.
  constexpr int HALF = WAVES * 32, SIDE = HALF / kTileKeys, WORDS = S4 ? 8 * BLOCKS : S8 ? 16 * BLOCKS : 32 * BLOCKS, TASKS = (4 * WORDS + HALF - 1) / HALF;
  static_assert(S8 || (TASKS == 1 && 4 * WORDS == HALF));
  constexpr int CHUNKS = S4 ? 1 : S8 ? BLOCKS : 4;  // of 16 bytes of a key to a thread
  const unsigned row_bytes = S4 ? size / 2 : size;                 // S8 and S4
  const bool for_keys = threadIdx.x < HALF;
  const unsigned me = threadIdx.x % HALF;
  u32x4 raw[S4 ? 2 * TASKS : S8 && BLOCKS <= 2 ? 2 : 4];  // 16 bytes of a key each, or TASKS times eight words, float32: two keys' values in each
  // Each thread asks for the pages of its own rows, through the vector loads: they come back in order, after the rows that were asked for before.
  // (Entries through the scalar cache would be waited for with the LDS reads.)
  float scale = 0.0f;
  bool gone = false;
  // WHOLE: pages of a multiple of 16 rows, else of 4, 16 at least: the eight keys of a task then lie four and four
  constexpr int PAGES = WHOLE ? 1 : 2;
  int named[TASKS][PAGES];
  // the first key of the step's that the thread's task k fetches of its n-th page
  const auto key_of = [&](int k, int n) {
    const unsigned group = (me + HALF * k) / WORDS;
    return for_keys ? (!S8 ? me / SIDE : WHOLE ? me / 16 % 2 * 16 : me % 32) : group / 2 % 2 * 16 + (WHOLE ? 0 : 4 * (group % 2) + 8 * n);
  };
  const auto inside_page = [&](unsigned key) { return key - p.cache.page_size.quotient(key) * p.cache.page_size.d; };
  const auto ask_pages = [&](int at) {
#pragma unroll
    for (int k = 0; k < TASKS; ++k)
#pragma unroll
      for (int n = 0; n < PAGES; ++n) {
        const unsigned index = p.cache.page_size.quotient((unsigned)at + key_of(k, n));
        named[k][n] = index < p.table_width ? table[index] : -1;
      }
  };
  const auto fetch = [&](int at) {
    const unsigned halves[2] = {inside_page((unsigned)at), inside_page((unsigned)at + 16)};
    const auto page_row = [&](int k, int n, unsigned long long& held) {
      const bool none = (unsigned)named[k][n] >= p.cache.pages;
      held = none ? 0 : (unsigned)named[k][n];
      return none;
    };
    unsigned long long held;
    if (for_keys) {
      gone = page_row(0, 0, held);
      const unsigned inside = WHOLE ? (me / 16 % 2 ? halves[1] : halves[0]) + (me & 15) : inside_page((unsigned)at + key_of(0, 0));
      const Element* const row = keys + held * p.cache.page + inside * p.cache.row;
#pragma unroll
      for (int b = 0; b < CHUNKS; ++b) {
        const unsigned d = S8 ? 16 * (me / 32 + 4 * b) : 4 * (me % SIDE + SIDE * b);
        if constexpr (S4) {  // rows of a multiple of 8 bytes
          const u32x2 first = *reinterpret_cast<const u32x2*>(row + (d < row_bytes ? d : 0)), second = *reinterpret_cast<const u32x2*>(row + (d + 8 < row_bytes ? d + 8 : 0));
          raw[b] = u32x4{first[0], first[1], second[0], second[1]};
        } else {
          raw[b] = *reinterpret_cast<const u32x4*>(row + (d < size ? d : 0));
        }
      }
      if (S8 && threadIdx.x < 64) {
        const float* const s = (threadIdx.x < 32 ? p.cache.key_scales : p.cache.value_scales) + head * p.cache.scale_head;
        scale = s[held * p.cache.scale_page + inside];
      }
    } else {
#pragma unroll
      for (int k = 0; k < TASKS; ++k) {
        const unsigned task = me + HALF * k, word = task % WORDS, group = task / WORDS;
        if (4 * WORDS % HALF == 0 || group < 4) {
          const Element* row[2];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            (void)page_row(k, n < PAGES ? n : 0, held);
            const unsigned inside = WHOLE ? (group / 2 ? halves[1] : halves[0]) + 4 * (group % 2) + 8 * n : inside_page((unsigned)at + key_of(k, n));
            const unsigned d = S8 ? 4 * word : 2 * word;
            row[n] = values + held * p.cache.page + inside * p.cache.row + (d < (S8 ? row_bytes : size) ? d : 0);
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if constexpr (S8) raw[2 * k + j / 4][j % 4] = *reinterpret_cast<const unsigned*>(row[j / 4] + j % 4 * p.cache.row);
            else {
              const u32x2 two = *reinterpret_cast<const u32x2*>(row[j / 4] + j % 4 * p.cache.row);
              raw[j / 2][j % 2 * 2] = two[0];
              raw[j / 2][j % 2 * 2 + 1] = two[1];
            }
          }
        }
      }
    }
  };
  const auto store_s8 = [&](Stage& s) {
    if (for_keys) {
#pragma unroll
      for (int b = 0; b < CHUNKS; ++b) {
        const unsigned chunk = me / 32 + 4 * b;
        if constexpr (S4) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s.keys[0][2 * chunk + i / 2][i % 2 * 32 + me % 32] = __builtin_bit_cast(u32x4, word_int4(raw[b][i]));
        } else {
          s.keys[0][chunk][me % 32] = __builtin_bit_cast(u32x4, eight_int8(raw[b][0], raw[b][1]));
          s.keys[0][chunk][32 + me % 32] = __builtin_bit_cast(u32x4, eight_int8(raw[b][2], raw[b][3]));
        }
      }
      if (threadIdx.x < 32) {
        s.key_scale[threadIdx.x] = scale;
        const unsigned nowhere = (unsigned)__ballot(gone);
        if (threadIdx.x < 2) s.gone[threadIdx.x] = nowhere;
      } else if (threadIdx.x < 64) {
        s.value_scale[threadIdx.x - 32] = scale;
        s.value_log[threadIdx.x - 32] = frame_log(scale);
      }
    } else {
#pragma unroll
      for (int k = 0; k < TASKS; ++k) {
        const unsigned task = me + HALF * k, word = task % WORDS, group = task / WORDS;
        if (4 * WORDS % HALF == 0 || group < 4) {
          unsigned w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) w[j] = raw[2 * k + j / 4][j % 4];
          constexpr int EACH = S4 ? 8 : 4;  // values in a word, which go where four and four do
#pragma unroll
          for (int f = 0; f < EACH / 4; ++f) {
            f16x8 v[4];
            if constexpr (S4) {
              if (f == 0) four_of_int4<0>(w, v);
              else four_of_int4<1>(w, v);
            } else {
              v[0] = eight_of<0>(w);
              v[1] = eight_of<1>(w);
              v[2] = eight_of<2>(w);
              v[3] = eight_of<3>(w);
            }
            const unsigned four = EACH / 4 * word + f;
            const bool quarters = (four / 32 + 1) * 4 <= N;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const unsigned n = four / 32 * 4 + (quarters ? b : b % 2), L = quarters ? four % 32 : four % 16 + 16 * (b / 2);
              s.values[0][n][group / 2][32 * (group % 2) + L] = __builtin_bit_cast(u32x4, v[b]);
            }
          }
        }
      }
    }
  };
  // float32: the power of two that brings a row's largest value to 2^13 .. 2^14, and the row's pieces.  What is read together and written together
  // of the keys lies in different banks.
  const auto exchange = [](unsigned lane_of, unsigned step) { return lane_of ^ (lane_of / 32 * 4) ^ (WAVES == 8 ? step % 2 * 2 : 0); };
  bool odd = false;  // a number of kFar or above was among what some row sees
  const auto store_f32 = [&](Stage& s, int at) {
    const auto larger = [](unsigned a, unsigned b) { return a > b ? a : b; };
    const auto size_of = [&](unsigned v) { return v & 0x7fffffffu; };
    if (at < t.low || at + kTileKeys > t.high) {  // what no row sees may be anything
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = at + (int)(for_keys ? me / SIDE : me / WORDS / 2 * 16 + 4 * (me / WORDS % 2) + 8 * (j / 4) + j % 4);
        const bool none = key < t.low || key >= t.high;
        raw[j / 2][j % 2 * 2] = none ? 0u : raw[j / 2][j % 2 * 2];
        raw[j / 2][j % 2 * 2 + 1] = none ? 0u : raw[j / 2][j % 2 * 2 + 1];
      }
    }
    unsigned most = 0, rows[8];  // of all, and of two values side by side: those that a thread for values has of a row
    const auto measure = [&] {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        rows[j] = larger(size_of(raw[j / 2][j % 2 * 2]), size_of(raw[j / 2][j % 2 * 2 + 1]));
        most = larger(most, rows[j]);
      }
    };
    measure();
    if (__any(most >= kFar)) {  // rare; for the rows that do not see it, as zeros, which change nothing
      odd = true;
      most = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[b][i] = size_of(raw[b][i]) >= kFar ? 0u : raw[b][i];
      measure();
    }
    // in the place where float32 has it, e with |v| < 2^(e - 126), 26 or more: 2^(140 - e) brings v to 2^13 .. 2^14
    const auto exponent_of = [&](unsigned v) { return larger(v, 26u << 23) & 0x7f800000u; };
    constexpr unsigned kUp = 267u << 23;
    if (for_keys) {
      const unsigned e = exponent_of(lanes_max<SIDE>(most));
      const float up = __uint_as_float(kUp - e);
      const unsigned key = me / SIDE, part = me % SIDE;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        f16x2 hi[2], lo[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) split_two(__uint_as_float(raw[b][2 * i]) * up, __uint_as_float(raw[b][2 * i + 1]) * up, hi[i], lo[i]);
        const unsigned step = part / 4 + SIDE / 4 * b, to = exchange(part / 2 % 2 * 32 + key, step);
        reinterpret_cast<u32x2*>(&s.keys[0][step][to])[part % 2] = u32x2{__builtin_bit_cast(unsigned, hi[0]), __builtin_bit_cast(unsigned, hi[1])};
        reinterpret_cast<u32x2*>(&s.keys[PIECES - 1][step][to])[part % 2] = u32x2{__builtin_bit_cast(unsigned, lo[0]), __builtin_bit_cast(unsigned, lo[1])};
      }
      if (part == 0) s.key_scale[key] = __uint_as_float(e - (13u << 23));
      // a bit for each SIDE threads to neighbouring bits: of 8 by a product that moves bit 8 i to 56 + i
      u64 nowhere = __ballot(gone);
      if constexpr (SIDE == 8) {
        nowhere = (nowhere & 0x0101010101010101ull) * 0x0102040810204080ull >> 56;
      } else {
        nowhere &= 0x1111111111111111ull;
        nowhere = (nowhere | nowhere >> 3) & 0x0303030303030303ull;
        nowhere = (nowhere | nowhere >> 6) & 0x000f000f000f000full;
        nowhere = (nowhere | nowhere >> 12) & 0x000000ff000000ffull;
        nowhere |= nowhere >> 24;
      }
      if (lane == 0) s.gone[wave] = (unsigned)(nowhere & ((1ull << 64 / SIDE) - 1)) << (64 / SIDE * wave);
    } else {
      const unsigned word = me % WORDS, group = me / WORDS;
      unsigned exponent[8];
      float up[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // of the lanes that have the row
        exponent[j] = exponent_of(lanes_max<WORDS>(rows[j]));
        up[j] = __uint_as_float(kUp - exponent[j]);
      }
      unsigned e = exponent[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) e = word == (unsigned)j ? exponent[j] : e;
      if (word < 8) {
        const unsigned key = group / 2 * 16 + 4 * (group % 2) + 8 * (word / 4) + word % 4;
        s.value_scale[key] = __uint_as_float(e + (unsigned)((kLift - 13) * (1 << 23)));
        s.value_log[key] = (float)((int)(e >> 23) - 140 + kLift);
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        Half8 hi, lo;
#pragma unroll
        for (int j = 0; j < 4; ++j) split_two(__uint_as_float(raw[j][b]) * up[2 * j], __uint_as_float(raw[j][2 + b]) * up[2 * j + 1], hi.p[j], lo.p[j]);
        s.values[0][word / 32 * 2 + b][group / 2][32 * (group % 2) + word % 32] = __builtin_bit_cast(u32x4, hi.v);
        s.values[PIECES - 1][word / 32 * 2 + b][group / 2][32 * (group % 2) + word % 32] = __builtin_bit_cast(u32x4, lo.v);
      }
    }
  };
  const auto store = [&](Stage& s, int at) {
    if constexpr (S8) store_s8(s);
    else store_f32(s, at);
  };

  if (begin < end) {
    ask_pages(begin);
    fetch(begin);
    if (begin + kTileKeys < end) ask_pages(begin + kTileKeys);
  }
  // the row's query, as above: value 16 s + 8 (l / 32) + j in [s][j]
  f16x8 q_hi[KS], q_lo[KS];
  float row_scale;
  {
    const float* const q = p.q + (unsigned long long)(t.first + (t.row_token < 0 ? 0 : t.row_token)) * p.q_token + (head * p.group.d + t.row_head) * p.q_head;
    f32x4 x[2 * KS];
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < 2 * KS; ++s) {
      const unsigned d = 16 * (s / 2) + 8 * half + 4 * (s % 2);
      x[s] = f32x4{0, 0, 0, 0};
      if (t.row_token >= 0 && d < size) x[s] = *reinterpret_cast<const f32x4*>(q + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(x[s][j]));
    }
    float a, b;
    butterfly_pair<32>(top, a, b);
    const QueryScale scale = query_scale(fmaxf(a, b), p.scale);
    const float up = scale.up;
    row_scale = scale.scale;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      Half8 hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (S4) split_two(x[2 * s][j] * up, x[2 * s + 1][j] * up, hi.p[j], lo.p[j]);  // the order of a word's integers
        else split_two(x[2 * s + j / 2][j % 2 * 2] * up, x[2 * s + j / 2][j % 2 * 2 + 1] * up, hi.p[j], lo.p[j]);
      }
      q_hi[s] = hi.v;
      q_lo[s] = lo.v;
    }
  }
  f32x16 o[N];
#pragma unroll
  for (int n = 0; n < N; ++n) o[n] = f32x16{};
  float frame = -INFINITY, l = 0.0f;
  ScoreShape shape;
  if constexpr (SHAPED) {
    shape.start(p, t, head, row_scale);
    row_scale = shape.unit;
  }

  unsigned turn = 0;
#pragma unroll 1
  for (int kb = begin; kb < end; kb += kTileKeys, turn ^= 1) {
    Stage& s = stages[turn];
    store(s, kb);
    if (kb + kTileKeys < end) {
      fetch(kb + kTileKeys);
      if (kb + 2 * kTileKeys < end) ask_pages(kb + 2 * kTileKeys);
    }
    __syncthreads();
    if (kb >= high || kb + kTileKeys <= low) continue;
    f32x16 x = {};
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      const unsigned at = S8 ? lane : exchange(lane, k);
      const f16x8 a = __builtin_bit_cast(f16x8, s.keys[0][k][at]);
      if constexpr (!S8) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, s.keys[PIECES - 1][k][at]), q_hi[k], x, 0, 0, 0);
      x = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q_lo[k], x, 0, 0, 0);
      x = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q_hi[k], x, 0, 0, 0);
    }
    f32x4 value_scale[4], value_log[4];
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const f32x4 key_scale = *reinterpret_cast<const f32x4*>(s.key_scale + 8 * a + 4 * half);
      if constexpr (S8) {
        value_scale[a] = *reinterpret_cast<const f32x4*>(s.value_scale + 8 * a + 4 * half);
        value_log[a] = *reinterpret_cast<const f32x4*>(s.value_log + 8 * a + 4 * half);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * a + i] *= key_scale[i];
    }
    if constexpr (SHAPED) {
      float formed[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) formed[i] = x[i];
      shape.apply(formed, kb + 4 * (int)half, [](int i) { return 8 * (i / 4) + i % 4; });
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = formed[i];
    }
    unsigned none = s.gone[0];
#pragma unroll
    for (int i = 1; i < WAVES / 2; ++i) none |= s.gone[i];
    if (none != 0 || kb < all_low || kb + kTileKeys > all_high) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int key = kb + 8 * (i / 4) + 4 * (int)half + i % 4;
        const bool seen = (none >> (key - kb) & 1) == 0 && key >= t.row_low && key < t.row_high;
        x[i] = seen ? x[i] : -INFINITY;
        if constexpr (S8) value_scale[i / 4][i % 4] = seen ? value_scale[i / 4][i % 4] : 0.0f;  // it may be anything
      }
    }
    if constexpr (!S8) {
#pragma unroll
      for (int a = 0; a < 4; ++a) value_log[a] = *reinterpret_cast<const f32x4*>(s.value_log + 8 * a + 4 * half);
    }
    float top = -INFINITY, a, b;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fmaf(x[i], row_scale, value_log[i / 4][i % 4]));
    butterfly_pair<32>(top, a, b);
    top = fmaxf(a, b);
    if (__any(top - frame > 15.0f)) {
      const float next = top - frame > 15.0f ? top - 8.0f : frame, h = next == frame ? 1.0f : half_step(frame, next), f = h * h;
      frame = next;
      l = l * h * h;
#pragma unroll
      for (int n = 0; n < N; ++n) o[n] *= f;
    }
    const float zero = frame == -INFINITY ? 0.0f : frame;
    if constexpr (!S8) {
#pragma unroll
      for (int a = 0; a < 4; ++a) value_scale[a] = *reinterpret_cast<const f32x4*>(s.value_scale + 8 * a + 4 * half);
    }
    Half8 w_hi[2], w_lo[2];
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e = __builtin_amdgcn_exp2f(fmaf(x[i], row_scale, -zero));
      l += e;
      w[i] = e * value_scale[i / 4][i % 4];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) split_two(w[2 * i], w[2 * i + 1], w_hi[i / 4].p[i % 4], w_lo[i / 4].p[i % 4]);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const f16x8 v = __builtin_bit_cast(f16x8, s.values[0][n][h][lane]);
        if constexpr (!S8) o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, s.values[PIECES - 1][n][h][lane]), w_hi[h].v, o[n], 0, 0, 0);
        o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, w_lo[h].v, o[n], 0, 0, 0);
        o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, w_hi[h].v, o[n], 0, 0, 0);
      }
  }
  float a, b;
  butterfly_pair<32>(l, a, b);
  l = a + b;
  frame = frame_out(frame, l);
  if (t.row_token >= 0) {
    const unsigned long long token = t.first + t.row_token, query_head = head * p.group.d + t.row_head;
    float* to = p.out + token * p.out_token + query_head * p.out_head;
    if constexpr (!S8) {
#pragma unroll
      for (int n = 0; n < N; ++n) o[n] *= power(-kLift);
    }
    float factor = 1.0f;
    if (p.splits > 1) {
      const unsigned long long place = ((unsigned long long)split * p.tokens + token) * p.cache.heads * p.group.d + query_head;
      to = p.partial + place * size;
      if (half == 0) {
        p.statistics[place * 2] = frame;
        p.statistics[place * 2 + 1] = l;
      }
    } else {
      factor = frame == -INFINITY ? 0.0f : 1.0f / l;
    }
    if constexpr (S8) {
#pragma unroll
      for (int n = 0; n < N; n += n / 4 * 4 + 4 <= N ? 4 : 2)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const unsigned d = value_of<BLOCKS, S8>(8 * (i / 4) + 4 * half + i % 4, n);
          if (d >= size) continue;
          if (n / 4 * 4 + 4 <= N) {
            *reinterpret_cast<f32x4*>(to + d) = f32x4{o[n][i], o[n + 1][i], o[n + 2][i], o[n + 3][i]} * factor;
          } else {
            *reinterpret_cast<f32x2*>(to + d) = f32x2{o[n][i] * factor, o[n + 1][i] * factor};
          }
        }
    } else {
#pragma unroll
      for (int n = 0; n < N; n += 2)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const unsigned d = value_of<BLOCKS, S8>(8 * (i / 4) + 4 * half + i % 4, n);
          if (d < size) *reinterpret_cast<f32x4*>(to + d) = f32x4{o[n][i], o[n + 1][i], o[n][i + 1], o[n + 1][i + 1]} * factor;
        }
    }
  }
  if constexpr (!S8) {
    __shared__ unsigned odds[WAVES];
    if (lane == 0) odds[wave] = odd ? 1u : 0u;
    __syncthreads();
    unsigned any = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) any |= odds[w];
    if (any != 0) stream_far_rows_apart<BLOCKS, WAVES, SHAPED>(*(const AttentionArgs*)__builtin_amdgcn_kernarg_segment_ptr());  // the kernel's one argument, where it lies
  }
}

// Integers in any layout, a page for each key, loaded when it is due: pages of fewer than 16 rows, scales that do not lie in a row, int8 rows that cannot be read 16 bytes at a time
// (32 sequences of 4096, 8 heads of 128, pages of 8 rows: int8 129 us, 4 bits 69; of 32 rows, by the ring, 49 and 34).
template <int TYPE, int BLOCKS, int WAVES, bool SHAPED>
__global__ __launch_bounds__(WAVES * 64) void attention_scaled_any_kernel(AttentionArgs p) {
  constexpr int STEP = 32 * WAVES;
  typedef ScaledLayout<TYPE, BLOCKS> Layout;
  __shared__ Joining<64 * BLOCKS, WAVES> joining;
  Tile t;
  unsigned head, split;
  int begin, end;
  if (!take_work<SHAPED>(p, kAttentionRows, threadIdx.x % 16, t, head, split, begin, end)) return;
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x / 64, g = lane / 16, c = lane % 16;
  const unsigned size = p.cache.size / Layout::PER;  // of a row, in bytes
  const int8_t* const keys = static_cast<const int8_t*>(p.cache.keys) + head * p.cache.head;
  const int8_t* const values = static_cast<const int8_t*>(p.cache.values) + head * p.cache.head;
  const float* const key_scales = p.cache.key_scales + head * p.cache.scale_head;
  const float* const value_scales = p.cache.value_scales + head * p.cache.scale_head;
  const int* const table = p.table + t.sequence * p.table_stride;
  const auto locate = [&](int key, unsigned long long& row, unsigned long long& scale) {
    const unsigned index = p.cache.page_size.quotient((unsigned)key), inside = (unsigned)key - index * p.cache.page_size.d;
    const int page = page_of(p, table, index);
    row = page < 0 ? 0 : page * p.cache.page + inside * p.cache.row;
    scale = page < 0 ? 0 : page * p.cache.scale_page + inside * p.cache.scale_row;
    return page >= 0;
  };
  ScaledRows<TYPE, BLOCKS, SHAPED> rows;
  rows.start(p, t, head, g);
#pragma unroll 1
  for (int kb = begin + 32 * (int)wave; kb < end; kb += STEP) {
    unsigned k[2][Layout::KEY_WORDS], v[8][Layout::VALUE_WORDS], missing = 0;
    f32x4 key_scale[2], value_scale[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unsigned long long row, scale;
      locate(kb + 16 * h + (int)c, row, scale);
#pragma unroll
      for (int b = 0; b < Layout::KEY_WORDS; b += 2) {  // rows are 8-byte aligned
        constexpr int RUN = Layout::RUN / Layout::PER / 4;  // words
        const unsigned d = 4 * (4 * RUN * (b / RUN) + RUN * g + b % RUN);
        const u32x2 w = *reinterpret_cast<const u32x2*>(keys + row + (d < size ? d : 0));
        k[h][b] = w[0];
        k[h][b + 1] = w[1];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        missing |= locate(kb + 16 * h + 4 * (int)g + i, row, scale) ? 0u : 1u << (4 * h + i);
        key_scale[h][i] = key_scales[scale];
        value_scale[h][i] = value_scales[scale];
#pragma unroll
        for (int b = 0; b < Layout::VALUE_WORDS; ++b) {
          const unsigned d = Layout::BYTES / 16 * c + 4 * b;
          const int8_t* const at = values + row + (d < size ? d : 0);
          v[4 * h + i][b] = Layout::BYTES < 64 ? *reinterpret_cast<const unsigned short*>(at) : *reinterpret_cast<const unsigned*>(at);
        }
      }
    }
    float s[8];
    rows.score(k, key_scale, s);
    rows.form(kb, g, s);
    rows.hide(t, kb, g, missing, s, value_scale);
    rows.add(s, value_scale, v);
  }
  rows.template finish<WAVES>(joining, p, t, head, split, g);
}

// float32: 16 keys in one step of a wavefront (2 sequences of 30011, 8 heads of 128, 478 MB: 89 us, 5.4 TB/s, then 5 for the join).
template <int BLOCKS, int WAVES, int PAGES, bool SHAPED>
__global__ __launch_bounds__(WAVES * 64) void attention_f32_kernel(AttentionArgs p) {
  constexpr int DPAD = 64 * BLOCKS, STEP = 16 * WAVES;
  __shared__ Joining<DPAD, WAVES> joining;
  Tile t;
  unsigned head, split;
  int begin, end;
  if (!take_work<SHAPED>(p, kAttentionRows, threadIdx.x % 16, t, head, split, begin, end)) return;
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x / 64, g = lane / 16;
  const auto store = [&](const f32x4 (&o)[BLOCKS][4], float m, float l) {
    l = across_groups_sum(l);
    float list[DPAD / 4];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) list[(b * 4 + i) * 4 + j] = o[b][j][i];
    join_and_store(joining, p, t, head, split, frame_out(m, l), l, list, [&](int at) { return 64 * (at / 16) + 4 * (4 * (int)g + at % 16 / 4); });
  };
  stream_rows<BLOCKS, STEP, PAGES, SHAPED>(p, t, head, begin + 16 * (int)wave, end, p.table + t.sequence * p.table_stride,
                                   [](int, const f32x4 (&)[4 * BLOCKS], const f32x4 (&)[4][BLOCKS], unsigned) {}, store);
}

// What a step's 16 keys may lie in: 1 page, up to 2, or any number (0).
int pages_of_step(unsigned page_size) { return page_size % 16 == 0 ? 1 : page_size >= 16 ? 2 : 0; }

template <int TYPE, int BLOCKS, int WAVES, bool SHAPED>
void launch_scaled_of(const AttentionArgs& a, dim3 grid, hipStream_t s, bool wide) {
  const auto start = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(WAVES * 64), 0, s, a); };
  const unsigned rows = a.cache.page_size.d;
  if (!wide) return start(attention_scaled_any_kernel<TYPE, BLOCKS, WAVES, SHAPED>);
  if constexpr (TYPE == TFCC_ROCM_S4) {
    const unsigned long long bytes = a.cache.size / 2 | a.cache.page | a.cache.head | a.cache.row | reinterpret_cast<uintptr_t>(a.cache.keys) | reinterpret_cast<uintptr_t>(a.cache.values);
    if (bytes % 16 != 0) return start(attention_scaled_kernel<TYPE, BLOCKS, WAVES, -1, SHAPED>);
    if (rows % 32 == 0) return start(attention_scaled_kernel<TYPE, BLOCKS, WAVES, 32, SHAPED>);
  }
  start(rows % 16 == 0 ? attention_scaled_kernel<TYPE, BLOCKS, WAVES, 16, SHAPED> : attention_scaled_kernel<TYPE, BLOCKS, WAVES, 0, SHAPED>);
}
template <int TYPE, int BLOCKS, bool SHAPED>
void launch_scaled(const AttentionArgs& a, dim3 grid, hipStream_t s, unsigned waves, bool wide) {
  if constexpr (TYPE == TFCC_ROCM_S4 && BLOCKS <= 2)
    if (waves == 12) return launch_scaled_of<TYPE, BLOCKS, 12, SHAPED>(a, grid, s, wide);
  if constexpr (TYPE == TFCC_ROCM_S8 ? BLOCKS <= 2 : BLOCKS == 4)
    if (waves == 8) return launch_scaled_of<TYPE, BLOCKS, 8, SHAPED>(a, grid, s, wide);
  launch_scaled_of<TYPE, BLOCKS, 4, SHAPED>(a, grid, s, wide);
}
template <int TYPE, int BLOCKS, bool SHAPED>
void launch_tiles(const AttentionArgs& a, dim3 grid, hipStream_t s) {
  const bool whole = a.cache.page_size.d % 16 == 0;
  hipLaunchKernelGGL((whole ? attention_tile_kernel<TYPE, BLOCKS, 4, true, SHAPED> : attention_tile_kernel<TYPE, BLOCKS, 4, false, SHAPED>), grid, dim3(256), 0, s, a);
}
template <int BLOCKS, bool SHAPED>
void launch_f32(const AttentionArgs& a, dim3 grid, hipStream_t s, unsigned waves) {
  const auto start = [&](auto one, auto two, auto any, unsigned width) {
    const int pages = pages_of_step(a.cache.page_size.d);
    hipLaunchKernelGGL((pages == 1 ? one : pages == 2 ? two : any), grid, dim3(width * 64), 0, s, a);
  };
  if constexpr (BLOCKS <= 2)
    if (waves == 8) return start(attention_f32_kernel<BLOCKS, 8, 1, SHAPED>, attention_f32_kernel<BLOCKS, 8, 2, SHAPED>, attention_f32_kernel<BLOCKS, 8, 0, SHAPED>, 8);
  start(attention_f32_kernel<BLOCKS, 4, 1, SHAPED>, attention_f32_kernel<BLOCKS, 4, 2, SHAPED>, attention_f32_kernel<BLOCKS, 4, 0, SHAPED>, 4);
}

// The kernel of a call that has been dealt out, BLOCKS of 64 values in a head; wide: a cache of integers that can be read 16 bytes at a time.
template <bool SHAPED>
void launch_attention(const AttentionArgs& a, int type, bool wide, const PagedAttentionPlan& plan, hipStream_t s) {
  const dim3 grid(plan.tiles * plan.splits * a.cache.heads);
  const unsigned blocks = (a.cache.size + 63) / 64;
  const auto scaled = [&](auto code) {
    constexpr int TYPE = decltype(code)::value;
    if (blocks == 1) launch_scaled<TYPE, 1, SHAPED>(a, grid, s, plan.waves, wide);
    else if (blocks == 2) launch_scaled<TYPE, 2, SHAPED>(a, grid, s, plan.waves, wide);
    else launch_scaled<TYPE, 4, SHAPED>(a, grid, s, plan.waves, wide);
  };
  if (plan.rows != kAttentionRows && type == TFCC_ROCM_F32) {
    if (blocks == 1) hipLaunchKernelGGL((attention_tile_kernel<TFCC_ROCM_F32, 1, 4, false, SHAPED>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attention_tile_kernel<TFCC_ROCM_F32, 2, 8, false, SHAPED>), grid, dim3(512), 0, s, a);
  } else if (plan.rows != kAttentionRows) {
    if (type == TFCC_ROCM_S4) launch_tiles<TFCC_ROCM_S4, 2, SHAPED>(a, grid, s);
    else if (blocks == 1) launch_tiles<TFCC_ROCM_S8, 1, SHAPED>(a, grid, s);
    else if (blocks == 2) launch_tiles<TFCC_ROCM_S8, 2, SHAPED>(a, grid, s);
    else if (blocks == 3) launch_tiles<TFCC_ROCM_S8, 3, SHAPED>(a, grid, s);
    else launch_tiles<TFCC_ROCM_S8, 4, SHAPED>(a, grid, s);
  } else if (type != TFCC_ROCM_F32) {
    if (type == TFCC_ROCM_S4) scaled(std::integral_constant<int, TFCC_ROCM_S4>());
    else scaled(std::integral_constant<int, TFCC_ROCM_S8>());
  } else {
    if (blocks == 1) launch_f32<1, SHAPED>(a, grid, s, plan.waves);
    else if (blocks == 2) launch_f32<2, SHAPED>(a, grid, s, plan.waves);
    else if (blocks == 3) launch_f32<3, SHAPED>(a, grid, s, plan.waves);
    else launch_f32<4, SHAPED>(a, grid, s, plan.waves);
  }
}

}  // namespace

// launch_attention for shaped scores, in a file of its own: each has the kernels once.
void launch_shaped_attention(const AttentionArgs& a, int type, bool wide, const PagedAttentionPlan& plan, hipStream_t s);

}  // namespace tfcc_rocm
