// Attention of new tokens over a paged cache: out = softmax(c q k^T) v for the chunk of each sequence, one pass over the keys with
// the running maximum and sum of each row.
//
// The query heads of a token that share a cache head are rows of one product: row r of a sequence is token r / group, head r % group, and
// a tile holds 16 rows.  Both products run transposed on the matrix cores, with a row in each column:
//   S^T = K Q^T   (16 keys x 16 rows): lane l holds row l % 16 and keys 4 (l / 16) + i, i < 4
//   O^T = V^T P^T (16 values x 16 rows)
// so a row's maximum, sum and scale sit in the lanes that hold its scores, and the scores are where the second product wants its
// right operand: a contraction may run over the keys in any order, so lane group g contracts the keys that it holds.  Nothing is
// exchanged between lanes but two steps of the row maximum.  V is loaded as it lies, row by row; which column of the
// product stands for which value of a head is free as well and follows the loads.
//
// An int8 cache keeps float32 accuracy: an int8 is exact in fp16, a float32 is nearly the sum of two (22 bits), so each product is two
// fp16 matrix operations.  Queries are scaled by a power of two per row, weights times value scales by one per row that follows
// the largest such product, so that the largest are near 2^14 and what fp16 cannot hold is 2^-38 of it.  A float32 cache
// goes through the fp32 matrix operations.
//
// The keys of a tile are dealt to the four wavefronts of a workgroup in turns, and in pieces to several workgroups where there are few
// tiles; each wavefront keeps maximum, sum and output of its own, joined in LDS, the pieces by a second launch.
#include "paged_attention_plan.hpp"
#include "paged_cache.hpp"

namespace tfcc_rocm {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = 4;

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
};

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
};

// The chunks' tiles are counted off along the batch, 64 sequences at a time.
__device__ Tile find_tile(const AttentionArgs& p, unsigned tile, unsigned rows_of_tile, unsigned row) {
  const unsigned lane = threadIdx.x & 63;
  Tile t;
  t.any = false;
  unsigned before = 0;
  for (unsigned base = 0; base < p.batch; base += 64) {
    const unsigned b = base + lane;
    int first = 0, count = 0;
    if (b < p.batch) {
      first = p.starts[b];
      int next = p.starts[b + 1];
      next = next > (int)p.tokens ? (int)p.tokens : next;
      count = first >= 0 && next > first ? next - first : 0;
    }
    const unsigned mine = ((unsigned)count * p.group.d + rows_of_tile - 1) / rows_of_tile;
    unsigned upto = mine;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
      const unsigned o = (unsigned)__shfl_up((int)upto, m, 64);
      if (lane >= (unsigned)m) upto += o;
    }
    upto += before;
    const unsigned long long past = __ballot(upto > tile);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      t.any = true;
      t.sequence = base + at;
      t.first = __builtin_amdgcn_readlane(first, at);
      t.count = __builtin_amdgcn_readlane(count, at);
      t.row0 = (int)((tile - (unsigned)__builtin_amdgcn_readlane((int)(upto - mine), at)) * rows_of_tile);
      break;
    }
    before = (unsigned)__builtin_amdgcn_readlane((int)upto, 63);
  }
  if (!t.any) return t;
  int length = p.lengths[t.sequence];
  length = length < 0 ? 0 : length;
  const int position0 = length - t.count;  // of the chunk's first token
  t.length = length < (int)p.max_length ? length : (int)p.max_length;
  const int rows = t.count * (int)p.group.d;
  const int last_row = t.row0 + (int)rows_of_tile < rows ? t.row0 + (int)rows_of_tile - 1 : rows - 1;
  const int token0 = (int)p.group.quotient((unsigned)t.row0), token1 = (int)p.group.quotient((unsigned)last_row);
  const auto sight = [&](int token, int& low, int& high) {
    low = 0;
    high = t.length;
    if (p.causal) {
      const int position = position0 + token;
      high = position + 1 < t.length ? position + 1 : t.length;
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
  if (r < rows) {
    t.row_token = (int)p.group.quotient((unsigned)r);
    t.row_head = r - t.row_token * (int)p.group.d;
    sight(t.row_token, t.row_low, t.row_high);
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

// 2^e for e in [-126, 127]; infinity for 128
__device__ __forceinline__ float power(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
// e with |v| < 2^e, from -100 to 128, so that 2^(14 - e) and its inverse are normal numbers
__device__ __forceinline__ int bound_of(float v) {
  const int e = (int)((__float_as_uint(v) >> 23) & 255) - 126;
  return e < -100 ? -100 : (e > 128 ? 128 : e);
}

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

// float32 as the sum of two fp16, both cut off: 22 bits, the error at most 2^-21 of the value
__device__ __forceinline__ void split_two(float a, float b, f16x2& hi, f16x2& lo) {
  hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(a, b));
  lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(a - (float)hi[0], b - (float)hi[1]));
}

// Joins the four wavefronts' outputs and writes them: to `out` where the keys are in one piece, else to the piece's part of the workspace.
// o[] of a lane is its row's value `place(n)`; four neighbours in n are four neighbours in memory.
template <int DPAD, class Place>
__device__ void join_and_store(const AttentionArgs& p, const Tile& t, unsigned head, unsigned split, float m, float l, const float* o, Place place) {
  constexpr int LD = DPAD + 4;
  __shared__ __align__(16) float outputs[kWaves][kAttentionRows][LD];
  __shared__ float maxima[kWaves][kAttentionRows], sums[kWaves][kAttentionRows];
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x / 64, row = lane % 16;
  constexpr int N = DPAD / 4;  // of a lane: 16 rows of DPAD values over 64 lanes
  if (lane < 16) {
    maxima[wave][row] = m;
    sums[wave][row] = l;
  }
#pragma unroll
  for (int n = 0; n < N; n += 4) {
    const f32x4 v = {o[n], o[n + 1], o[n + 2], o[n + 3]};
    *reinterpret_cast<f32x4*>(&outputs[wave][row][place(n)]) = v;
  }
  __syncthreads();
  const unsigned size = p.cache.size, heads = p.cache.heads * p.group.d;
  const int rows = t.count * (int)p.group.d;
  for (unsigned at = threadIdx.x; at < kAttentionRows * (DPAD / 4); at += kThreads) {
    const unsigned r = at / (DPAD / 4), d = at % (DPAD / 4) * 4;
    const int in_chunk = t.row0 + (int)r;
    if (in_chunk >= rows || d >= size) continue;
    float top = maxima[0][r];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, maxima[w][r]);
    float total = 0;
    f32x4 sum = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (sums[w][r] == 0.0f) continue;  // a wavefront that saw no key of this row
      const float f = __builtin_amdgcn_exp2f(maxima[w][r] - top);
      total += f * sums[w][r];
      sum += f * *reinterpret_cast<const f32x4*>(&outputs[w][r][d]);
    }
    const unsigned token = p.group.quotient((unsigned)in_chunk), inner = (unsigned)in_chunk - token * p.group.d;
    const unsigned long long global = t.first + token, query_head = head * p.group.d + inner;
    if (p.splits == 1) {
      const f32x4 none = {0, 0, 0, 0};
      *reinterpret_cast<f32x4*>(p.out + global * p.out_token + query_head * p.out_head + d) = total == 0.0f ? none : sum / total;
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
__device__ __forceinline__ bool take_work(const AttentionArgs& p, Tile& t, unsigned& head, unsigned& split, int& begin, int& end) {
  // cache heads first, then pieces, then tiles
  const unsigned outer = p.cache_heads.quotient(blockIdx.x), tile = p.pieces.quotient(outer);
  head = blockIdx.x - outer * p.cache_heads.d;
  split = outer - tile * p.pieces.d;
  t = find_tile(p, tile, kAttentionRows, threadIdx.x % 16);
  if (!t.any) return false;
  const long long from = (t.low & ~31) + (long long)split * p.split_keys, upto = from + p.split_keys;
  end = upto < t.high ? (int)upto : t.high;
  begin = from < end ? (int)from : end;
  if (begin >= end && p.splits > 1) {
    if (threadIdx.x < kAttentionRows && t.row_token >= 0) {
      const unsigned long long at = ((unsigned long long)split * p.tokens + t.first + t.row_token) * p.cache.heads * p.group.d + head * p.group.d + t.row_head;
      p.statistics[at * 2] = -INFINITY;
      p.statistics[at * 2 + 1] = 0.0f;
    }
    return false;
  }
  return true;
}

// The page that holds a key; -1: none.
__device__ __forceinline__ int page_of(const AttentionArgs& p, const int* table, unsigned index) {
  if (index >= p.table_width) return -1;
  const int page = table[index];
  return page >= 0 && (unsigned)page < p.cache.pages ? page : -1;
}

// int8: 32 keys in one step of a wavefront.  FAST: pages of a multiple of 16 rows, rows and scales that can be read 16 bytes at a time.
template <int BLOCKS, bool FAST>
__global__ __launch_bounds__(kThreads) void attention_s8_kernel(AttentionArgs p) {
  constexpr int DPAD = 64 * BLOCKS;
  Tile t;
  unsigned head, split;
  int begin, end;
  if (!take_work(p, t, head, split, begin, end)) return;
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x / 64, g = lane / 16, c = lane % 16;
  const unsigned size = p.cache.size;
  const int8_t* const keys = static_cast<const int8_t*>(p.cache.keys) + head * p.cache.head;
  const int8_t* const values = static_cast<const int8_t*>(p.cache.values) + head * p.cache.head;
  const float* const key_scales = p.cache.key_scales + head * p.cache.scale_head;
  const float* const value_scales = p.cache.value_scales + head * p.cache.scale_head;
  const int* const table = p.table + t.sequence * p.table_stride;

  // the row's query: value 64 b + 16 g + 8 h + j of the head in q[2 b + h][j], as two fp16 under a power of two
  f16x8 q_hi[2 * BLOCKS], q_lo[2 * BLOCKS];
  float row_scale = 0.0f;
  {
    f32x4 x[4 * BLOCKS];
    float top = 0.0f;
    const float* q = p.q + (unsigned long long)(t.first + (t.row_token < 0 ? 0 : t.row_token)) * p.q_token + (head * p.group.d + t.row_head) * p.q_head;
#pragma unroll
    for (int b = 0; b < 4 * BLOCKS; ++b) {
      const unsigned d = 64 * (b / 4) + 16 * g + 4 * (b % 4);
      f32x4 v = {0, 0, 0, 0};
      if (t.row_token >= 0 && d < size) v = *reinterpret_cast<const f32x4*>(q + d);
      x[b] = v;
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(v[j]));
    }
    top = across_groups_max(top);
    const int e = bound_of(top);
    const float up = power(14 - e);
    row_scale = power(e - 14) * p.scale;
#pragma unroll
    for (int b = 0; b < 2 * BLOCKS; ++b) {
      Half8 hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) split_two(x[2 * b + j / 2][j % 2 * 2] * up, x[2 * b + j / 2][j % 2 * 2 + 1] * up, hi.p[j], lo.p[j]);
      q_hi[b] = hi.v;
      q_lo[b] = lo.v;
    }
  }

  // V: value (DPAD / 16) c + n of the head in tile n
  constexpr int N = DPAD / 16;
  f32x4 o[N];
#pragma unroll
  for (int n = 0; n < N; ++n) o[n] = f32x4{0, 0, 0, 0};
  // weights times value scales were at most w_most, which is at most w_limit = 2^w_e, and enter times w_up = 2^(14 - w_e)
  float m = -INFINITY, l = 0.0f, w_most = 0.0f, w_limit = 0.0f, w_up = 0.0f;
  int w_e = -100;

  for (int kb = begin + 32 * (int)wave; kb < end; kb += 32 * kWaves) {
    unsigned long long key_at[2], value_at[8];
    float ks[8], vs[8];
    bool there[8];
    if constexpr (FAST) {
      const unsigned index0 = p.cache.page_size.quotient((unsigned)kb), index1 = p.cache.page_size.quotient((unsigned)kb + 16);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned index = h ? index1 : index0;
        const unsigned inside = (unsigned)kb + 16 * h - index * p.cache.page_size.d;
        const int page = page_of(p, table, index);
        const unsigned long long base = page < 0 ? 0 : page * p.cache.page + inside * p.cache.row;
        const unsigned long long scale_base = page < 0 ? 0 : page * p.cache.scale_page + inside;
        const unsigned long long row = page < 0 ? 0 : p.cache.row;
        key_at[h] = base + c * row;
        const f32x4 a = *reinterpret_cast<const f32x4*>(key_scales + scale_base + 4 * g), b = *reinterpret_cast<const f32x4*>(value_scales + scale_base + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          value_at[4 * h + i] = base + (4 * g + i) * row;
          ks[4 * h + i] = a[i];
          vs[4 * h + i] = b[i];
          there[4 * h + i] = page >= 0;
        }
      }
    } else {
      const auto locate = [&](int key, unsigned long long& at, unsigned long long& scale_at) {
        const unsigned index = p.cache.page_size.quotient((unsigned)key), inside = (unsigned)key - index * p.cache.page_size.d;
        const int page = page_of(p, table, index);
        at = page < 0 ? 0 : page * p.cache.page + inside * p.cache.row;
        scale_at = page < 0 ? 0 : page * p.cache.scale_page + inside * p.cache.scale_row;
        return page >= 0;
      };
      unsigned long long unused;
#pragma unroll
      for (int h = 0; h < 2; ++h) locate(kb + 16 * h + (int)c, key_at[h], unused);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        unsigned long long scale_at;
        there[i] = locate(kb + 16 * (i / 4) + 4 * (int)g + i % 4, value_at[i], scale_at);
        ks[i] = key_scales[scale_at];
        vs[i] = value_scales[scale_at];
      }
    }
    float s[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 acc = {0, 0, 0, 0};
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const unsigned d = 64 * b + 16 * g;
        u32x4 w;
        if constexpr (FAST) {
          w = *reinterpret_cast<const u32x4*>(keys + key_at[h] + (d < size ? d : 0));
        } else {
          const u32x2 w0 = *reinterpret_cast<const u32x2*>(keys + key_at[h] + (d < size ? d : 0));
          const u32x2 w1 = *reinterpret_cast<const u32x2*>(keys + key_at[h] + (d + 8 < size ? d + 8 : 0));
          w = u32x4{w0[0], w0[1], w1[0], w1[1]};
        }
        const f16x8 k0 = eight_int8(w[0], w[1]), k1 = eight_int8(w[2], w[3]);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q_lo[2 * b], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q_lo[2 * b + 1], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q_hi[2 * b], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q_hi[2 * b + 1], acc, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[4 * h + i] = acc[i] * (row_scale * ks[4 * h + i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int key = kb + 16 * (i / 4) + 4 * (int)g + i % 4;
      const bool seen = there[i] && key >= t.row_low && key < t.row_high;
      s[i] = seen ? s[i] : -INFINITY;
    }
    float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    top = across_groups_max(top);
    const float next = fmaxf(m, top), zero = next == -INFINITY ? 0.0f : next;
    Half8 w_hi, w_lo;
    float w[8], w_top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = __builtin_amdgcn_exp2f(s[i] - zero);
      s[i] = e;
      w[i] = e == 0.0f ? 0.0f : e * vs[i];
      w_top = fmaxf(w_top, fabsf(w[i]));
    }
    w_top = across_groups_max(w_top);
    if (__any(next > m || w_top > w_limit)) {
      const float f = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= f;
      w_most = fmaxf(w_top, w_most * f);
      const int e = bound_of(w_most), step = w_e - e;
      w_e = e;
      w_limit = power(e);
      w_up = power(14 - e);
      const float both = f * power(step < -126 ? -126 : step > 127 ? 127 : step);
#pragma unroll
      for (int n = 0; n < N; ++n) o[n] *= both;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      l += s[i];
      w[i] *= w_up;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) split_two(w[2 * i], w[2 * i + 1], w_hi.p[i], w_lo.p[i]);
    // DPAD / 16 bytes of each of the lane's eight keys, four at a time
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      unsigned word[8];
      const unsigned d = 4 * BLOCKS * c + 4 * b;
#pragma unroll
      for (int i = 0; i < 8; ++i) word[i] = *reinterpret_cast<const unsigned*>(values + value_at[i] + (d < size ? d : 0));
      const f16x8 v0 = eight_of<0>(word), v1 = eight_of<1>(word), v2 = eight_of<2>(word), v3 = eight_of<3>(word);
      o[4 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, w_lo.v, o[4 * b], 0, 0, 0);
      o[4 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, w_lo.v, o[4 * b + 1], 0, 0, 0);
      o[4 * b + 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v2, w_lo.v, o[4 * b + 2], 0, 0, 0);
      o[4 * b + 3] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v3, w_lo.v, o[4 * b + 3], 0, 0, 0);
      o[4 * b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, w_hi.v, o[4 * b], 0, 0, 0);
      o[4 * b + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, w_hi.v, o[4 * b + 1], 0, 0, 0);
      o[4 * b + 2] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v2, w_hi.v, o[4 * b + 2], 0, 0, 0);
      o[4 * b + 3] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v3, w_hi.v, o[4 * b + 3], 0, 0, 0);
    }
  }
  l = across_groups_sum(l);
  const float down = power(w_e - 14);
  // o[n][i] is value N (4 g + i) + n: rearranged so that neighbours of the list are neighbours of the head
  float list[DPAD / 4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int n = 0; n < N; ++n) list[i * N + n] = o[n][i] * down;
  join_and_store<DPAD>(p, t, head, split, m, l, list, [&](int at) { return N * (4 * (int)g + at / N) + at % N; });
}

// float32: 16 keys in one step of a wavefront.  UNIFORM: pages of a multiple of 16 rows.
template <int BLOCKS, bool UNIFORM>
__global__ __launch_bounds__(kThreads) void attention_f32_kernel(AttentionArgs p) {
  constexpr int DPAD = 64 * BLOCKS;
  Tile t;
  unsigned head, split;
  int begin, end;
  if (!take_work(p, t, head, split, begin, end)) return;
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x / 64, g = lane / 16, c = lane % 16;
  const unsigned size = p.cache.size;
  const float* const keys = static_cast<const float*>(p.cache.keys) + head * p.cache.head;
  const float* const values = static_cast<const float*>(p.cache.values) + head * p.cache.head;
  const int* const table = p.table + t.sequence * p.table_stride;

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
  // value 64 b + 4 (4 g + i) + j of the output in o[b][j][i]
  f32x4 o[BLOCKS][4];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[b][j] = f32x4{0, 0, 0, 0};
  float m = -INFINITY, l = 0.0f;

  for (int kb = begin + 16 * (int)wave; kb < end; kb += 16 * kWaves) {
    unsigned long long key_at, value_at[4];
    bool there[4], every = true;
    if constexpr (UNIFORM) {
      const unsigned index = p.cache.page_size.quotient((unsigned)kb), inside = (unsigned)kb - index * p.cache.page_size.d;
      const int page = page_of(p, table, index);
      const unsigned long long base = page < 0 ? 0 : page * p.cache.page + inside * p.cache.row, row = page < 0 ? 0 : p.cache.row;
      key_at = base + c * row;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        value_at[i] = base + (4 * g + i) * row;
        there[i] = page >= 0;
      }
      every = page >= 0;
    } else {
      const auto locate = [&](int key, unsigned long long& at) {
        const unsigned index = p.cache.page_size.quotient((unsigned)key), inside = (unsigned)key - index * p.cache.page_size.d;
        const int page = page_of(p, table, index);
        at = page < 0 ? 0 : page * p.cache.page + inside * p.cache.row;
        return page >= 0;
      };
      locate(kb + (int)c, key_at);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        there[i] = locate(kb + 4 * (int)g + i, value_at[i]);
        every = every && there[i];
      }
      every = __all(every);
    }
    f32x4 k[4 * BLOCKS], v[4][BLOCKS];
#pragma unroll
    for (int b = 0; b < 4 * BLOCKS; ++b) {
      const unsigned d = 16 * b + 4 * g;
      k[b] = *reinterpret_cast<const f32x4*>(keys + key_at + (d < size ? d : 0));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const unsigned d = 64 * b + 4 * c;
        v[i][b] = *reinterpret_cast<const f32x4*>(values + value_at[i] + (d < size ? d : 0));
      }
    f32x4 s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < 4 * BLOCKS; ++b) {
      f32x4 x = k[b];
      if (size != DPAD && 16 * b + 4 * g >= size) x = f32x4{0, 0, 0, 0};
      s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(x[0], q[b][0], s0, 0, 0, 0);
      s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(x[1], q[b][1], s1, 0, 0, 0);
      s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(x[2], q[b][2], s0, 0, 0, 0);
      s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(x[3], q[b][3], s1, 0, 0, 0);
    }
    f32x4 s = s0 + s1;
    const bool edge = !every || kb < t.all_low || kb + 16 > t.all_high;
    unsigned foreign = 0;  // values that are not finite, of keys that some row does not see
    if (edge) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = kb + 4 * (int)g + i;
        s[i] = there[i] && key >= t.row_low && key < t.row_high ? s[i] : -INFINITY;
        const bool none = !there[i] || key < t.low || key >= t.high;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool odd = (__float_as_uint(v[i][b][j]) & 0x7f800000u) == 0x7f800000u;
            foreign |= odd && !none ? 1u : 0u;
            v[i][b][j] = none || odd ? 0.0f : v[i][b][j];
          }
      }
    }
    const float top = across_groups_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
    if (__any(top > m)) {
      const float next = fmaxf(m, top);
      const float f = next == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - next);
      m = next;
      l *= f;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[b][j] *= f;
    }
    const float zero = m == -INFINITY ? 0.0f : m;
    float e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      e[i] = __builtin_amdgcn_exp2f(s[i] - zero);
      l += e[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[b][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[i][b][j], e[i], o[b][j], 0, 0, 0);
    if (edge && __any(foreign != 0)) {
      // Rare: a key with an infinity or a NaN among its values that only some of the rows see.  A product over all rows would hand
      // 0 x infinity to the others, so it went in as zeros and is added here, to the rows that see it.
      for (int at = 0; at < 16; ++at) {
        const int key = kb + at;
        const unsigned from = c + 16 * (at / 4);
        const float e0 = __shfl(e[0], (int)from, 64), e1 = __shfl(e[1], (int)from, 64), e2 = __shfl(e[2], (int)from, 64), e3 = __shfl(e[3], (int)from, 64);
        const float weight = at % 4 == 0 ? e0 : at % 4 == 1 ? e1 : at % 4 == 2 ? e2 : e3;
        const unsigned index = p.cache.page_size.quotient((unsigned)key), inside = (unsigned)key - index * p.cache.page_size.d;
        const int page = page_of(p, table, index);
        if (page < 0 || key < t.row_low || key >= t.row_high) continue;
        const float* row = values + page * p.cache.page + inside * p.cache.row;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const unsigned d = 64 * b + 4 * (4 * g + i) + j;
              const float x = d < size ? row[d] : 0.0f;
              if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) o[b][j][i] += weight * x;
            }
      }
    }
  }
  l = across_groups_sum(l);
  float list[DPAD / 4];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) list[(b * 4 + i) * 4 + j] = o[b][j][i];
  join_and_store<DPAD>(p, t, head, split, m, l, list, [&](int at) { return 64 * (at / 16) + 4 * (4 * (int)g + at % 16 / 4); });
}

// The pieces of a row joined: one wavefront to a row.
__global__ __launch_bounds__(kThreads) void join_pieces_kernel(AttentionArgs p) {
  __shared__ float weights[kWaves][kAttentionMostSplits];
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x / 64, heads = p.cache.heads * p.group.d, size = p.cache.size;
  const unsigned long long row = (unsigned long long)blockIdx.x * kWaves + wave, rows = (unsigned long long)p.tokens * heads;
  if (row >= rows) return;
  const unsigned token = (unsigned)(row / heads), head = (unsigned)(row - (unsigned long long)token * heads);
  if ((int)token >= p.starts[p.batch] || (int)token < p.starts[0]) return;
  float top = -INFINITY;
  for (unsigned i = lane; i < p.splits; i += 64) {
    const float* s = p.statistics + (i * rows + row) * 2;
    if (s[1] != 0.0f) top = fmaxf(top, s[0]);
  }
  top = wave_max(top);
  float total = 0.0f;
  for (unsigned i = lane; i < p.splits; i += 64) {
    const float* s = p.statistics + (i * rows + row) * 2;
    const float w = s[1] != 0.0f ? __builtin_amdgcn_exp2f(s[0] - top) : 0.0f;
    weights[wave][i] = s[1] != 0.0f ? w : -1.0f;  // below 0: the piece has no key of this row, and wrote no output
    total += w * s[1];
  }
  total = wave_sum(total);
  wave_lds_order();
  for (unsigned d = lane * 4; d < size; d += 256) {
    f32x4 sum = {0, 0, 0, 0};
    for (unsigned i = 0; i < p.splits; ++i) {
      const float w = weights[wave][i];
      if (!(w < 0.0f)) sum += w * *reinterpret_cast<const f32x4*>(p.partial + (i * rows + row) * size + d);
    }
    const f32x4 none = {0, 0, 0, 0};
    *reinterpret_cast<f32x4*>(p.out + token * p.out_token + head * p.out_head + d) = total == 0.0f ? none : sum / total;
  }
}

int check_attention(const tfcc_rocm_paged_attention_desc& d) {
  if (int e = check_cache(d.cache, "paged_attention")) return e;
  TFCC_REQUIRE(d.heads > 0 && d.heads % d.cache.heads == 0, "paged_attention: %u heads over %u cache heads", d.heads, d.cache.heads);
  TFCC_REQUIRE(d.tokens <= 0x7fffffffu && d.batch <= 0x7fffffffu && (uint64_t)d.tokens * d.heads <= 0x7fffffffu, "paged_attention: %u tokens of %u heads", d.tokens, d.heads);
  TFCC_REQUIRE(d.window == 0 || d.causal, "paged_attention: a window without causal");
  TFCC_REQUIRE((uint64_t)d.table_width * d.cache.page_size <= 0x7fffffffu - 4096, "paged_attention: a table of %u pages of %u rows", d.table_width, d.cache.page_size);
  TFCC_REQUIRE(((d.q_token_stride | d.q_head_stride | d.out_token_stride | d.out_head_stride) % 4) == 0 &&
                   ((reinterpret_cast<uintptr_t>(d.q) | reinterpret_cast<uintptr_t>(d.out) | reinterpret_cast<uintptr_t>(d.workspace)) % 16) == 0,
               "paged_attention: q, out or the workspace off 16 bytes");
  return TFCC_ROCM_OK;
}

unsigned most_keys(const tfcc_rocm_paged_attention_desc& d) {
  const unsigned held = d.table_width * d.cache.page_size;
  return d.max_length > 0 && d.max_length < held ? d.max_length : held;
}

PagedAttentionPlan plan_of(const tfcc_rocm_paged_attention_desc& d) {
  return paged_attention_plan(d.tokens, d.batch, d.heads / d.cache.heads, d.cache.heads, most_keys(d), d.causal, d.window);
}

size_t workspace_of(const tfcc_rocm_paged_attention_desc& d, const PagedAttentionPlan& plan) {
  return plan.splits == 1 ? 0 : (size_t)plan.splits * d.tokens * d.heads * (d.cache.size + 2) * sizeof(float);
}

}  // namespace
}  // namespace tfcc_rocm

using namespace tfcc_rocm;

extern "C" {

size_t tfcc_rocm_paged_attention_workspace(const tfcc_rocm_paged_attention_desc* desc) {
  if (desc == nullptr || check_attention(*desc) != TFCC_ROCM_OK || desc->tokens == 0 || desc->batch == 0) return 0;
  return workspace_of(*desc, plan_of(*desc));
}

int tfcc_rocm_paged_attention_f32(void* stream, const tfcc_rocm_paged_attention_desc* desc) {
  TFCC_REQUIRE(desc != nullptr, "paged_attention: null descriptor");
  const tfcc_rocm_paged_attention_desc& d = *desc;
  if (int e = check_attention(d)) return e;
  if (d.tokens == 0 || d.batch == 0) return TFCC_ROCM_OK;
  TFCC_REQUIRE(d.q && d.out && d.starts && d.lengths && (d.table || d.table_width == 0), "paged_attention: null argument");
  const PagedAttentionPlan plan = plan_of(d);
  const size_t needs = workspace_of(d, plan);
  TFCC_REQUIRE(needs == 0 || (d.workspace != nullptr && d.workspace_bytes >= needs), "paged_attention: a workspace of %zu bytes where %zu are needed",
               d.workspace == nullptr ? (size_t)0 : d.workspace_bytes, needs);
  const uint64_t groups = (uint64_t)plan.tiles * plan.splits * d.cache.heads;
  TFCC_REQUIRE(groups <= 0x7fffffffu / kThreads, "paged_attention: %u tiles of rows", plan.tiles);
  AttentionArgs a{};
  a.cache = view_of(d.cache);
  a.q = d.q;
  a.out = d.out;
  a.q_token = d.q_token_stride;
  a.q_head = d.q_head_stride;
  a.out_token = d.out_token_stride;
  a.out_head = d.out_head_stride;
  a.tokens = d.tokens;
  a.batch = d.batch;
  a.starts = d.starts;
  a.lengths = d.lengths;
  a.table = d.table;
  a.table_stride = d.table_stride;
  a.table_width = d.table_width;
  a.max_length = most_keys(d);
  a.scale = d.scale * 1.44269504088896341f;
  a.causal = d.causal;
  a.window = d.window;
  a.group = Divisor::of(d.heads / d.cache.heads);
  a.cache_heads = Divisor::of(d.cache.heads);
  a.pieces = Divisor::of(plan.splits);
  a.splits = plan.splits;
  a.split_keys = plan.split_keys;
  a.statistics = static_cast<float*>(d.workspace) + (size_t)plan.splits * d.tokens * d.heads * d.cache.size;
  a.partial = static_cast<float*>(d.workspace);
  const hipStream_t s = as_stream(stream);
  const dim3 grid((unsigned)groups);
  const auto start = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, a); };
  const tfcc_rocm_paged_cache& c = d.cache;
  const unsigned blocks = (c.size + 63) / 64;
  if (c.type == TFCC_ROCM_S8) {
    const bool fast = c.page_size % 16 == 0 && c.size % 16 == 0 && (c.page_stride | c.head_stride | c.row_stride) % 16 == 0 && c.scale_row_stride == 1 &&
                      (c.scale_page_stride | c.scale_head_stride) % 4 == 0 &&
                      (reinterpret_cast<uintptr_t>(c.keys) | reinterpret_cast<uintptr_t>(c.values) | reinterpret_cast<uintptr_t>(c.key_scales) |
                       reinterpret_cast<uintptr_t>(c.value_scales)) % 16 == 0;
    if (blocks == 1) start(fast ? attention_s8_kernel<1, true> : attention_s8_kernel<1, false>);
    else if (blocks == 2) start(fast ? attention_s8_kernel<2, true> : attention_s8_kernel<2, false>);
    else if (blocks == 3) start(fast ? attention_s8_kernel<3, true> : attention_s8_kernel<3, false>);
    else start(fast ? attention_s8_kernel<4, true> : attention_s8_kernel<4, false>);
  } else {
    const bool uniform = c.page_size % 16 == 0;
    if (blocks == 1) start(uniform ? attention_f32_kernel<1, true> : attention_f32_kernel<1, false>);
    else if (blocks == 2) start(uniform ? attention_f32_kernel<2, true> : attention_f32_kernel<2, false>);
    else if (blocks == 3) start(uniform ? attention_f32_kernel<3, true> : attention_f32_kernel<3, false>);
    else start(uniform ? attention_f32_kernel<4, true> : attention_f32_kernel<4, false>);
  }
  if (int e = check_launch("paged_attention")) return e;
  if (plan.splits > 1) {
    const unsigned rows = d.tokens * d.heads;
    hipLaunchKernelGGL(join_pieces_kernel, dim3((rows + kWaves - 1) / kWaves), dim3(kThreads), 0, s, a);
    return check_launch("paged_attention join");
  }
  return TFCC_ROCM_OK;
}

}  // extern "C"
