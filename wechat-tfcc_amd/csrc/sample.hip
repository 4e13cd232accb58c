// One token for each row of logits: temperature, top-k, top-p, min-p and a given random number.
//
// Weights exp((x - max) / temperature) are formed in 64 bits and summed as integers of 2^-shift of the largest one.  Sums of integers
// do not depend on their order, so a row's token does not either, however the row is shared out; and a token is decided at borders
// between sums of up to a million weights, where float32 sums would choose a neighbour now and then.
//
// The kept tokens are the first of the order of falling logits, equal ones by position: those down to one of them, the border.  Four
// launches find it, all but the last with several workgroups to a row, since a row on one CU would be bound by that CU's vector unit:
//   tops    the largest and the smallest logit
//   bins    2048 bins of equal width below the largest: counts where top-k is asked for, else sums of weights for top-p
//   runs    the bin that holds the border is found from those; what lies above it is summed up in runs of 1024 positions, the
//           bin's own tokens (for top-k all down to it) are listed
//   pick    the list is sorted, the border found in it, the kept weights summed, and the token looked up in its run
// (That the last workgroup of `runs` did what `pick` does cost 110 us more than the launch, for 128 rows of 100003: each of them
// has to push the L2 of its part of the GPU out to memory first.)
// 128 rows of 100003 with top-p and min-p take 12 + 23 + 26 + 11 us, of which the first is bound by HBM, the two in the middle by the vector
// unit (about 40 operations of four cycles a logit, half of them in 64 bits), the last by the latency of what it does one after another,
// and so are all four for a single row of 32000: 4 + 5 + 8 + 7.
// A bin of more tokens than the list holds - a vocabulary of equal logits, top-k of thousands, top-k at low temperatures, whose last bin holds all
// from 32 temperatures below the largest on - goes a slower way there: eight bits of the logits' order at a time over the whole row (k = 50, 128 rows of
// 100003: 57 us at a temperature of 0.7, 101 at 0.3, 739 at 0.2).
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
  unsigned parts, runs;      // workgroups, and runs of positions, of a row
  unsigned char* workspace;  // `bytes` for each row
  u64 bytes;
};

constexpr unsigned kSampleThreads = 256, kSampleWaves = kSampleThreads / 64;
constexpr unsigned kBins = 2048, kList = 4096, kListOfPart = 2048, kRun = 1024, kMostParts = 256;
constexpr float kBinsOfUnit = 64.0f;  // bins of one e-folding of the weights
constexpr unsigned kNoToken = 0x007fffffu;  // the key of -infinity; that of a NaN is below

// Order of logits as unsigned integers; both zeros are one.
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);
  return x != x ? 0u : (u & 0x80000000u ? ~u : u | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// 2^(j / 32), to the nearest
__constant__ double kPowers[32] = {
    1, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.6457554781539649,
    1.681792830507429, 1.7186192981224779, 1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};

// What the weights of a row's logits follow from.  exp((x - top) / temperature) * 2^shift is 2^(e + shift) 2^(j / 32) e^f with |f| <= ln 2 / 64
// and the Taylor polynomial of e^f to the fifth power, whose rest is below 3e-15 of it; the 32 powers, with 2^shift in them, lie in LDS.
// Below `cutoff` a weight is less than 2^-2, the integer 0: it is taken for 0, and so is that of a NaN or of -infinity.  From there on e is -64 or more.
struct Row {
  float top, slope, cutoff;
  double steps;  // of ln 2 / 32 in a logit
  int shift;
  const double* powers;
  __device__ __forceinline__ double weight(float x) const {
    // (infinity less infinity is no number, of which the smaller of it and 0 is 0)
    const double t = fmin((double)x - (double)top, 0.0) * steps;
    const double m = t + 6755399441055744.0;  // 1.5 * 2^52: the nearest integer is in the low bits
    const int i = (int)(unsigned)(u64)__double_as_longlong(m);
    const double f = (t - (m - 6755399441055744.0)) * 0.021660849392498290195;
    double e = fma(f, 1.0 / 120, 1.0 / 24);
    e = fma(e, f, 1.0 / 6);
    e = fma(e, f, 0.5);
    e = fma(e, f, 1.0);
    e = fma(e, f, 1.0);
    const double w = ldexp(e * powers[i & 31], i >> 5);
    return x >= cutoff ? w : 0.0;  // (what is formed for others is anything)
  }
};
__device__ Row row_of(float top, float temperature, int shift, double* powers) {  // powers: 32 in LDS, filled here; the caller waits
  if (threadIdx.x < 32) powers[threadIdx.x] = ldexp(kPowers[threadIdx.x], shift);
  const double slope = 1.0 / (double)temperature, least = -0.6931471805599453 * (shift + 2);
  // the lowest float whose weight is 2^-2 or more: the one below may be any number of e-foldings away
  float cutoff = top == INFINITY ? INFINITY : fmaxf((float)fmax((double)top + least / slope, -3.4028234663852886e38), -3.402823466e38f);
  if (((double)cutoff - (double)top) * slope < least) cutoff = value_of(key_of(cutoff) + 1);
  return {top, (float)slope, cutoff, slope * 46.166241308446828384, shift, powers};
}
// to the nearest integer, below 2^52
__device__ __forceinline__ u64 integer_of(double w) { return (u64)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull; }

// v of the lane that a data-parallel move names, `otherwise` where there is none.
template <int CONTROL, int ROWS>
__device__ __forceinline__ u64 moved(u64 v, u64 otherwise) {
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp((int)(unsigned)otherwise, (int)(unsigned)v, CONTROL, ROWS, 0xf, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp((int)(unsigned)(otherwise >> 32), (int)(unsigned)(v >> 32), CONTROL, ROWS, 0xf, false);
  return (u64)hi << 32 | lo;
}
// join over the lanes up to this one: 1, 2, 4 and 8 lanes along the rows of 16, then the last lane of a row to the next, then of the
// lower half to the upper.  (Through the LDS crossbar a step takes six times as long.)
template <class F>
__device__ __forceinline__ u64 wave_scan64(u64 v, F join) {
  v = join(v, moved<0x111, 0xf>(v, 0));
  v = join(v, moved<0x112, 0xf>(v, 0));
  v = join(v, moved<0x114, 0xf>(v, 0));
  v = join(v, moved<0x118, 0xf>(v, 0));
  v = join(v, moved<0x142, 0xa>(v, 0));
  v = join(v, moved<0x143, 0xc>(v, 0));
  return v;
}
__device__ __forceinline__ u64 lane_63(u64 v) {
  const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, 63), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), 63);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 add64(u64 a, u64 b) { return a + b; }
__device__ __forceinline__ u64 max64(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 wave_sum64(u64 v) { return lane_63(wave_scan64(v, add64)); }
__device__ __forceinline__ u64 wave_max64(u64 v) { return lane_63(wave_scan64(v, max64)); }

struct Shared {
  unsigned counts[256];
  u64 weights[256];
  u64 totals[kSampleWaves];
  unsigned digit;
  u64 above;
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
  const u64 upto = wave_scan64(mine, add64) + start;
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

// The weight that top-p of `all` asks for.
__device__ __forceinline__ u64 reach_of(float top_p, u64 all) {
  if (!(top_p < 1.0f)) return all;
  const u64 target = top_p > 0.0f ? (u64)ceil((double)top_p * (double)all) : 1;
  return target < 1 ? 1 : target > all ? all : target;
}

// What a row asks for.  All of it is loaded at once, from the random numbers where there is nothing to load: a load after another
// is a microsecond.
struct Wishes {
  float temperature, top_p, min_p, random;
  int top_k;
  double least;  // of a kept weight
};
__device__ __forceinline__ Wishes wishes_of(const SampleArgs& p, unsigned r) {
  const float temperature = (p.temperature ? p.temperature : p.random)[r], top_p = (p.top_p ? p.top_p : p.random)[r];
  const float min_p = (p.min_p ? p.min_p : p.random)[r], random = p.random[r];
  const int top_k = (p.top_k ? p.top_k : reinterpret_cast<const int*>(p.random))[r];
  return {p.temperature ? temperature : 1.0f, p.top_p ? top_p : 1.0f, p.min_p ? min_p : 0.0f, random, p.top_k ? top_k : 0,
          ldexp(fmin(p.min_p ? (double)min_p : 0.0, 1.0), p.shift)};
}

// The whole of a row by one workgroup.
__device__ void choose_slowly(const SampleArgs& p, unsigned r, const Wishes& wishes, const Row& row, Shared& s) {
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  const float* x = p.logits + r * p.row_stride;
  Border border{kNoToken + 1, ~0ull};
  u64 total = 0;
  const int k = wishes.top_k;
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
  if (wishes.top_p < 1.0f) {
    border = find_border<true>(x, p.length, row, reach_of(wishes.top_p, total), s, total);
  }
  if (border.key <= kNoToken) border = {kNoToken + 1, ~0ull};
  const double least = wishes.least;
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
  u64 target = wishes.random > 0.0f ? (u64)((double)wishes.random * (double)sum) : 0;
  if (target >= sum) target = sum - 1;
  if (target < before || target >= before + mine) return;  // the token is another wavefront's
  seen = seen0;
  for (unsigned base = first; base < first + run; base += 64) {
    const u64 w = kept(base + lane, seen);
    const u64 upto = wave_scan64(w, add64) + before;
    const u64 past = __ballot(upto > target);
    if (past != 0) {
      if (lane == (unsigned)__builtin_ctzll(past)) {
        p.tokens[r] = base + lane;
        if (p.probabilities) p.probabilities[r] = (float)(row.weight(x[base + lane]) / (double)sum);
      }
      return;
    }
    before = lane_63(upto);
  }
}

// Where a row's border is to be looked for: `bin` (kBins: nowhere, everything is above), what the bins above it hold, and what
// has to be reached, both in counts or in weights.
struct Goal {
  u64 above, target;
  u64 bin;
};

// What the launches hand on for a row.
struct RowSpace {
  u64* weights;      // [kBins]
  u64* list;         // [kList], sort_key()s
  u64* runs;         // [runs]
  u64* tops;         // [parts], sort_key()s
  unsigned* counts;  // [kBins]
  unsigned* lows;    // [parts], keys
  unsigned* listed;  // how many are in the list, or would be
  Goal* goal;
};
u64 space_bytes(unsigned parts, unsigned runs) {
  return ((kBins + kList + 3 + (u64)runs + parts) * 8 + (kBins + (u64)parts + 1) * 4 + 15) / 16 * 16;
}
__device__ RowSpace space_of(const SampleArgs& p, unsigned row) {
  RowSpace s;
  s.weights = reinterpret_cast<u64*>(p.workspace + row * p.bytes);
  s.list = s.weights + kBins;
  s.runs = s.list + kList;
  s.tops = s.runs + p.runs;
  s.goal = reinterpret_cast<Goal*>(s.tops + p.parts);
  s.counts = reinterpret_cast<unsigned*>(s.goal + 1);
  s.lows = s.counts + kBins;
  s.listed = s.lows + p.parts;
  return s;
}

// Falling logits, then rising positions, as falling integers.
__device__ __forceinline__ u64 sort_key(unsigned key, unsigned position) { return (u64)key << 32 | (unsigned)~position; }

struct alignas(4) Four { float v[4]; };
// Four neighbours of a row, NaN behind its end.
__device__ __forceinline__ Four four_at(const float* x, unsigned at, unsigned length) {
  Four f;
  if (at + 4 <= length) {
    f = *reinterpret_cast<const Four*>(x + at);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = at + i < length ? x[at + i] : NAN;
  }
  return f;
}

// A lane's part of a run, loaded a run ahead: with one load on its way a wavefront would wait longer than it works.
struct Ahead {
  Four f[4];
};
__device__ __forceinline__ Ahead run_at(const float* x, unsigned run, unsigned length) {
  Ahead a;
  const unsigned at = run * kRun + 4 * (threadIdx.x & 63);
  if ((run + 1) * kRun <= length) {  // the same for the wavefront
#pragma unroll
    for (int j = 0; j < 4; ++j) a.f[j] = *reinterpret_cast<const Four*>(x + at + 256 * j);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) a.f[j] = four_at(x, at + 256 * j, length);
  }
  return a;
}

// Runs [first, behind) of a wavefront.
struct Share {
  unsigned first, behind;
};
__device__ __forceinline__ Share share_of(const SampleArgs& p, unsigned part, unsigned wave) {
  const unsigned each = (p.runs + p.parts * kSampleWaves - 1) / (p.parts * kSampleWaves), first = (part * kSampleWaves + wave) * each;
  return {first < p.runs ? first : p.runs, first + each < p.runs ? first + each : p.runs};
}

__global__ __launch_bounds__(kSampleThreads) void sample_tops_kernel(SampleArgs p) {
  __shared__ u64 tops[kSampleWaves];
  __shared__ unsigned lows[kSampleWaves];
  const unsigned r = blockIdx.x / p.parts, part = blockIdx.x - r * p.parts, lane = threadIdx.x & 63;
  const unsigned wave = (unsigned)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64));
  const RowSpace space = space_of(p, r);
  const float* x = p.logits + r * p.row_stride;
  for (unsigned i = part * kSampleThreads + threadIdx.x; i < kBins; i += p.parts * kSampleThreads) {
    space.weights[i] = 0;
    space.counts[i] = 0;
  }
  if (part == 0 && threadIdx.x == 0) *space.listed = 0;
  u64 top = 0;
  unsigned low = ~0u;
  const Share share = share_of(p, part, wave);
  for (unsigned base = share.first * kRun; base < share.behind * kRun; base += 256) {
    const unsigned at = base + 4 * lane;
    const Four f = four_at(x, at, p.length);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned key = key_of(f.v[i]);
      const u64 k = sort_key(key, at + i);
      top = top > k ? top : k;
      low = key > kNoToken && key < low ? key : low;
    }
  }
  top = wave_max64(top);
  low = ~(unsigned)wave_max64(~low);
  if (lane == 0) {
    tops[wave] = top;
    lows[wave] = low;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (unsigned w = 1; w < kSampleWaves; ++w) {
      top = top > tops[w] ? top : tops[w];
      low = low < lows[w] ? low : lows[w];
    }
    space.tops[part] = top;
    space.lows[part] = low;
  }
}

// A row's largest logit, its position and what follows from them; the same in every wavefront.
struct Head {
  u64 top;
  Row row;
  float bins_of_logit;  // bins of a difference of one
  bool by_count, by_weight;
  int top_k;
  float top_p;
  bool greedy;
};
__device__ Head head_of(const SampleArgs& p, const RowSpace& space, const Wishes& wishes, double* powers) {
  Head h;
  const unsigned lane = threadIdx.x & 63;
  u64 top = 0;
  unsigned low = ~0u;
#pragma unroll 1
  for (unsigned i = lane; i < p.parts; i += 64) {
    const u64 t = space.tops[i];
    const unsigned l = space.lows[i];
    top = top > t ? top : t;
    low = low < l ? low : l;
  }
  h.top = wave_max64(top);
  low = ~(unsigned)wave_max64(~low);
  h.greedy = !(wishes.temperature > 0.0f);
  h.row = row_of(value_of((unsigned)(h.top >> 32)), wishes.temperature, p.shift, powers);
  h.top_k = wishes.top_k;
  h.top_p = wishes.top_p;
  h.by_count = h.top_k > 0 && (unsigned)h.top_k < p.length;
  h.by_weight = !h.by_count && h.top_p < 1.0f;
  // 64 bins of an e-folding reach down to e^-32; narrower ones where the smallest logit is not so far below
  const float span = h.row.top - value_of(low), wide = h.row.slope * kBinsOfUnit, all = (kBins - 1) / span;
  h.bins_of_logit = all > wide && all < 1e30f ? all : wide;
  return h;
}
// Falls with the logit: a rounded difference times a factor, cut off.  What is not a number, between infinities or for a factor of infinity, is
// in the first (the middle one of three of which one is no number is the smaller of the others).
__device__ __forceinline__ unsigned bin_of(const Head& h, float x) {
  return (unsigned)__builtin_amdgcn_fmed3f((h.row.top - x) * h.bins_of_logit, 0.0f, (float)(kBins - 1));
}

__global__ __launch_bounds__(kSampleThreads) void sample_bins_kernel(SampleArgs p) {
  __shared__ u64 weights[kBins];
  __shared__ double powers[32];
  unsigned* const counts = reinterpret_cast<unsigned*>(weights);
  const unsigned r = blockIdx.x / p.parts, part = blockIdx.x - r * p.parts, lane = threadIdx.x & 63;
  const unsigned wave = (unsigned)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64));
  const RowSpace space = space_of(p, r);
  const float* x = p.logits + r * p.row_stride;
  const Share share = share_of(p, part, wave);
  Ahead next = run_at(x, share.first, p.length);
  for (unsigned i = threadIdx.x; i < kBins; i += kSampleThreads) weights[i] = 0;
  const Wishes wishes = wishes_of(p, r);
  const Head h = head_of(p, space, wishes, powers);
  if ((!h.by_count && !h.by_weight) || h.greedy || (unsigned)(h.top >> 32) <= kNoToken) return;
  __syncthreads();
  if (h.by_count) {
    for (unsigned run = share.first; run < share.behind; ++run) {
      const Ahead now = next;
      next = run_at(x, run + 1, p.length);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (now.f[j].v[i] > -INFINITY) atomicAdd(&counts[bin_of(h, now.f[j].v[i])], 1u);
    }
  } else {
    for (unsigned run = share.first; run < share.behind; ++run) {
      const Ahead now = next;
      next = run_at(x, run + 1, p.length);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const Four f = now.f[j];
        u64 w[4];
        unsigned bin[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // all before the first is added: they wait for LDS together
          w[i] = integer_of(h.row.weight(f.v[i]));
          bin[i] = bin_of(h, f.v[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (f.v[i] >= h.row.cutoff) atomicAdd(&weights[bin[i]], w[i]);
      }
    }
  }
  __syncthreads();
  for (unsigned i = threadIdx.x; i < kBins; i += kSampleThreads) {
    if (h.by_count) {
      if (counts[i] != 0) atomicAdd(&space.counts[i], counts[i]);
    } else if (weights[i] != 0) {
      atomicAdd(&space.weights[i], weights[i]);
    }
  }
}

// Sum of what the threads before this one have; `all`: of everybody.
__device__ u64 before_me(u64 mine, u64* totals, u64& all) {
  const unsigned lane = threadIdx.x & 63, wave = threadIdx.x / 64;
  const u64 upto = wave_scan64(mine, add64);
  __syncthreads();
  if (lane == 63) totals[wave] = upto;
  __syncthreads();
  u64 before = upto - mine;
  all = 0;
  for (unsigned w = 0; w < kSampleWaves; ++w) {
    if (w < wave) before += totals[w];
    all += totals[w];
  }
  return before;
}

struct Finding {
  u64 totals[kSampleWaves];
  Goal goal;
};
// A thread's bins, both kinds: asked for before it is known which kind counts.
struct Bins {
  static constexpr unsigned each = kBins / kSampleThreads;
  u64 weights[each];
  unsigned counts[each];
  __device__ __forceinline__ explicit Bins(const RowSpace& space) {
#pragma unroll
    for (unsigned i = 0; i < each; ++i) {
      weights[i] = space.weights[threadIdx.x * each + i];
      counts[i] = space.counts[threadIdx.x * each + i];
    }
  }
};
__device__ Goal goal_of(const Head& h, const Bins& bins, Finding& s) {
  if (threadIdx.x == 0) s.goal = {0, 0, kBins};
  __syncthreads();
  if (!h.by_count && !h.by_weight) return s.goal;
  constexpr unsigned each = Bins::each;
  u64 v[each], mine = 0, all;
#pragma unroll
  for (unsigned i = 0; i < each; ++i) {
    v[i] = h.by_count ? bins.counts[i] : bins.weights[i];
    mine += v[i];
  }
  u64 upto = before_me(mine, s.totals, all);
  u64 target;
  if (h.by_count) {
    target = (u64)h.top_k < all ? (u64)h.top_k : all;
  } else {
    target = reach_of(h.top_p, all);
  }
#pragma unroll
  for (unsigned i = 0; i < each; ++i) {
    if (upto < target && upto + v[i] >= target) s.goal = {upto, target, threadIdx.x * each + i};
    upto += v[i];
  }
  __syncthreads();
  return s.goal;
}

__global__ __launch_bounds__(kSampleThreads) void sample_runs_kernel(SampleArgs p) {
  __shared__ Finding finding;
  __shared__ u64 list[kListOfPart];
  __shared__ float aboves[kSampleWaves][kRun];
  __shared__ double powers[32];
  __shared__ unsigned listed, place_of_list;
  const unsigned r = blockIdx.x / p.parts, part = blockIdx.x - r * p.parts, lane = threadIdx.x & 63;
  const unsigned wave = (unsigned)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64));
  const RowSpace space = space_of(p, r);
  const float* x = p.logits + r * p.row_stride;
  const Share share = share_of(p, part, wave);
  const Bins bins(space);
  Ahead next = run_at(x, share.first, p.length);
  const Wishes wishes = wishes_of(p, r);
  const double least = wishes.least;
  const Head h = head_of(p, space, wishes, powers);
  if ((unsigned)(h.top >> 32) <= kNoToken || h.greedy) return;
  if (threadIdx.x == 0) listed = 0;
  const Goal goal = goal_of(h, bins, finding);
  if (part == 0 && threadIdx.x == 0) *space.goal = goal;
  const unsigned border_bin = (unsigned)goal.bin;
  float* const above = aboves[wave];
  // below this a weight is too small for min-p or nothing at all; what is near it is looked at more closely
  const float enough = wishes.min_p > 0.0f ? fmaxf(h.row.cutoff, h.row.top + (logf(fminf(wishes.min_p, 1.0f)) - 1e-3f) * wishes.temperature * 1.0001f - 1e-6f * fabsf(h.row.top))
                                           : h.row.cutoff;
  for (unsigned run = share.first; run < share.behind; ++run) {
    // The logits that are kept for sure are few for most rows: they are gathered, and a wavefront forms their weights 64 at a time (all formed
    // where a lane wants one: 33 us, gathered 32, with those that min-p leaves out left out before 26).
    unsigned gathered = 0;
    const Ahead now = next;
    next = run_at(x, run + 1, p.length);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const Four f = now.f[j];
      const unsigned at = run * kRun + 256 * j + 4 * lane;
      u64 for_list[4], any = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned bin = bin_of(h, f.v[i]);
        const bool there = f.v[i] > -INFINITY;
        for_list[i] = __ballot(there && (h.by_count ? bin <= border_bin : bin == border_bin));
        any |= for_list[i];
        const u64 inner = __ballot(f.v[i] >= enough && !h.by_count && bin < border_bin);
        if (inner >> lane & 1) above[gathered + __builtin_amdgcn_mbcnt_hi((unsigned)(inner >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)inner, 0))] = f.v[i];
        gathered += __popcll(inner);
      }
      if (any != 0) {
        const unsigned all = __popcll(for_list[0]) + __popcll(for_list[1]) + __popcll(for_list[2]) + __popcll(for_list[3]);
        unsigned place = 0;
        if (lane == 0) place = atomicAdd(&listed, all);
        place = (unsigned)__builtin_amdgcn_readfirstlane((int)place);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned mine = place + __builtin_amdgcn_mbcnt_hi((unsigned)(for_list[i] >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)for_list[i], 0));
          if ((for_list[i] >> lane & 1) && mine < kListOfPart) list[mine] = sort_key(key_of(f.v[i]), at + i);
          place += __popcll(for_list[i]);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    u64 mine = 0;
#pragma unroll 2
    for (unsigned i = lane; i < gathered; i += 64) {
      const double w = h.row.weight(above[i]);
      mine += w >= least ? integer_of(w) : 0;
    }
    mine = wave_sum64(mine);
    if (lane == 0) space.runs[run] = mine;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  __syncthreads();
  const unsigned n = listed;
  if (n == 0) return;
  // more than a list holds: only that matters
  if (threadIdx.x == 0) place_of_list = atomicAdd(space.listed, n <= kListOfPart ? n : kList + 1);
  __syncthreads();
  const unsigned place = place_of_list, fits = n <= kListOfPart && place < kList && n <= kList - place ? n : 0;
#pragma unroll 1
  for (unsigned i = threadIdx.x; i < fits; i += kSampleThreads) space.list[place + i] = list[i];
}

struct Picking {
  u64 list[kList];
  struct alignas(16) {
    u64 key, weight;
  } pairs[kSampleThreads];
  u64 runs[(1u << 20) / kRun];
  u64 totals[kSampleWaves];
  u64 above, all, border;
  unsigned run;
};

// The border among a row's n listed tokens (down to which, in their order, they are kept): more than a thread has one of, so they are
// sorted.  `above`: the weights before them; limit: how many may be kept.
__device__ u64 border_sorted(const Head& h, const Goal& goal, const u64* from, unsigned n, Picking& s) {
  unsigned padded = 2 * kSampleThreads;
  while (padded < n) padded *= 2;
#pragma unroll 1
  for (unsigned i = threadIdx.x; i < padded; i += kSampleThreads) s.list[i] = i < n ? from[i] : 0;
  for (unsigned size = 2; size <= padded; size *= 2)
    for (unsigned step = size / 2; step > 0; step /= 2) {
      __syncthreads();
#pragma unroll 1
      for (unsigned i = threadIdx.x; i < padded / 2; i += kSampleThreads) {
        const unsigned lo = 2 * i - (i & (step - 1)), hi = lo + step;
        const u64 a = s.list[lo], b = s.list[hi];
        if ((a < b) == ((lo & size) == 0)) {
          s.list[lo] = b;
          s.list[hi] = a;
        }
      }
    }
  __syncthreads();
  const unsigned each = padded / kSampleThreads, first = threadIdx.x * each;
  const unsigned limit = h.by_count && goal.target < n ? (unsigned)goal.target : n;
  u64 mine = 0, all;
#pragma unroll 1
  for (unsigned i = first; i < first + each && i < limit; ++i) mine += integer_of(h.row.weight(value_of((unsigned)(s.list[i] >> 32))));
  const u64 base = before_me(mine, s.totals, all);
  u64 upto = base + (h.by_count ? 0 : goal.above);
  const u64 target = h.by_count ? reach_of(h.top_p, all) : goal.target;
  if (threadIdx.x == 0) s.border = s.list[limit - 1];
  __syncthreads();
#pragma unroll 1
  for (unsigned i = first; i < first + each && i < limit; ++i) {
    const u64 next = upto + integer_of(h.row.weight(value_of((unsigned)(s.list[i] >> 32))));
    if (upto < target && next >= target) s.border = s.list[i];
    upto = next;
  }
  __syncthreads();
  return s.border;
}

// The same for at most one token to a thread: each adds up what comes before its own.
__device__ u64 border_counted(const Head& h, const Goal& goal, u64 mine, unsigned n, Picking& s) {
  const u64 weight = threadIdx.x < n ? integer_of(h.row.weight(value_of((unsigned)(mine >> 32)))) : 0;
  s.list[threadIdx.x] = mine;
  s.pairs[threadIdx.x] = {threadIdx.x < n ? mine : 0, weight};
  __syncthreads();
  unsigned before = 0;
  u64 upto = weight;
  for (unsigned i = 0; i < n; i += 8) {  // to a multiple of eight: what is behind the last has key 0
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const u64 key = s.pairs[i + j].key, w = s.pairs[i + j].weight;
      const bool earlier = key > mine;
      before += earlier ? 1 : 0;
      upto += earlier ? w : 0;
    }
  }
  const unsigned limit = h.by_count && goal.target < n ? (unsigned)goal.target : n;
  if (threadIdx.x < n && before == limit - 1) {
    s.border = mine;
    s.all = upto;
  }
  __syncthreads();
  const u64 target = h.by_count ? reach_of(h.top_p, s.all) : goal.target;
  if (!h.by_count) upto += goal.above;
  if (threadIdx.x < n && before < limit && upto - weight < target && upto >= target) s.border = mine;
  __syncthreads();
  return s.border;
}

// One workgroup to a row.
__global__ __launch_bounds__(kSampleThreads) void sample_pick_kernel(SampleArgs p) {
  __shared__ union {
    Picking c;
    Shared slow;
  } shared;
  __shared__ double powers[32];
  Picking& s = shared.c;
  u64* const totals = s.totals;
  const unsigned r = blockIdx.x;
  const RowSpace space = space_of(p, r);
  // all that may be wanted is asked for at once; what was not written is not looked at
  const unsigned n = *space.listed;
  const u64 listed = space.list[threadIdx.x];
  const Goal goal = *space.goal;
  const Wishes wishes = wishes_of(p, r);
  const double least = wishes.least;
  const Head h = head_of(p, space, wishes, powers);
  if ((unsigned)(h.top >> 32) <= kNoToken || h.greedy) {
    if (threadIdx.x == 0) {
      const bool none = (unsigned)(h.top >> 32) <= kNoToken;
      p.tokens[r] = none ? -1ll : (long long)(unsigned)~(unsigned)h.top;
      if (p.probabilities) p.probabilities[r] = none ? 0.0f : 1.0f;
    }
    return;
  }
  if (n > kList) {
    __syncthreads();
    choose_slowly(p, r, wishes, h.row, shared.slow);
    return;
  }
  const float* x = p.logits + r * p.row_stride;
#pragma unroll 1
  for (unsigned i = threadIdx.x; i < p.runs; i += kSampleThreads) s.runs[i] = space.runs[i];
  __syncthreads();
  u64 border = 0;
  if (n > kSampleThreads) border = border_sorted(h, goal, space.list, n, s);
  else if (n > 0) border = border_counted(h, goal, threadIdx.x < n ? listed : 0, n, s);
#pragma unroll 1
  for (unsigned i = threadIdx.x; i < n; i += kSampleThreads) {
    const u64 k = s.list[i];
    const double w = k >= border ? h.row.weight(value_of((unsigned)(k >> 32))) : 0.0;
    if (k >= border && w >= least) atomicAdd(&s.runs[(unsigned)~(unsigned)k / kRun], integer_of(w));
  }
  __syncthreads();
  const unsigned each = (p.runs + kSampleThreads - 1) / kSampleThreads;
  u64 mine = 0, sum;
#pragma unroll 1
  for (unsigned i = threadIdx.x * each; i < (threadIdx.x + 1) * each && i < p.runs; ++i) mine += s.runs[i];
  u64 upto = before_me(mine, totals, sum);
  u64 target = wishes.random > 0.0f ? (u64)((double)wishes.random * (double)sum) : 0;
  if (target >= sum) target = sum - 1;
#pragma unroll 1
  for (unsigned i = threadIdx.x * each; i < (threadIdx.x + 1) * each && i < p.runs; ++i) {
    if (upto <= target && target < upto + s.runs[i]) {
      s.run = i;
      s.above = upto;
    }
    upto += s.runs[i];
  }
  __syncthreads();
  // the token's run: four positions to a thread
  const unsigned at = s.run * kRun + 4 * threadIdx.x;
  const u64 start = s.above;
  const Four f = four_at(x, at, p.length);
  u64 w[4];
  mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned key = key_of(f.v[i]);
    w[i] = 0;
    if (key > kNoToken && sort_key(key, at + i) >= border) {
      const double v = h.row.weight(f.v[i]);
      w[i] = v >= least ? integer_of(v) : 0;
    }
    mine += w[i];
  }
  u64 unused;
  upto = start + before_me(mine, totals, unused);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (upto <= target && target < upto + w[i]) {
      p.tokens[r] = at + i;
      if (p.probabilities) p.probabilities[r] = (float)(h.row.weight(f.v[i]) / (double)sum);
    }
    upto += w[i];
  }
}

// Up to 1024 workgroups in all, which run at the same time; each wavefront has the same number of runs but for the last ones.
unsigned parts_of(unsigned rows, unsigned length) {
  const unsigned long long runs = (length + kRun - 1) / kRun, waves = 1024 * kSampleWaves;
  unsigned long long each = (runs * rows + waves - 1) / waves, least = (runs + kMostParts * kSampleWaves - 1) / (kMostParts * kSampleWaves);
  each = each < least ? least : each;
  return (unsigned)((runs + each * kSampleWaves - 1) / (each * kSampleWaves));
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

size_t tfcc_rocm_sample_workspace(unsigned rows, unsigned length) {
  if (length == 0 || length > (1u << 20)) return 0;
  return (size_t)rows * space_bytes(parts_of(rows, length), (length + kRun - 1) / kRun);
}

int tfcc_rocm_sample_f32(void* stream, const tfcc_rocm_sample_desc* desc) {
  TFCC_REQUIRE(desc != nullptr, "sample: null descriptor");
  const tfcc_rocm_sample_desc& d = *desc;
  TFCC_REQUIRE(d.length > 0 && d.length <= (1u << 20), "sample: rows of %u logits (1 to 2^20)", d.length);
  TFCC_REQUIRE(d.rows <= 0x3fffffu, "sample: %u rows", d.rows);
  if (d.rows == 0) return TFCC_ROCM_OK;
  TFCC_REQUIRE(d.logits && d.random && d.tokens, "sample: null argument");
  const size_t needs = tfcc_rocm_sample_workspace(d.rows, d.length);
  TFCC_REQUIRE(d.workspace != nullptr && d.workspace_bytes >= needs && reinterpret_cast<uintptr_t>(d.workspace) % 16 == 0,
               "sample: a workspace of %zu bytes where %zu are needed, 16-byte aligned", d.workspace == nullptr ? (size_t)0 : d.workspace_bytes, needs);
  const unsigned parts = parts_of(d.rows, d.length), runs = (d.length + kRun - 1) / kRun;
  SampleArgs a{d.logits, d.row_stride, d.rows, d.length, shift_for(d.length), d.random, d.temperature, d.top_k, d.top_p, d.min_p,
               reinterpret_cast<long long*>(d.tokens), d.probabilities, parts, runs, static_cast<unsigned char*>(d.workspace), space_bytes(parts, runs)};
  const dim3 grid(d.rows * parts), block(kSampleThreads);
  const hipStream_t s = as_stream(stream);
  hipLaunchKernelGGL(sample_tops_kernel, grid, block, 0, s, a);
  if (int e = check_launch("sample tops")) return e;
  if (d.top_k || d.top_p) {
    hipLaunchKernelGGL(sample_bins_kernel, grid, block, 0, s, a);
    if (int e = check_launch("sample bins")) return e;
  }
  hipLaunchKernelGGL(sample_runs_kernel, grid, block, 0, s, a);
  if (int e = check_launch("sample runs")) return e;
  hipLaunchKernelGGL(sample_pick_kernel, dim3(d.rows), block, 0, s, a);
  return check_launch("sample pick");
}

}  // extern "C"
