// Attention over a paged cache: the calls, how they are dealt out, and the launch that joins pieces of the keys.
#include "paged_attention.hpp"

#include <algorithm>

namespace tfcc_rocm {
namespace {

constexpr int kThreads = 256;  // of the launch that joins pieces

// The pieces of a row joined: a workgroup to 64 values of a row, whose threads take four values each of one in every kShares pieces.  Bound: latency, so the first loads of
// pieces are under way before their weights are known (float32, 2 sequences of 10335, 8 heads over 1 of 256, 81 pieces: 27.1 us in all, with a workgroup to a row, weights first, 32.4; int8, one of 100000, 8 heads over 1 of 128: 19.8 and 23.2).
constexpr unsigned kShares = kThreads / 16, kAtOnce = 8;
__global__ __launch_bounds__(kThreads) void join_pieces_kernel(AttentionArgs p) {
  __shared__ float weights[kAttentionMostSplits];
  __shared__ __align__(16) f32x4 sums[kThreads];
  const unsigned lane = threadIdx.x & 63, heads = p.cache.heads * p.group.d, size = p.cache.size;
  const unsigned share = threadIdx.x / 16, d = blockIdx.y * 64 + threadIdx.x % 16 * 4;
  const unsigned long long row = blockIdx.x, rows = (unsigned long long)p.tokens * heads;
  const unsigned token = blockIdx.x / heads, head = blockIdx.x - token * heads;
  if ((int)token >= p.starts[p.batch] || (int)token < p.starts[0]) return;
  const float* const partial = p.partial + row * size + (d < size ? d : 0);
  f32x2 statistics[kAttentionMostSplits / 64];
#pragma unroll
  for (unsigned k = 0; k < kAttentionMostSplits / 64; ++k) {
    const unsigned i = lane + 64 * k;
    statistics[k] = f32x2{-INFINITY, 0.0f};
    if (i < p.splits) statistics[k] = *reinterpret_cast<const f32x2*>(p.statistics + (i * rows + row) * 2);
  }
  f32x4 part[kAtOnce];
#pragma unroll
  for (unsigned k = 0; k < kAtOnce; ++k) {
    const unsigned i = share + kShares * k;
    part[k] = f32x4{0, 0, 0, 0};
    if (i < p.splits) part[k] = *reinterpret_cast<const f32x4*>(partial + i * rows * size);
  }
  float top = -INFINITY, total = 0.0f;
#pragma unroll
  for (unsigned k = 0; k < kAttentionMostSplits / 64; ++k) top = fmaxf(top, statistics[k][0]);
  top = wave_max(top);
#pragma unroll
  for (unsigned k = 0; k < kAttentionMostSplits / 64; ++k) {
    const bool none = statistics[k][0] == -INFINITY;  // no such piece, or one without a key of this row
    const float h = none ? 0.0f : half_step(statistics[k][0], top);
    weights[lane + 64 * k] = none ? -1.0f : h * h;  // (all wavefronts write the same)
    total += none ? 0.0f : statistics[k][1] * h * h;
  }
  total = wave_sum(total);
  __syncthreads();
  f32x4 sum = {0, 0, 0, 0};
#pragma unroll
  for (unsigned k = 0; k < kAtOnce; ++k) {
    const float w = weights[share + kShares * k];
    if (!(w < 0.0f)) sum += w * part[k];
  }
  for (unsigned i = share + kShares * kAtOnce; i < p.splits; i += kShares) {
    const float w = weights[i];
    if (!(w < 0.0f)) sum += w * *reinterpret_cast<const f32x4*>(partial + i * rows * size);
  }
  sums[threadIdx.x] = sum;
  __syncthreads();
  if (share == 0 && d < size) {
#pragma unroll
    for (unsigned i = 1; i < kShares; ++i) sum += sums[threadIdx.x + 16 * i];
    const f32x4 none = {0, 0, 0, 0};
    *reinterpret_cast<f32x4*>(p.out + token * p.out_token + head * p.out_head + d) = top == -INFINITY ? none : sum / total;
  }
}

// Few pieces: LANES lanes to a row (at least a quarter of its values), which sum them one after the other.  HBM is its bound where there are many rows
// (10 chunks of 512, 12 heads of 64, two pieces: 12 us, and 77 with a workgroup to a row).
template <unsigned LANES>
__global__ __launch_bounds__(kThreads) void join_few_kernel(AttentionArgs p) {
  const unsigned heads = p.cache.heads * p.group.d, size = p.cache.size, d = threadIdx.x % LANES * 4;
  const unsigned row = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES, rows = p.tokens * heads;
  if (row >= rows || d >= size) return;
  const unsigned token = row / heads, head = row - token * heads;
  if ((int)token >= p.starts[p.batch] || (int)token < p.starts[0]) return;
  const unsigned long long each = (unsigned long long)rows * size;  // of a piece
  const float* const partial = p.partial + (unsigned long long)row * size + d;
  const f32x2* const statistics = reinterpret_cast<const f32x2*>(p.statistics) + row;
  float top = -INFINITY, total = 0.0f;
  f32x4 sum = {0, 0, 0, 0};
  // four pieces' loads at a time; what is summed so far is in units of 2^top
  for (unsigned first = 0; first < p.splits; first += 4) {
    f32x2 held[4];
    f32x4 part[4];
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) {
      const unsigned piece = first + i < p.splits ? first + i : first;
      held[i] = statistics[(unsigned long long)piece * rows];
      part[i] = *reinterpret_cast<const f32x4*>(partial + piece * each);
    }
    const float before = top;
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) top = fmaxf(top, held[i][0]);
    if (before != -INFINITY && before != top) {
      const float h = half_step(before, top);
      total = total * h * h;
      sum *= h * h;
    }
#pragma unroll
    for (unsigned i = 0; i < 4; ++i) {
      if (first + i >= p.splits || held[i][0] == -INFINITY) continue;  // none, or one without a key of this row
      const float h = half_step(held[i][0], top);
      total += held[i][1] * h * h;
      sum += h * h * part[i];
    }
  }
  const f32x4 none = {0, 0, 0, 0};
  *reinterpret_cast<f32x4*>(p.out + token * p.out_token + head * p.out_head + d) = top == -INFINITY ? none : sum / total;
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

// A cache of integers with pages of 16 rows and more whose scales lie in a row; int8: which can be read 16 bytes at a time.
bool wide_reads(const tfcc_rocm_paged_cache& c) {
  return has_scales(c) && c.page_size >= 16 && c.scale_row_stride == 1 && c.row_stride < (1u << 26) &&
         (c.type == TFCC_ROCM_S4 || (c.size % 16 == 0 && (c.page_stride | c.head_stride | c.row_stride) % 16 == 0 &&
                                     (reinterpret_cast<uintptr_t>(c.keys) | reinterpret_cast<uintptr_t>(c.values)) % 16 == 0));
}

// Rows of the tiles that chunks of many tokens may take, 0: none.
unsigned chunk_rows(const tfcc_rocm_paged_cache& c) {
  if (c.page_size < 16 || c.page_size % 4 != 0) return 0;
  if (c.type == TFCC_ROCM_F32) return c.size <= 64 ? 128 : c.size <= 128 ? 256 : 0;
  if (c.type == TFCC_ROCM_S4) return wide_reads(c) && c.size > 64 && c.size <= 128 ? 128 : 0;  // others stay with 16 rows (4 chunks of 1024 over 4096, 12 heads of 64: 114 us, with 128 rows 208; 16 heads over 8 of 256 554, int8 with 128 rows 826)
  return wide_reads(c) ? 128 : 0;
}

PagedAttentionPlan plan_of(const tfcc_rocm_paged_attention_desc& d, bool shaped) {
  return paged_attention_plan(d.tokens, d.batch, d.heads / d.cache.heads, d.cache.heads, d.cache.size, most_keys(d), d.causal, d.window, chunk_rows(d.cache),
                              d.cache.type == TFCC_ROCM_F32, d.cache.type == TFCC_ROCM_S4, shaped);
}

// Checks a call and deals it out; one without tokens or sequences has nothing to deal out.
int plan_call(const tfcc_rocm_paged_attention_desc& d, bool shaped, PagedAttentionPlan& plan) {
  if (int e = check_attention(d)) return e;
  if (d.tokens == 0 || d.batch == 0) return TFCC_ROCM_OK;
  plan = plan_of(d, shaped);
  // a launch takes 2^32 - 1 threads; pieces, whose join has a workgroup for each row, are made of fewer rows than that is for
  const uint64_t groups = (uint64_t)plan.tiles * plan.splits * d.cache.heads;
  TFCC_REQUIRE(groups * plan.waves * 64 <= 0xffffffffu && (plan.splits == 1 || (uint64_t)d.tokens * d.heads * kThreads <= 0xffffffffu),
               "paged_attention: %llu workgroups of %u threads", (unsigned long long)groups, plan.waves * 64);
  return TFCC_ROCM_OK;
}

size_t workspace_of(const tfcc_rocm_paged_attention_desc& d, const PagedAttentionPlan& plan) {
  return plan.splits == 1 ? 0 : (size_t)plan.splits * d.tokens * d.heads * (d.cache.size + 2) * sizeof(float);
}

int attend(void* stream, const tfcc_rocm_paged_attention_desc& d, const tfcc_rocm_attention_scores* scores) {
  PagedAttentionPlan plan;
  if (int e = plan_call(d, scores != nullptr, plan)) return e;
  if (d.tokens == 0 || d.batch == 0) return TFCC_ROCM_OK;
  TFCC_REQUIRE(d.q && d.out && d.starts && d.lengths && (d.table || d.table_width == 0), "paged_attention: null argument");
  const size_t needs = workspace_of(d, plan);
  TFCC_REQUIRE(needs == 0 || (d.workspace != nullptr && d.workspace_bytes >= needs), "paged_attention: a workspace of %zu bytes where %zu are needed",
               d.workspace == nullptr ? (size_t)0 : d.workspace_bytes, needs);
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
  if (attention_longest_first(plan, d.tokens, d.batch, a.max_length, a.window, d.cache.type == TFCC_ROCM_F32)) {
    int shift = 0;
    while (a.max_length >> shift > 16) ++shift;
    a.longest_first = shift + 1;
  }
  a.statistics = static_cast<float*>(d.workspace) + (size_t)plan.splits * d.tokens * d.heads * d.cache.size;
  a.partial = static_cast<float*>(d.workspace);
  const hipStream_t s = as_stream(stream);
  if (scores != nullptr) {
    // caps that no score comes near are none: in the units of log2 they may not be numbers
    a.cap = scores->cap < 1.2676506e30f ? scores->cap * 1.44269504088896341f : 0.0f;
    a.cap_inverse = a.cap > 0.0f ? fminf(1.0f / a.cap, 3.4028234e38f) : 0.0f;
    a.slopes = scores->slopes;
    a.prefixes = scores->prefixes;
    launch_shaped_attention(a, d.cache.type, wide_reads(d.cache), plan, s);
  } else {
    launch_attention<false>(a, d.cache.type, wide_reads(d.cache), plan, s);
  }
  if (int e = check_launch("paged_attention")) return e;
  if (plan.splits > 1) {
    const unsigned rows = d.tokens * d.heads;
    if (!attention_joins_few(plan.splits, rows, a.cache.size)) {
      hipLaunchKernelGGL(join_pieces_kernel, dim3(rows, (a.cache.size + 63) / 64), dim3(kThreads), 0, s, a);
    } else {
      const unsigned lanes = a.cache.size <= 64 ? 16 : a.cache.size <= 128 ? 32 : 64, each = kThreads / lanes;
      hipLaunchKernelGGL((lanes == 16 ? join_few_kernel<16> : lanes == 32 ? join_few_kernel<32> : join_few_kernel<64>), dim3((rows + each - 1) / each), dim3(kThreads), 0, s, a);
    }
    return check_launch("paged_attention join");
  }
  return TFCC_ROCM_OK;
}

}  // namespace
}  // namespace tfcc_rocm

using namespace tfcc_rocm;

extern "C" {

size_t tfcc_rocm_paged_attention_workspace(const tfcc_rocm_paged_attention_desc* desc) {
  if (desc == nullptr) return 0;
  size_t needs = 0;
  for (const bool shaped : {false, true}) {  // one workspace is for both calls
    PagedAttentionPlan plan;
    if (plan_call(*desc, shaped, plan) != TFCC_ROCM_OK || desc->tokens == 0 || desc->batch == 0) return 0;
    needs = std::max(needs, workspace_of(*desc, plan));
  }
  return needs;
}

int tfcc_rocm_paged_attention_f32(void* stream, const tfcc_rocm_paged_attention_desc* desc) {
  TFCC_REQUIRE(desc != nullptr, "paged_attention: null descriptor");
  return attend(stream, *desc, nullptr);
}

int tfcc_rocm_paged_attention_scores_f32(void* stream, const tfcc_rocm_paged_attention_desc* desc, const tfcc_rocm_attention_scores* scores) {
  TFCC_REQUIRE(desc != nullptr && scores != nullptr, "paged_attention: null descriptor");
  const tfcc_rocm_attention_scores& s = *scores;
  TFCC_REQUIRE(s.cap >= 0.0f && s.cap <= 3.4028234e38f, "paged_attention: a cap of %g", s.cap);
  TFCC_REQUIRE(s.prefixes == nullptr || (desc->causal && desc->window == 0), "paged_attention: a prefix with a window or without causal");
  return attend(stream, *desc, s.cap > 0.0f || s.slopes != nullptr || s.prefixes != nullptr ? scores : nullptr);
}

}  // extern "C"
