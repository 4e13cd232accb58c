// tfcc::rocm::generation: norms, caches of 4-bit integers, copies inside a cache and shaped scores.  Refusals on a host-memory device, and known answers on
// the ROCm device.
// usage: serving_tests cpu | gpu
#include <cmath>
#include <cstdio>
#include <limits>
#include <memory>
#include <string>

#include "tfcc_rocm_device.h"

using namespace tfcc;
using namespace tfcc::rocm::generation;

static int failures = 0;
#define EXPECT(cond)                                         \
  do {                                                       \
    if (!(cond)) {                                           \
      ++failures;                                            \
      std::printf("FAIL line %d: %s\n", __LINE__, #cond);    \
    }                                                        \
  } while (0)
#define REFUSED(expr, TYPE)                                                       \
  do {                                                                            \
    bool caught = false;                                                          \
    try {                                                                         \
      (void)(expr);                                                               \
    } catch (const TYPE&) {                                                       \
      caught = true;                                                              \
    }                                                                             \
    if (!caught) {                                                                \
      ++failures;                                                                 \
      std::printf("FAIL line %d: %s did not throw %s\n", __LINE__, #expr, #TYPE); \
    }                                                                             \
  } while (0)

static void refusals(bool gpu) {
  Variable<float> x({3, 8}), other({2, 8}), weight({8}), short_weight({7}), three({3}), two({2});
  Variable<int32_t> sums({3, 8});
  Variable<uint8_t> steps({3, 8});
  const float nan = std::numeric_limits<float>::quiet_NaN();
  REFUSED(rms_norm(x, short_weight, 1e-6f), InvalidArgumentError);
  REFUSED(rms_norm(x, x, 1e-6f), InvalidArgumentError);
  REFUSED(rms_norm(x, weight, 1e-6f, &other), InvalidArgumentError);
  REFUSED(rms_norm(x, weight, -1.0f), InvalidArgumentError);
  REFUSED(rms_norm_quantized(x, short_weight, 1e-6f), InvalidArgumentError);
  REFUSED(rms_norm_quantized(x, weight, 1e-6f, &weight), InvalidArgumentError);
  REFUSED(rms_norm_quantized(x, weight, nan), InvalidArgumentError);
  REFUSED(dequantize_rows(sums, two), InvalidArgumentError);
  REFUSED(dequantize_rows(steps, three, 128, &three), InvalidArgumentError);
  REFUSED(PagedCache<Int4>(0, 2, 16, 8), InvalidArgumentError);
  REFUSED(PagedCache<Int4>(2, 2, 16, 7), InvalidArgumentError);
  REFUSED(PagedCache<Int4>(2, 2, 16, 1), InvalidArgumentError);
  REFUSED(PagedCache<Int4>(1u << 16, 1u << 16, 1, 16), InvalidArgumentError);  // 2^35 bytes
  if (!gpu) {
    REFUSED(rms_norm(x, weight, 1e-6f), NotImplementedError);
    REFUSED(rms_norm_quantized(x, weight, 1e-6f), NotImplementedError);
    REFUSED(dequantize_rows(sums, three), NotImplementedError);
    REFUSED(PagedCache<Int4>(1, 2, 16, 16), NotImplementedError);
    return;
  }
  PagedCache<Int4> cache(2, 2, 16, 16);
  Variable<float> q({3, 4, 16}), k({3, 2, 16}), narrow({3, 2, 8}), slopes({4}), few({3});
  Variable<int32_t> table({1, 2}), starts({2}), lengths({1}), pair({2}), single({1}), square({2, 2});
  REFUSED(cache_write(cache, narrow, narrow, sums), InvalidArgumentError);
  REFUSED(cache_write(cache, narrow, narrow, lengths), InvalidArgumentError);
  REFUSED(cache_copy(cache, square, pair), InvalidArgumentError);
  REFUSED(cache_copy(cache, pair, single), InvalidArgumentError);
  REFUSED(cache_copy(cache, pair, pair, &single), InvalidArgumentError);
  const auto attend = [&](const ScoreShape& shape, bool causal = true, unsigned window = 0) {
    return paged_attention(q, cache, table, starts, lengths, 1.0f, causal, window, 0, shape);
  };
  REFUSED(attend({-1.0f, nullptr, nullptr}), InvalidArgumentError);
  REFUSED(attend({nan, nullptr, nullptr}), InvalidArgumentError);
  REFUSED(attend({std::numeric_limits<float>::infinity(), nullptr, nullptr}), InvalidArgumentError);
  REFUSED(attend({0.0f, &few, nullptr}), InvalidArgumentError);
  REFUSED(attend({0.0f, nullptr, &pair}), InvalidArgumentError);
  REFUSED(attend({0.0f, nullptr, &single}, false), InvalidArgumentError);
  REFUSED(attend({0.0f, nullptr, &single}, true, 3), InvalidArgumentError);
  PagedCache<Int4> odd(2, 2, 16, 12);  // heads that are no multiple of sixteen values
  Variable<float> k12({3, 2, 12});
  Variable<int32_t> slots({3});
  REFUSED(cache_write(odd, k12, k12, slots), ROCMRuntimeError);
  // what was moved out of, or replaced, names no memory
  const auto lost = [&](PagedCache<Int4>& c) {
    REFUSED(cache_write(c, k, k, slots), InvalidArgumentError);
    REFUSED(cache_copy(c, single, single), InvalidArgumentError);
    REFUSED(cache_read(c, table, starts, 1), InvalidArgumentError);
    REFUSED(paged_attention(q, c, table, starts, lengths, 1.0f), InvalidArgumentError);
  };
  for (int which = 0; which < 3; ++which) {
    PagedCache<Int4> c(2, 2, 16, 16);
    if (which == 0) c.values = Variable<uint8_t>({2, 2, 16, 4});
    if (which == 1) c.keyScales = Variable<float>({1, 2, 16});
    if (which == 2) c.valueScales = Variable<float>();
    lost(c);
  }
  PagedCache<Int4> taken(std::move(cache));
  lost(cache);
}

static void norms() {
  const unsigned rows = 37, width = 256;
  std::vector<float> x(rows * width), half(x.size()), weight(width), factors(rows), columns(width);
  for (unsigned r = 0; r < rows; ++r)
    for (unsigned j = 0; j < width; ++j) {
      x[r * width + j] = ((r + j) % 3 == 0 ? -2.0f : 2.0f) * static_cast<float>(r + 1);
      half[r * width + j] = 0.5f * x[r * width + j];
    }
  for (unsigned j = 0; j < width; ++j) weight[j] = static_cast<float>(j % 128);
  for (unsigned r = 0; r < rows; ++r) factors[r] = std::ldexp(1.0f, static_cast<int>(r % 9) - 4);
  for (unsigned j = 0; j < width; ++j) columns[j] = std::ldexp(1.0f, static_cast<int>(j % 5) - 2);
  Variable<float> dx = data::set(x, Shape({rows, width})), dhalf = data::set(half, Shape({rows, width})), dw = data::set(weight, Shape({width}));
  Variable<float> out, sum;
  // the root of a row's mean square is its magnitude, so that the results are the weights with the row's signs
  std::tie(out, sum) = rms_norm(dx, dw, 0.0f);
  EXPECT(sum.size() == 0);
  const std::vector<float> y = data::get(out);
  bool same = true;
  for (unsigned i = 0; i < y.size(); ++i) same = same && y[i] == (x[i] < 0 ? -1.0f : 1.0f) * weight[i % width];
  EXPECT(same);
  std::tie(out, sum) = rms_norm(dhalf, dw, 0.0f, &dhalf);
  EXPECT(data::get(out) == y && data::get(sum) == x);
  const QuantizedRows quantized = rms_norm_quantized(dhalf, dw, 0.0f, &dhalf);
  const std::vector<uint8_t> steps = data::get(quantized.steps);
  const std::vector<int32_t> sums = data::get(quantized.sums);
  EXPECT(data::get(quantized.sum) == x && data::get(quantized.scales) == std::vector<float>(rows, 1.0f) && quantized.scales.shape() == Shape({rows}));
  same = true;
  for (unsigned r = 0; r < rows; ++r) {
    int total = 0;
    for (unsigned j = 0; j < width; ++j) {
      same = same && static_cast<float>(steps[r * width + j]) - 128.0f == y[r * width + j];
      total += steps[r * width + j];
    }
    same = same && total == sums[r];
  }
  EXPECT(same);
  EXPECT(data::get(dequantize_rows(quantized.steps, quantized.scales, 128)) == y);
  // powers of two: every product is exact
  std::vector<int32_t> n(x.size());
  for (unsigned i = 0; i < n.size(); ++i) n[i] = static_cast<int32_t>(i * 2654435761u >> 10) - (1 << 21);
  Variable<float> dc = data::set(columns, Shape({width}));
  const std::vector<float> back = data::get(dequantize_rows(data::set(n, Shape({rows, width})), data::set(factors, Shape({rows})), -5, &dc));
  same = true;
  for (unsigned i = 0; i < n.size(); ++i) same = same && back[i] == static_cast<float>(n[i] + 5) * factors[i / width] * columns[i % width];
  EXPECT(same);
  // a row alone
  std::tie(out, sum) = rms_norm(dw, dw, 1.0f);
  EXPECT(out.shape() == dw.shape());
  EXPECT(rms_norm_quantized(dw, dw, 1.0f).scales.size() == 1);
}

// Two answers to one prompt: they share its whole pages, and its last one is copied for the second.
template <class T>
static void forked() {
  const unsigned heads = 2, size = 32, page = 16, tokens = 37;
  PagedCache<T> cache(6, heads, page, size);
  std::vector<float> k(tokens * heads * size), v(k.size());
  for (size_t i = 0; i < k.size(); ++i) {
    k[i] = static_cast<float>(static_cast<int>(i * 2654435761u >> 20) - 2048);
    v[i] = static_cast<float>(static_cast<int>(i * 2246822519u >> 20) - 2048);
  }
  std::vector<int32_t> slots(tokens);
  for (unsigned t = 0; t < tokens; ++t) slots[t] = static_cast<int32_t>(t);
  Variable<int32_t> dslots = data::set(slots, Shape({tokens}));
  cache_write(cache, data::set(k, Shape({tokens, heads, size})), data::set(v, Shape({tokens, heads, size})), dslots);
  const std::vector<int32_t> sources = {32, 33, -1}, destinations = {80, 65, 5}, rows = {5, 2, 9};
  Variable<int32_t> ds = data::set(sources, Shape({3u})), dd = data::set(destinations, Shape({3u})), dr = data::set(rows, Shape({3u}));
  cache_copy(cache, ds, dd, &dr);
  Variable<int32_t> tables = data::set(std::vector<int32_t>{0, 1, 2, 0, 1, 5}, Shape({2u, 3u})), starts = data::set(std::vector<int32_t>{0, 48, 96}, Shape({3u}));
  Variable<float> dk, dv;
  std::tie(dk, dv) = cache_read(cache, tables, starts, 96);
  for (const std::vector<float>& got : {data::get(dk), data::get(dv)}) {
    const size_t half = got.size() / 2;
    EXPECT(std::vector<float>(got.begin(), got.begin() + half) == std::vector<float>(got.begin() + half, got.end()));
    EXPECT(got[half - 1] == 0.0f && got[36 * heads * size + 1] != 0.0f);  // rows behind the fifth are still zeros
  }
  // two rows between other pages, then a whole page
  Variable<int32_t> middle = data::set(std::vector<int32_t>{2, 4}, Shape({2u, 1u})), short_starts = data::set(std::vector<int32_t>{0, 3, 6}, Shape({3u}));
  std::tie(dk, dv) = cache_read(cache, middle, short_starts, 6);
  std::vector<float> got = data::get(dk);
  const size_t row = heads * size;
  EXPECT(std::vector<float>(got.begin() + row, got.begin() + 3 * row) == std::vector<float>(got.begin() + 4 * row, got.end()) && got[3 * row + 1] == 0.0f);
  cache_copy(cache, data::set(std::vector<int32_t>{0}, Shape({1u})), data::set(std::vector<int32_t>{48}, Shape({1u})));
  std::tie(dk, dv) = cache_read(cache, data::set(std::vector<int32_t>{0, 3}, Shape({2u, 1u})), data::set(std::vector<int32_t>{0, 16, 32}, Shape({3u})), 32);
  got = data::get(dv);
  EXPECT(std::vector<float>(got.begin(), got.begin() + 16 * row) == std::vector<float>(got.begin() + 16 * row, got.end()) && got[row - 1] != 0.0f);  // the largest of its row
}

// All values of a key alike, -3 .. 3, so that a score is a multiple of it: the weights are those of a few lines of host arithmetic.
template <class T>
static void shaped() {
  const unsigned heads = 2, group = 3, size = 64, page = 16, pages = 14, tokens = 200;
  PagedCache<T> cache(pages, heads, page, size);
  std::vector<float> k(tokens * heads * size), v(k.size()), q(tokens * heads * group * size, 0.25f);
  for (unsigned t = 0; t < tokens; ++t)
    for (unsigned i = 0; i < heads * size; ++i) {
      k[t * heads * size + i] = static_cast<float>(static_cast<int>(t * 5 % 7) - 3);
      v[t * heads * size + i] = i % size == 0 ? 1.75f : 0.25f * static_cast<float>(static_cast<int>((t * 7 + i) % 15) - 7);
    }
  std::vector<int32_t> slots(tokens), table(pages);
  for (unsigned t = 0; t < tokens; ++t) slots[t] = static_cast<int32_t>((pages - 1 - t / page) * page + t % page);
  for (unsigned i = 0; i < pages; ++i) table[i] = static_cast<int32_t>(pages - 1 - i);
  std::vector<float> slopes = {0.5f, 0.25f, 0.0f, 0.0625f, -0.01f, 2.0f};
  Variable<float> dq = data::set(q, Shape({tokens, heads * group, size})), dk = data::set(k, Shape({tokens, heads, size})), dv = data::set(v, Shape({tokens, heads, size}));
  Variable<float> dslopes = data::set(slopes, Shape({heads * group}));
  Variable<int32_t> dtable = data::set(table, Shape({1u, pages})), starts = data::set(std::vector<int32_t>{0, static_cast<int32_t>(tokens)}, Shape({2u}));
  Variable<int32_t> lengths = data::set(std::vector<int32_t>{static_cast<int32_t>(tokens)}, Shape({1u})), prefixes = data::set(std::vector<int32_t>{50}, Shape({1u}));
  cache_write(cache, dk, dv, data::set(slots, Shape({tokens})));
  Variable<float> readK, readV;
  std::tie(readK, readV) = cache_read(cache, dtable, starts, tokens);
  const std::vector<float> gotK = data::get(readK), gotV = data::get(readV);
  double worst = 0;
  for (size_t i = 0; i < k.size(); ++i) worst = std::fmax(worst, std::fmax(std::fabs(gotK[i] - k[i]), std::fabs(gotV[i] - v[i])));
  EXPECT(worst <= (std::is_same<T, int8_t>::value ? 1.75 / 254 + 1e-6 : 1e-6));  // 4 bits hold all of them but for the roundings of a scale and of a product
  for (int which = 0; which < 8; ++which) {
    ScoreShape shape;
    shape.cap = which & 1 ? 2.0f : 0.0f;
    shape.slopes = which & 2 ? &dslopes : nullptr;
    shape.prefixes = which & 4 ? &prefixes : nullptr;
    const std::vector<float> y = data::get(paged_attention(dq, cache, dtable, starts, lengths, 0.125f, true, 0, 0, shape));
    worst = 0;
    for (unsigned t = 0; t < tokens; t += 3)
      for (unsigned h = 0; h < heads * group; ++h) {
        const unsigned seen = which & 4 && t < 50 ? 50 : t + 1;
        std::vector<double> w(seen);
        double top = -1e300, total = 0;
        for (unsigned s = 0; s < seen; ++s) {
          double x = 0;
          for (unsigned d = 0; d < size; ++d) x += 0.125 * 0.25 * gotK[(s * heads + h / group) * size + d];
          if (which & 1) x = 2.0 * std::tanh(x / 2.0);
          if (which & 2) x -= slopes[h] * std::fabs(static_cast<double>(t) - s);
          w[s] = x;
          top = std::fmax(top, x);
        }
        for (double& x : w) total += x = std::exp(x - top);
        for (unsigned d = 0; d < size; d += 7) {
          double want = 0;
          for (unsigned s = 0; s < seen; ++s) want += w[s] / total * gotV[(s * heads + h / group) * size + d];
          worst = std::fmax(worst, std::fabs(y[(t * heads * group + h) * size + d] - want));
        }
      }
    // scores of up to 2 x 200 lie 2^-24 of that off, their weights as much, which twice over, with sums of 200, is below 1e-4 of values of up to 1.75
    EXPECT(worst <= 2e-4);
  }
}

int main(int argc, char** argv) {
  const bool gpu = argc > 1 && std::string(argv[1]) == "gpu";
  std::unique_ptr<HostDevice> device;
  std::unique_ptr<HostSession> session;
  if (gpu) {
    initialize_rocm();
  } else {
    device.reset(new HostDevice());
    session.reset(new HostSession(*device));
    Device::setThreadDefault(device.get());
    Session::setThreadDefault(session.get());
  }
  refusals(gpu);
  if (gpu) {
    norms();
    forked<float>();
    forked<int8_t>();
    forked<Int4>();
    shaped<float>();
    shaped<int8_t>();
    shaped<Int4>();
  } else {
    Session::setThreadDefault(nullptr);
    Device::setThreadDefault(nullptr);
  }
  if (failures == 0) std::printf("serving: all passed\n");
  return failures != 0;
}
