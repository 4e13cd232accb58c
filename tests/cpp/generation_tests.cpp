// tfcc::rocm::generation: refusals on a host-memory device, and known answers of the four operators in a row on the ROCm device.
// usage: generation_tests cpu | gpu
#include <cmath>
#include <cstdio>
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
  Variable<float> q({3, 4, 8}), k({3, 2, 8}), short_k({2, 2, 8}), flat({3, 8}), logits({3, 5}), random({3}), one({1});
  Variable<int32_t> positions({3}), one_position({1});
  Variable<double> frequencies({4}), many({5});
  EXPECT(std::get<0>(rotary_frequencies(8)).size() == 4 && std::get<1>(rotary_frequencies(8)) == 1.0f);
  REFUSED(rotary_frequencies(7), InvalidArgumentError);
  REFUSED(rotary_frequencies(0), InvalidArgumentError);
  REFUSED(rotary(flat, k, positions, frequencies), InvalidArgumentError);
  REFUSED(rotary(q, short_k, positions, frequencies), InvalidArgumentError);
  REFUSED(rotary(q, k, one_position, frequencies), InvalidArgumentError);
  REFUSED(rotary(q, k, positions, many), InvalidArgumentError);
  REFUSED(PagedCache<float>(0, 2, 16, 8), InvalidArgumentError);
  REFUSED(sample(random, random), InvalidArgumentError);
  REFUSED(sample(logits, one), InvalidArgumentError);
  SampleFilters filters;
  filters.topP = &one;
  REFUSED(sample(logits, random, filters), InvalidArgumentError);
  if (!gpu) {
    REFUSED(rotary(q, k, positions, frequencies), NotImplementedError);
    REFUSED(PagedCache<float>(1, 2, 16, 8), NotImplementedError);
    REFUSED(sample(logits, random), NotImplementedError);
    return;
  }
  PagedCache<float> cache(2, 2, 16, 8);
  Variable<int32_t> table({1, 2}), starts({2}), lengths({1}), other({2});
  REFUSED(cache_write(cache, q, q, positions), InvalidArgumentError);
  REFUSED(cache_write(cache, k, short_k, positions), InvalidArgumentError);
  REFUSED(cache_write(cache, k, k, one_position), InvalidArgumentError);
  REFUSED(cache_read(cache, starts, starts, 1), InvalidArgumentError);
  REFUSED(cache_read(cache, table, lengths, 1), InvalidArgumentError);
  REFUSED(paged_attention(flat, cache, table, starts, lengths, 1.0f), InvalidArgumentError);
  REFUSED(paged_attention(q, cache, table, lengths, lengths, 1.0f), InvalidArgumentError);
  REFUSED(paged_attention(q, cache, table, starts, other, 1.0f), InvalidArgumentError);
  REFUSED(paged_attention(q, cache, table, starts, lengths, 1.0f, false, 3), InvalidArgumentError);
  PagedCache<float> odd(2, 2, 16, 6);  // heads that are no multiple of four values
  Variable<float> k6({3, 2, 6});
  REFUSED(cache_write(odd, k6, k6, positions), ROCMRuntimeError);
}

// Sizes whose product does not fit the 32 bits in which a tensor counts its elements: refused before anything is allocated.
static void sizes(bool gpu) {
  REFUSED(PagedCache<int8_t>(262145, 8, 16, 128), InvalidArgumentError);  // 2^32 + 16384
  REFUSED(PagedCache<float>(262145, 8, 16, 128), InvalidArgumentError);
  REFUSED(PagedCache<int8_t>(1u << 16, 1u << 16, 1, 8), InvalidArgumentError);  // 2^35: nothing is left in 32 bits
  REFUSED(PagedCache<int8_t>(0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu), InvalidArgumentError);
  REFUSED(PagedCache<int8_t>(0xffffffffu, 0xffffffffu, 0, 8), InvalidArgumentError);
  if (!gpu) return;
  PagedCache<float> cache(2, 1, 16, 256);
  Variable<int32_t> table({1, 2}), starts({2});
  REFUSED(cache_read(cache, table, starts, (1u << 24) + 1), InvalidArgumentError);  // 2^32 + 256
  REFUSED(cache_read(cache, table, starts, 0xffffffffu), InvalidArgumentError);
}

// A cache whose tensors were replaced by smaller ones, or moved out: its descriptor would name memory that is not there.
static void replaced() {
  Variable<float> k({3, 2, 8}), q({3, 4, 8});
  Variable<int32_t> slots({3}), table({1, 2}), starts({2}), lengths({1});
  const auto refused = [&](PagedCache<int8_t>& cache) {
    REFUSED(cache_write(cache, k, k, slots), InvalidArgumentError);
    REFUSED(cache_read(cache, table, starts, 1), InvalidArgumentError);
    REFUSED(paged_attention(q, cache, table, starts, lengths, 1.0f), InvalidArgumentError);
  };
  for (int which = 0; which < 4; ++which) {
    PagedCache<int8_t> cache(2, 2, 16, 8);
    if (which == 0) cache.values = Variable<int8_t>({1, 2, 16, 8});
    if (which == 1) cache.keys = Variable<int8_t>({2, 2, 16});
    if (which == 2) cache.keyScales = Variable<float>({2, 2, 8});
    if (which == 3) cache.valueScales = Variable<float>();
    refused(cache);
  }
  PagedCache<int8_t> cache(2, 2, 16, 8), other(std::move(cache));
  refused(cache);
}

// Keys that are all alike: the weights of a row are equal, and it gets the mean of the values that it sees.
template <class T>
static void means() {
  const unsigned tokens = 600, heads = 2, group = 3, size = 64, page = 16, pages = 40;
  PagedCache<T> cache(pages, heads, page, size);
  std::vector<float> k(tokens * heads * size), v(k.size()), q(tokens * heads * group * size);
  for (unsigned t = 0; t < tokens; ++t)
    for (unsigned i = 0; i < heads * size; ++i) {
      k[t * heads * size + i] = 1.0f;
      v[t * heads * size + i] = (i % size == 0 ? 127.0f : static_cast<float>(static_cast<int>((t * 7 + i) % 255) - 127)) / 32.0f;
    }
  for (size_t i = 0; i < q.size(); ++i) q[i] = static_cast<float>(static_cast<int>(i * 2654435761u >> 20) % 100) * 0.01f;
  std::vector<int32_t> slots(tokens), table(2 * pages, -1), starts = {0, 500, 600}, lengths = {500, 100};
  for (unsigned t = 0; t < tokens; ++t) {
    const unsigned sequence = t < 500 ? 0 : 1, at = t < 500 ? t : t - 500, held = pages - 1 - (sequence == 0 ? at / page : 32 + at / page);
    slots[t] = static_cast<int32_t>(held * page + at % page);
    table[sequence * pages + at / page] = static_cast<int32_t>(held);
  }
  std::vector<int32_t> positions(tokens, 0);  // nothing turns at position 0
  std::vector<double> frequencies = std::get<0>(rotary_frequencies(size));
  const unsigned half = static_cast<unsigned>(frequencies.size());
  Variable<float> dq = data::set(q, Shape({tokens, heads * group, size})), dk = data::set(k, Shape({tokens, heads, size})), dv = data::set(v, Shape({tokens, heads, size}));
  Variable<int32_t> dstarts = data::set(starts, Shape({3u})), dlengths = data::set(lengths, Shape({2u})), dtable = data::set(table, Shape({2u, pages}));
  Variable<float> turnedQ, turnedK;
  std::tie(turnedQ, turnedK) = rotary(dq, dk, data::set(positions, Shape({tokens})), data::set(frequencies, Shape({half})));
  EXPECT(data::get(turnedQ) == q && data::get(turnedK) == k);
  cache_write(cache, turnedK, dv, data::set(slots, Shape({tokens})));
  Variable<float> backK, backV;
  std::tie(backK, backV) = cache_read(cache, dtable, dstarts, tokens);
  const std::vector<float> gotK = data::get(backK), gotV = data::get(backV);
  double worst = 0;
  for (size_t i = 0; i < k.size(); ++i) worst = std::fmax(worst, std::fmax(std::fabs(gotK[i] - k[i]), std::fabs(gotV[i] - v[i])));
  EXPECT(worst <= 4e-6);  // whole steps of 1 / 32 or of 1 / 127: nothing but the scale is rounded
  for (unsigned window : {0u, 70u}) {
    const std::vector<float> y = data::get(paged_attention(turnedQ, cache, dtable, dstarts, dlengths, 0.125f, true, window));
    worst = 0;
    for (unsigned t = 0; t < tokens; ++t) {
      const unsigned base = t < 500 ? 0 : 500, first = window > 0 && t + 1 > base + window ? t + 1 - window : base;
      for (unsigned h = 0; h < heads * group; h += 5)
        for (unsigned d = 0; d < size; d += 3) {
          double mean = 0;
          for (unsigned s = first; s <= t; ++s) mean += gotV[(s * heads + h / group) * size + d];
          worst = std::fmax(worst, std::fabs(y[(t * heads * group + h) * size + d] - mean / (t + 1 - first)));
        }
    }
    EXPECT(worst <= 1e-3);  // values up to 4 times what float32 sums of 500 may be off by, 4 x (500 + 200) 2^-24, and more than that
  }
}

static void tokens() {
  const unsigned rows = 3, length = 1000;
  std::vector<float> logits(rows * length), random = {0.0f, 0.5f, 0.99f};
  for (unsigned i = 0; i < rows * length; ++i) logits[i] = static_cast<float>(i % length == 17 + i / length ? 20 : 0);
  std::vector<int32_t> k = {1, 1, 1};
  std::vector<float> cold = {0.0f, 0.0f, 0.0f};
  Variable<float> dl = data::set(logits, Shape({rows, length})), dr = data::set(random, Shape({rows})), dt = data::set(cold, Shape({rows}));
  Variable<int32_t> dk = data::set(k, Shape({rows}));
  for (int turn = 0; turn < 2; ++turn) {
    SampleFilters filters;
    if (turn == 0) filters.topK = &dk;
    else filters.temperature = &dt;
    Variable<int64_t> chosen;
    Variable<float> odds;
    std::tie(chosen, odds) = sample(dl, dr, filters);
    EXPECT((data::get(chosen) == std::vector<int64_t>{17, 18, 19}));
    EXPECT((data::get(odds) == std::vector<float>{1.0f, 1.0f, 1.0f}));
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
  sizes(gpu);
  if (gpu) {
    replaced();
    means<float>();
    means<int8_t>();
    tokens();
  } else {
    Session::setThreadDefault(nullptr);
    Device::setThreadDefault(nullptr);
  }
  if (failures == 0) std::printf("generation: all passed\n");
  return failures != 0;
}
