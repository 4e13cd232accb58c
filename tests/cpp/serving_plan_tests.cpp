// How attention over caches of 4-bit integers, and over float32 ones in pieces, is dealt out (wechat-tfcc_amd/csrc/paged_attention_plan.hpp), on the host: both
// sides of the rules' lines, and that tiles and pieces hold every row and key.  No GPU.
#include <cstdio>
#include <random>
#include <vector>

#include "paged_attention_plan.hpp"

using namespace tfcc_rocm;

static int failures = 0;
#define EXPECT(cond)                                         \
  do {                                                       \
    if (!(cond)) {                                           \
      ++failures;                                            \
      std::printf("FAIL line %d: %s\n", __LINE__, #cond);    \
    }                                                        \
  } while (0)

static PagedAttentionPlan four(unsigned tokens, unsigned batch, unsigned group, unsigned heads, unsigned size, unsigned most) {
  return paged_attention_plan(tokens, batch, group, heads, size, most, 1, 0, 128, false, true);
}
static PagedAttentionPlan float32(unsigned tokens, unsigned batch, unsigned group, unsigned heads, unsigned size, unsigned most) {
  return paged_attention_plan(tokens, batch, group, heads, size, most, 1, 0, size <= 64 ? 128 : 256, true);
}

int main() {
  // single tokens: one workgroup of twelve wavefronts to a CU, heads wider than 128 eight, or several of four
  EXPECT(four(32, 32, 4, 8, 128, 4096).waves == 12 && four(32, 32, 4, 8, 256, 4096).waves == 8 && four(64, 64, 4, 8, 128, 4096).waves == 4);
  EXPECT(four(32, 32, 4, 8, 128, 512).waves == 4 && four(32, 32, 4, 8, 128, 513).waves == 12 && four(16, 16, 4, 8, 128, 513).waves == 12 && four(15, 15, 4, 8, 128, 513).waves == 4);
  EXPECT(four(32, 32, 4, 8, 256, 1024).waves == 4 && four(32, 32, 4, 8, 256, 1025).waves == 8);
  EXPECT(four(1, 1, 1, 12, 64, 4096).waves == 4 && four(1, 1, 1, 12, 64, 9000).waves == 12);  // enough to do for all
  EXPECT(four(32, 32, 4, 8, 128, 4096).splits == 1 && four(1, 1, 4, 8, 128, 4096).splits > 1);
  // wide tiles: workgroups for nearly two to a CU, over few keys for more than one
  EXPECT(four(57 * 128, 1, 1, 8, 128, 4096).rows == 128 && four(56 * 128, 1, 1, 8, 128, 4096).rows == 16);
  EXPECT(four(35 * 128, 1, 1, 8, 128, 512).rows == 128 && four(34 * 128, 1, 1, 8, 128, 512).rows == 16 && four(35 * 128, 1, 1, 8, 128, 513).rows == 16);
  EXPECT(four(100 * 63, 100, 1, 8, 128, 512).rows == 16 && four(100 * 64, 100, 1, 8, 128, 512).rows == 128);  // chunks that fill half of one
  // float32: wide tiles from 8192 rows on over 1000 keys, in as many pieces as run at the same time
  EXPECT(float32(5 * 512, 5, 1, 12, 64, 1000).rows == 128 && float32(5 * 512, 5, 1, 12, 64, 999).rows == 16 && float32(5 * 512, 5, 1, 12, 64, 1000).splits == 2);
  EXPECT(float32(4 * 128, 4, 1, 12, 64, 1500).rows == 16 && float32(4 * 128, 4, 4, 8, 128, 1500).rows == 256 && float32(4 * 128, 4, 4, 8, 128, 1500).splits == 4);
  EXPECT(float32(2 * 512, 2, 4, 8, 128, 512).splits == 2 && float32(2 * 512, 2, 4, 8, 128, 511).splits == 1);
  EXPECT(float32(2 * 512, 2, 4, 8, 128, 512).split_keys == 256 && float32(5 * 512, 5, 1, 12, 64, 1000).split_keys == 512);
  // one more over long contexts
  EXPECT(float32(5 * 600, 5, 1, 12, 64, 1024).splits == 2 && float32(5 * 600, 5, 1, 12, 64, 1023).splits == 1 && float32(6 * 600, 6, 1, 12, 64, 1200).splits == 1);
  EXPECT(float32(3 * 600, 3, 1, 12, 64, 1536).splits == 3 && float32(3 * 600, 3, 1, 12, 64, 1535).splits == 2 && float32(1024, 1, 1, 12, 64, 4096).splits == 5);
  EXPECT(float32(20 * 64, 20, 4, 8, 128, 4000).splits == 1);
  std::mt19937 g(2);
  for (int turn = 0; turn < 20000; ++turn) {
    const unsigned batch = 1 + g() % 70, group = 1 + g() % 9, heads = 1 + g() % 40, size = 16 * (1 + g() % 16), most = g() % 3 ? g() % 9000 : g() % 300;
    std::vector<unsigned> chunks(batch);
    unsigned tokens = 0;
    for (unsigned& n : chunks) tokens += n = g() % 3 == 0 ? 0 : g() % (turn % 2 ? 4 : 400);
    tokens += g() % 5;  // rows behind the last sequence
    const int causal = g() % 4 != 0;
    const unsigned window = causal && g() % 2 ? 1 + g() % 700 : 0;
    const PagedAttentionPlan p = paged_attention_plan(tokens, batch, group, heads, size, most, causal, window, size == 128 && g() % 3 ? 128 : 0, false, true);
    unsigned tiles = 0;
    for (unsigned n : chunks) tiles += (n * group + p.rows - 1) / p.rows;
    EXPECT(tiles <= p.tiles);
    EXPECT(p.rows == kAttentionRows || (p.rows == 128 && p.waves == 4));
    EXPECT(p.waves == 4 || p.waves == (size <= 128 ? 12u : 8u));
    EXPECT(p.splits >= 1 && p.splits <= kAttentionMostSplits && p.split_keys > 0 && p.split_keys % (p.waves * 32) == 0);
    unsigned long long span = most;
    if (window > 0 && window + p.rows + 31ull < span) span = window + p.rows + 31ull;
    EXPECT((unsigned long long)p.splits * p.split_keys >= span);
  }
  if (failures == 0) std::printf("serving plan: all passed\n");
  return failures != 0;
}
