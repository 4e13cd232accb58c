// How attention over a paged cache is dealt out (wechat-tfcc_amd/csrc/paged_attention_plan.hpp), on the host: both sides of the rule's lines, that
// the launched tiles hold every chunk however the tokens are spread, and that the pieces hold every key.  No GPU.
#include <cstdio>
#include <initializer_list>
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

int main() {
  // one token of each sequence: a workgroup of eight wavefronts to a CU, pieces where there are fewer workgroups than CUs
  PagedAttentionPlan p = paged_attention_plan(32, 32, 4, 8, 128, 8192, 1, 0, 128, false);
  EXPECT(p.rows == 16 && p.waves == 8 && p.splits == 1 && p.tiles >= 32);
  p = paged_attention_plan(1, 1, 4, 8, 128, 8192, 1, 0, 128, false);
  EXPECT(p.rows == 16 && p.splits == 32 && p.split_keys == 256);
  EXPECT(paged_attention_plan(1, 1, 4, 8, 128, 600, 1, 0, 128, false).splits == 1);
  EXPECT(paged_attention_plan(1, 1, 4, 8, 128, 100000, 1, 512, 128, false).splits <= 3);  // a window bounds the keys
  EXPECT(paged_attention_plan(32, 32, 4, 8, 256, 8192, 1, 0, 128, false).waves == 4);
  EXPECT(paged_attention_plan(100, 100, 4, 8, 128, 8192, 1, 0, 128, false).waves == 4);
  // tiles of 128 rows: chunks that fill half of one, and 20000 rows in all, 32000 over more than 1536 keys
  EXPECT(paged_attention_plan(4096, 16, 4, 8, 128, 4096, 1, 0, 128, false).rows == 128);
  EXPECT(paged_attention_plan(4096, 16, 4, 8, 128, 4096, 1, 0, 0, false).rows == 16);
  EXPECT(paged_attention_plan(1024, 1, 4, 8, 128, 4096, 1, 0, 128, false).rows == 128 && paged_attention_plan(1024, 1, 4, 8, 128, 4096, 1, 0, 128, false).splits == 2);
  EXPECT(paged_attention_plan(1024, 1, 4, 8, 128, 1000, 1, 0, 128, false).splits == 1);
  EXPECT(paged_attention_plan(1536, 1, 4, 8, 128, 4096, 1, 0, 128, false).splits == 1);
  EXPECT(paged_attention_plan(256, 1, 4, 8, 128, 4096, 1, 0, 128, false).rows == 16);
  EXPECT(paged_attention_plan(16 * 48, 16, 4, 8, 128, 4096, 1, 0, 128, false).rows == 16);
  EXPECT(paged_attention_plan(39 * 63, 39, 4, 8, 128, 510, 1, 0, 128, false).rows == 128);
  EXPECT(paged_attention_plan(16 * 48, 16, 4, 8, 128, 2048, 1, 0, 128, false).rows == 16);
  EXPECT(paged_attention_plan(12 * 138, 12, 8, 1, 256, 589, 1, 0, 128, false).rows == 16);
  EXPECT(paged_attention_plan(2000, 2000, 4, 8, 128, 510, 1, 0, 128, false).rows == 16);  // single tokens do not fill a tile
  // float32: tiles of 256 rows from fewer rows on, pieces of long contexts
  EXPECT(paged_attention_plan(15 * 205, 15, 8, 2, 128, 376, 1, 0, 256, true).rows == 256);
  EXPECT(paged_attention_plan(674, 1, 6, 4, 96, 675, 1, 0, 256, true).rows == 16);
  p = paged_attention_plan(1024, 1, 4, 8, 128, 4096, 1, 0, 256, true);
  EXPECT(p.rows == 256 && p.splits == 2 && p.split_keys == 2048);
  p = paged_attention_plan(256, 1, 4, 8, 128, 4096, 1, 0, 256, true);
  EXPECT(p.rows == 256 && p.splits == 8);
  EXPECT(paged_attention_plan(256, 1, 4, 8, 128, 4096, 1, 512, 256, true).rows == 16);
  EXPECT(paged_attention_plan(64, 64, 8, 8, 128, 4096, 1, 0, 256, true).rows == 16);  // single tokens do not fill a tile
  std::mt19937 g(1);
  for (int turn = 0; turn < 20000; ++turn) {
    const unsigned batch = 1 + g() % 70, group = 1 + g() % 9, heads = 1 + g() % 40, size = 8 * (1 + g() % 32), most = g() % 3 ? g() % 9000 : g() % 300;
    std::vector<unsigned> chunks(batch);
    unsigned tokens = 0;
    for (unsigned& n : chunks) tokens += n = g() % 3 == 0 ? 0 : g() % (turn % 2 ? 4 : 400);
    tokens += g() % 5;  // rows behind the last sequence
    const int causal = g() % 4 != 0;
    const unsigned window = causal && g() % 2 ? 1 + g() % 700 : 0;
    const bool float_cache = g() % 2;
    p = paged_attention_plan(tokens, batch, group, heads, size, most, causal, window, g() % 3 == 0 ? 0 : !float_cache || size <= 64 ? 128 : size <= 128 ? 256 : 0, float_cache);
    unsigned tiles = 0;
    for (unsigned n : chunks) tiles += (n * group + p.rows - 1) / p.rows;
    EXPECT(tiles <= p.tiles);
    EXPECT(p.rows == kAttentionRows || p.rows == 128 || p.rows == 256);
    EXPECT((p.waves == 4 || p.waves == 8) && (p.waves == 4 || size <= 128));
    EXPECT(p.splits >= 1 && p.splits <= kAttentionMostSplits && p.split_keys > 0 && p.split_keys % (p.waves * (float_cache ? 16 : 32)) == 0);
    // the keys that the rows of one tile see begin at a multiple of 32: with a window they are its rows' tokens and the window's
    unsigned long long span = most;
    if (window > 0 && window + p.rows + 31ull < span) span = window + p.rows + 31ull;
    EXPECT((unsigned long long)p.splits * p.split_keys >= span);
  }
  p = paged_attention_plan(0, 4, 4, 8, 128, 100, 1, 0, 128, false);
  EXPECT(p.tiles == 0 && p.splits == 1);
  if (failures == 0) std::printf("paged attention plan: all passed\n");
  return failures != 0;
}
