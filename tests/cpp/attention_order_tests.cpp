// When attention over a paged cache takes the longest sequences first, and which launch joins its pieces (wechat-tfcc_amd/csrc/paged_attention_plan.hpp): both sides of each line.  No GPU.
#include <cstdio>
#include <initializer_list>

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

enum Kind { EIGHT, FOUR, FLOAT };
static bool first(Kind kind, unsigned tokens, unsigned batch, unsigned group, unsigned heads, unsigned size, unsigned most, unsigned window = 0) {
  const unsigned rows = kind == FLOAT ? (size <= 64 ? 128 : size <= 128 ? 256 : 0) : kind == FOUR && (size <= 64 || size > 128) ? 0 : 128;
  const PagedAttentionPlan p = paged_attention_plan(tokens, batch, group, heads, size, most, 1, window, rows, kind == FLOAT, kind == FOUR, false);
  return attention_longest_first(p, tokens, batch, most, window, kind == FLOAT);
}

int main() {
  // single tokens
  for (const Kind kind : {EIGHT, FOUR}) {
    EXPECT(first(kind, 64, 64, 4, 8, 128, 4096) && first(kind, 64, 64, 4, 8, 128, 1025) && !first(kind, 64, 64, 4, 8, 128, 1024));
    EXPECT(!first(kind, 65, 65, 1, 8, 64, 165));     // 10.8 us, in order of length 12.8
    EXPECT(!first(kind, 32, 32, 4, 8, 128, 4096));   // one workgroup to a CU
    EXPECT(first(kind, 300, 30, 1, 12, 64, 513) && !first(kind, 300, 30, 1, 12, 64, 512));  // chunks
    EXPECT(!first(kind, 64, 64, 4, 8, 128, 8192, 4096) && first(kind, 64, 64, 4, 8, 128, 8192, 4097));
  }
  EXPECT(first(FLOAT, 64, 64, 4, 8, 128, 257) && !first(FLOAT, 64, 64, 4, 8, 128, 256));
  EXPECT(first(FLOAT, 9000, 30, 1, 12, 64, 900) && !first(FLOAT, 9000, 30, 1, 12, 64, 256) && !first(FLOAT, 9000, 30, 1, 12, 64, 900, 450) && first(FLOAT, 9000, 30, 1, 12, 64, 901, 451));
  EXPECT(!first(FLOAT, 2 * 56, 2, 4, 4, 80, 5150) && !first(FLOAT, 8, 8, 1, 12, 96, 4588));  // 96 workgroups in three pieces each
  EXPECT(first(EIGHT, 16 * 500, 16, 4, 8, 128, 500) && !first(EIGHT, 16 * 250, 16, 4, 8, 128, 256));  // wide tiles
  // joins
  EXPECT(attention_joins_few(8, 1, 64) && attention_joins_few(8, 100000, 256) && !attention_joins_few(9, 1, 64));
  EXPECT(!attention_joins_few(9, 512, 64) && attention_joins_few(9, 513, 64) && !attention_joins_few(16, 256, 128) && attention_joins_few(16, 257, 80) && !attention_joins_few(81, 16, 256));
  EXPECT(!attention_joins_few(12, 128, 256) && attention_joins_few(12, 129, 256));
  if (failures == 0) std::printf("attention order: all passed\n");
  return failures != 0;
}
