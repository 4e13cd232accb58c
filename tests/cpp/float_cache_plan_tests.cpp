// From where on chunks over a float32 cache are dealt out in wide tiles (wechat-tfcc_amd/csrc/paged_attention_plan.hpp), whose products are right to 2^-21 and not 2^-24: plain
// scores later than shaped ones, on both sides of each line.  No GPU.
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

static unsigned rows(bool shaped, unsigned tokens, unsigned batch, unsigned group, unsigned heads, unsigned size, unsigned most) {
  return paged_attention_plan(tokens, batch, group, heads, size, most, 1, 0, size <= 64 ? 128 : 256, true, false, shaped).rows;
}

int main() {
  // 8192 rows to 17999: over 2048 keys, with shaped scores over 1000
  EXPECT(rows(false, 4 * 128, 4, 4, 8, 128, 1500) == 16 && rows(true, 4 * 128, 4, 4, 8, 128, 1500) == 256);
  EXPECT(rows(false, 2 * 512, 2, 1, 12, 64, 1024) == 16 && rows(true, 2 * 512, 2, 1, 12, 64, 1024) == 128);
  EXPECT(rows(false, 700, 1, 1, 16, 64, 1500) == 16 && rows(true, 700, 1, 1, 16, 64, 1500) == 128);
  EXPECT(rows(false, 256, 1, 4, 8, 128, 2047) == 16 && rows(false, 256, 1, 4, 8, 128, 2048) == 256 && rows(false, 255, 1, 4, 8, 128, 2048) == 16);
  EXPECT(rows(true, 256, 1, 4, 8, 128, 999) == 16 && rows(true, 256, 1, 4, 8, 128, 1000) == 256 && rows(true, 255, 1, 4, 8, 128, 1000) == 16);
  // 18000 rows: for both, over 1000 keys
  for (const bool shaped : {false, true}) {
    EXPECT(rows(shaped, 563, 1, 4, 8, 128, 563) == 256 && rows(shaped, 562, 1, 4, 8, 128, 563) == 16);
    EXPECT(rows(shaped, 5 * 512, 5, 1, 12, 64, 1000) == 128 && rows(shaped, 5 * 512, 5, 1, 12, 64, 1024) == 128);
  }
  // plain ones of heads of 64 however few tiles and keys there are (12 heads of 64: 10 of 200 over 950 51 us, with tiles of 16 rows 89)
  EXPECT(rows(false, 10 * 200, 10, 1, 12, 64, 950) == 128 && rows(false, 5 * 512, 5, 1, 12, 64, 850) == 128 && rows(false, 2 * 750, 2, 1, 12, 64, 750) == 128);
  EXPECT(rows(false, 2 * 749, 2, 1, 12, 64, 750) == 16 && rows(false, 4 * 150, 4, 4, 8, 64, 999) == 128);
  // windows in two pieces of tiles of 256 rows, where these make no third round
  const auto window = [](unsigned tokens, unsigned batch, unsigned group, unsigned heads) {
    return paged_attention_plan(tokens, batch, group, heads, 128, 4000, 1, 512, 256, true, false, false).splits;
  };
  EXPECT(window(854, 14, 4, 8) == 1);   // 72 us, in two pieces 121
  EXPECT(window(971, 4, 2, 16) == 1);   // 78 and 111
  EXPECT(window(1024, 1, 4, 8) == 2 && window(2 * 512, 2, 4, 8) == 2);
  if (failures == 0) std::printf("float cache plan: all passed\n");
  return failures != 0;
}
