// How attention over a paged cache deals out calls, one to a line of the input:
//   tokens batch group cache_heads size max_length causal window chunk_rows float_cache
// printed as: rows of a tile, wavefronts, pieces, keys of a piece.  No GPU.
#include <cstdio>

#include "paged_attention_plan.hpp"

int main() {
  unsigned v[10];
  for (;;) {
    for (int i = 0; i < 10; ++i)
      if (std::scanf("%u", v + i) != 1) return i != 0;
    const tfcc_rocm::PagedAttentionPlan p = tfcc_rocm::paged_attention_plan(v[0], v[1], v[2], v[3], v[4], v[5], static_cast<int>(v[6]), v[7], v[8], v[9] != 0);
    std::printf("%u %u %u %u\n", p.rows, p.waves, p.splits, p.split_keys);
  }
}
