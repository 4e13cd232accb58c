// How attention over a paged cache is dealt out, in host arithmetic of its own so that tests reach it without a GPU.
#pragma once

#include <stdint.h>

namespace tfcc_rocm {

struct PagedAttentionPlan {
  unsigned tiles;       // an upper bound of the tiles of rows that all chunks make
  unsigned splits;      // pieces of the keys, each with a workgroup for every tile and cache head
  unsigned split_keys;  // keys of a piece, a multiple of 128
};

constexpr unsigned kAttentionRows = 16;    // rows (a token's query heads of one cache head) of a tile
constexpr unsigned kAttentionStep = 128;   // keys that the four wavefronts of a workgroup take in one step
constexpr unsigned kAttentionMostSplits = 256;

// A chunk of n tokens makes ceil(n * group / rows) tiles; how the tokens are spread over the sequences only the device knows.
inline unsigned paged_attention_tiles(unsigned tokens, unsigned batch, unsigned group, unsigned rows) {
  const unsigned chunks = tokens < batch ? tokens : batch;
  return (unsigned)(((uint64_t)tokens * group + (uint64_t)(rows - 1) * chunks) / rows);
}

inline PagedAttentionPlan paged_attention_plan(unsigned tokens, unsigned batch, unsigned group, unsigned cache_heads, unsigned max_length,
                                               int causal, unsigned window) {
  PagedAttentionPlan p;
  p.tiles = paged_attention_tiles(tokens, batch, group, kAttentionRows);
  // a tile spans at most `rows` tokens: the keys that one of them sees
  uint64_t keys = max_length;
  if (causal && window > 0 && (uint64_t)window + kAttentionRows + 32 < keys) keys = (uint64_t)window + kAttentionRows + 32;
  const uint64_t groups = (uint64_t)p.tiles * cache_heads;
  uint64_t splits = groups == 0 ? 1 : 1024 / groups;
  const uint64_t most = (keys + 2 * kAttentionStep - 1) / (2 * kAttentionStep);
  if (splits > most) splits = most;
  if (splits > kAttentionMostSplits) splits = kAttentionMostSplits;
  if (splits < 1) splits = 1;
  uint64_t each = (keys + splits - 1) / splits;
  each = (each + kAttentionStep - 1) / kAttentionStep * kAttentionStep;
  if (each == 0) each = kAttentionStep;
  p.split_keys = (unsigned)each;
  p.splits = (unsigned)((keys + each - 1) / each);
  if (p.splits < 1) p.splits = 1;
  return p;
}

}  // namespace tfcc_rocm
