// How attention over a paged cache is dealt out, in host arithmetic of its own so that tests reach it without a GPU.
#pragma once

#include <stdint.h>

namespace tfcc_rocm {

struct PagedAttentionPlan {
  unsigned rows;        // of a tile
  unsigned tiles;       // an upper bound of the tiles of rows that all chunks make
  unsigned waves;       // of a workgroup, 4 or 8
  unsigned splits;      // pieces of the keys, each with a workgroup for every tile and cache head
  unsigned split_keys;  // keys of a piece, a multiple of 256
};

constexpr unsigned kAttentionRows = 16;    // rows (a token's query heads of one cache head) of a tile
constexpr unsigned kAttentionChunkRows = 128;  // of a tile of a chunk of many tokens
constexpr unsigned kAttentionStep = 256;   // keys that eight wavefronts take in one step
constexpr unsigned kAttentionMostSplits = 256;

// A chunk of n tokens makes ceil(n * group / rows) tiles; how the tokens are spread over the sequences only the device knows.
inline unsigned paged_attention_tiles(unsigned tokens, unsigned batch, unsigned group, unsigned rows) {
  const unsigned chunks = tokens < batch ? tokens : batch;
  return (unsigned)(((uint64_t)tokens * group + (uint64_t)(rows - 1) * chunks) / rows);
}

inline PagedAttentionPlan paged_attention_plan(unsigned tokens, unsigned batch, unsigned group, unsigned cache_heads, unsigned size, unsigned max_length,
                                               int causal, unsigned window, bool chunk_tiles) {
  PagedAttentionPlan p;
  // chunks of about the same number of tokens
  const uint64_t chunks = tokens < batch ? tokens : batch, mean = chunks == 0 ? 0 : (tokens + chunks - 1) / chunks;
  const auto groups_of = [&](unsigned rows) { return chunks * ((mean * group + rows - 1) / rows) * cache_heads; };
  // Tiles of 128 rows where they make a workgroup for each CU, of chunks that fill two (16 chunks of 256 tokens, 32 heads over 8 of 128: 374 us,
  // with tiles of 16 rows 469; one chunk of 1024: 190 and 235; 16 of 64: 182 and 171; one of 256: 208 and 76).
  p.rows = chunk_tiles && mean * group >= 2 * kAttentionChunkRows && groups_of(kAttentionChunkRows) >= 256 ? kAttentionChunkRows : kAttentionRows;
  p.tiles = paged_attention_tiles(tokens, batch, group, p.rows);
  // a tile spans at most `rows` tokens: the keys that one of them sees
  uint64_t keys = max_length;
  if (causal && window > 0 && (uint64_t)window + p.rows + 32 < keys) keys = (uint64_t)window + p.rows + 32;
  const uint64_t groups = groups_of(p.rows);
  // One workgroup of eight wavefronts to a CU is best as long as there are no more than two for each CU: it has the CU's LDS for rows on
  // their way, and little time goes into beginnings and ends (64 sequences of up to 4096 keys, 8 heads of 128 in int8: 88 us, with
  // four wavefronts 97; 200 sequences of 700: 78 and 59).  Eight with heads wider than 128 do not have the registers.
  uint64_t splits = 1;
  p.waves = groups <= 512 && size <= 128 && keys > kAttentionStep / 2 ? 8 : 4;
  if (p.rows == kAttentionChunkRows) {
    p.waves = 4;
    splits = groups < 384 ? 2 : 1;  // two of these share a CU
    if (keys < 4 * kAttentionStep) splits = 1;
  } else if (groups > 0 && groups < 256) {
    // Fewer than CUs: pieces of the keys, where they save more steps than the launch that joins them costs, three steps of 256 keys with
    // heads of 128 and four with heads of 64 (16 sequences of 4096: two pieces 30 us, one 40; one sequence of 1024: four 12.4, one 14.4;
    // 16 of 1024: two 16.6, one 15.6).
    const uint64_t steps = (keys + kAttentionStep - 1) / kAttentionStep;
    splits = 256 / groups;
    splits = splits < steps ? splits : steps;
    if (splits > 1 && (steps - (steps + splits - 1) / splits) * (size + 128) < 3 * 256) splits = 1;
    if (splits < 1) splits = 1;
  }
  uint64_t each = (keys + splits - 1) / splits;
  each = (each + kAttentionStep - 1) / kAttentionStep * kAttentionStep;
  if (each == 0) each = kAttentionStep;
  p.split_keys = (unsigned)each;
  p.splits = (unsigned)((keys + each - 1) / each);
  if (p.splits < 1) p.splits = 1;
  return p;
}

}  // namespace tfcc_rocm
