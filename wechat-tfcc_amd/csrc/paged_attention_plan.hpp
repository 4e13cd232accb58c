// How attention over a paged cache is dealt out, in host arithmetic of its own so that tests reach it without a GPU.
#pragma once

#include <stdint.h>

namespace tfcc_rocm {

struct PagedAttentionPlan {
  unsigned rows;        // of a tile
  unsigned tiles;       // an upper bound of the tiles of rows that all chunks make
  unsigned waves;       // of a workgroup, 4 or 8
  unsigned splits;      // pieces of the keys, each with a workgroup for every tile and cache head
  unsigned split_keys;  // keys of a piece, a multiple of what its wavefronts take in one step
};

constexpr unsigned kAttentionRows = 16;    // rows (a token's query heads of one cache head) of a tile
constexpr unsigned kAttentionStep = 256;   // keys that eight wavefronts take of an int8 cache in one step
constexpr unsigned kAttentionMostSplits = 256;

// A chunk of n tokens makes ceil(n * group / rows) tiles; how the tokens are spread over the sequences only the device knows.
inline unsigned paged_attention_tiles(unsigned tokens, unsigned batch, unsigned group, unsigned rows) {
  const unsigned chunks = tokens < batch ? tokens : batch;
  return (unsigned)(((uint64_t)tokens * group + (uint64_t)(rows - 1) * chunks) / rows);
}

// chunk_rows: of the tiles that chunks of many tokens may take, 128 or 256; 0: there are none.
inline PagedAttentionPlan paged_attention_plan(unsigned tokens, unsigned batch, unsigned group, unsigned cache_heads, unsigned size, unsigned max_length,
                                               int causal, unsigned window, unsigned chunk_rows, bool float_cache) {
  PagedAttentionPlan p;
  // chunks of about the same number of tokens
  const uint64_t chunks = tokens < batch ? tokens : batch, mean = chunks == 0 ? 0 : (tokens + chunks - 1) / chunks;
  const auto groups_of = [&](unsigned rows) { return chunks * ((mean * group + rows - 1) / rows) * cache_heads; };
  // a tile spans at most `rows` tokens: the keys that one of them sees
  const auto keys_of = [&](unsigned rows) {
    const uint64_t span = (uint64_t)window + rows + 32;
    return causal && window > 0 && span < max_length ? span : (uint64_t)max_length;
  };
  const uint64_t all = mean * group * chunks * cache_heads;  // rows
  bool wide = false;
  if (chunk_rows > 0 && !float_cache) {
    // Wide tiles where chunks fill half of one and there are rows for the GPU, more of them over long contexts, whose steps tiles of 16 rows
    // take at the rate of HBM (rows in all: 39 chunks of up to 84 over 510, 32 heads over 8 of 128, 79000: 61 us, with tiles of 16 rows 99; 8 of 49 over 2706 with
    // a window of 293, 64 heads, 20500: 28 and 34; 12 of 184 over 589, 8 heads over 1 of 256, 13000: 74 and 57; over long contexts one of 1024 over
    // 4096, 32800: 186 and 228; 16 of 64 over 2048, 24600: 105 and 89).
    wide = 2 * mean * group >= chunk_rows && all >= (keys_of(chunk_rows) <= 1536 ? 20000 : 32000);
  } else if (chunk_rows > 0) {
    // float32, whose tiles of 16 rows run on slower matrix operations: earlier, and earlier still where long contexts can be cut into pieces
    // (32 heads over 8 of 128, tokens x rows of all tiles: 15 of 205 over 376, 16 heads over 2: 48 us, with tiles of 16 rows 94; 11 of 125 over 227: 35 and 45;
    // one of 674, 24 heads over 4 of 96: 73 and 62; one of 256 over 4096 in eight pieces 84 and 210).
    wide = 2 * mean * group >= chunk_rows && (all >= 18000 || (all >= 8192 && keys_of(chunk_rows) >= 2048));
  }
  p.rows = wide ? chunk_rows : kAttentionRows;
  p.tiles = paged_attention_tiles(tokens, batch, group, p.rows);
  const uint64_t keys = keys_of(p.rows), groups = groups_of(p.rows);
  // One workgroup of eight wavefronts to a CU is best as long as there are no more than two for each CU: it has the CU's LDS for rows on
  // their way, and little time goes into beginnings and ends (64 sequences of up to 4096 keys, 8 heads of 128 in int8: 88 us, with
  // four wavefronts 97; 200 sequences of 700: 78 and 59).  Eight with heads wider than 128 do not have the registers.
  uint64_t splits = 1, step = kAttentionStep;
  p.waves = groups <= 512 && size <= 128 && keys > kAttentionStep / 2 ? 8 : 4;
  if (!wide) step = p.waves * (float_cache ? 16 : 32);
  if (wide && float_cache) {
    // as many as run at the same time (one of 1024 tokens over 4096, 128 workgroups: two pieces 260 us, one 404)
    p.waves = chunk_rows / 32;
    const uint64_t fit = groups == 0 ? 1 : 256 * 256 / chunk_rows / groups;
    splits = keys < 2048 || fit < 1 ? 1 : fit < keys / 512 ? fit : keys / 512;
    if (splits > 8) splits = 8;
  } else if (wide) {
    p.waves = 4;
    splits = keys >= 2048 && groups < 384 && size <= 128 ? 2 : 1;  // two share a CU; of heads wider than 128 one has it, and they are enough
  } else if (groups > 0 && groups < 256) {
    // Fewer than CUs: pieces of the keys, where they save more steps than the launch that joins them costs (int8: 16 sequences of 4096, two
    // pieces 30 us, one 40; one of 1024: four 12.4, one 14.4; 2 of 938, 24 heads over 4 of 96: four 11.8, one 13.6; one of 777, 12 heads of 64:
    // four 11.4, one 9.8; float32: 12 of 429, 8 heads over 1 of 256: eight 18, one 35; 2 chunks of 3 over 737, 12 heads of 64: six 11.3, one 15.5;
    // 7 of 15 over 7203, 20 heads over 5 of 80, 140 workgroups: two 109, one 186).
    const uint64_t steps = (keys + step - 1) / step;
    splits = float_cache && keys >= 4096 ? (256 + groups - 1) / groups : 256 / groups;
    splits = splits < steps ? splits : steps;
    if (splits > 32 && splits > steps / 2) splits = steps / 2 > 32 ? steps / 2 : 32;  // joining them takes its time too (3 of 10389: 41 pieces 18.5 us, 82 21)
    if (splits < 1) splits = 1;
    const uint64_t saved = steps - (steps + splits - 1) / splits;
    if (float_cache ? saved * (size + 64) < 5 * 64 : saved * (size + 128) < 640) splits = 1;
  }
  uint64_t each = (keys + splits - 1) / splits;
  each = (each + step - 1) / step * step;
  if (each == 0) each = step;
  p.split_keys = (unsigned)each;
  p.splits = (unsigned)((keys + each - 1) / each);
  if (p.splits < 1) p.splits = 1;
  return p;
}

}  // namespace tfcc_rocm
