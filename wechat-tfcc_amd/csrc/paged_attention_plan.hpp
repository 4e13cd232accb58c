// How attention over a paged cache is dealt out, in host arithmetic of its own so that tests reach it without a GPU.
#pragma once

#include <stdint.h>

namespace tfcc_rocm {

struct PagedAttentionPlan {
  unsigned rows;        // of a tile
  unsigned tiles;       // an upper bound of the tiles of rows that all chunks make
  unsigned waves;       // of a workgroup, 4, 8 or 12
  unsigned splits;      // pieces of the keys, each with a workgroup for every tile and cache head
  unsigned split_keys;  // keys of a piece, a multiple of what its wavefronts take in one step
  uint64_t groups;      // workgroups of all pieces and cache heads, if the chunks are about the same
};

constexpr unsigned kAttentionRows = 16;    // rows (a token's query heads of one cache head) of a tile
constexpr unsigned kAttentionStep = 256;   // keys that eight wavefronts take of an int8 cache in one step
constexpr unsigned kAttentionMostSplits = 256;

// A chunk of n tokens makes ceil(n * group / rows) tiles; how the tokens are spread over the sequences only the device knows.
inline unsigned paged_attention_tiles(unsigned tokens, unsigned batch, unsigned group, unsigned rows) {
  const unsigned chunks = tokens < batch ? tokens : batch;
  return (unsigned)(((uint64_t)tokens * group + (uint64_t)(rows - 1) * chunks) / rows);
}

// chunk_rows: of the tiles that chunks of many tokens may take, 128 or 256; 0: there are none.  halves: a cache of 4-bit integers.  shaped: with a cap, slopes or prefixes.
inline PagedAttentionPlan paged_attention_plan(unsigned tokens, unsigned batch, unsigned group, unsigned cache_heads, unsigned size, unsigned max_length,
                                               int causal, unsigned window, unsigned chunk_rows, bool float_cache, bool halves = false, bool shaped = true) {
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
  if (chunk_rows > 0 && halves) {
    // 4-bit integers are cheap to unpack, and tiles of 16 rows, whose wavefronts wait for nobody, are ahead until there are wide tiles for nearly two to a CU, or over few keys for more than one
    // (us with wide tiles and with 16 rows, 8 heads of 128, groups of 4 or 8: 2 chunks of 700 over 2500, 272 workgroups: 153 and 92; 10 of 200 over 1000, 400: 65 and 59; one of 1024 over
    // 1100, groups of 8, 512: 75 and 81; 8 of 200 over 300, 320: 27 and 34; 16 of 512, 1536: 103 and 163).
    wide = 2 * mean * group >= chunk_rows && groups_of(chunk_rows) >= (keys_of(chunk_rows) <= 512 ? 280 : 450);
  } else if (chunk_rows > 0 && !float_cache) {
    // Wide tiles where chunks fill half of one and there are rows for the GPU, more of them over long contexts, whose steps tiles of 16 rows
    // take at the rate of HBM (rows in all: 39 chunks of up to 84 over 510, 32 heads over 8 of 128, 79000: 61 us, with tiles of 16 rows 99; 8 of 49 over 2706 with
    // a window of 293, 64 heads, 20500: 28 and 34; 12 of 184 over 589, 8 heads over 1 of 256, 13000: 74 and 57; over long contexts one of 1024 over
    // 4096, 32800: 186 and 228; 16 of 64 over 2048, 24600: 105 and 89).
    wide = 2 * mean * group >= chunk_rows && all >= (keys_of(chunk_rows) <= 1536 ? 20000 : 32000);
  } else if (chunk_rows > 0) {
    // float32, whose tiles of 16 rows run on slower matrix operations: earlier, and earlier still where long contexts can be cut into pieces
    // (32 heads over 8 of 128: 15 of 205 over 376, 16 heads over 2: 48 us, with tiles of 16 rows 94; 11 of 125 over 227: 35 and 45;
    // one of 674, 24 heads over 4 of 96: 73 and 62; one of 256 over 4096 in eight pieces 84 and 210; 4 of 128 over 1500 in four 68 and 162; 12 heads of 64: 5 of 512 over 2000 in two
    // pieces 99 and 185, over 850 49 and 79; 10 of 200 over 950 51 and 89; 2 of 800 over 800 38 and 42, of up to 800 36 and 32; 2 of 512 over 1024 38 and 46, over 512 27 and 22).
    // What they cost is bits: their products of pieces are right to 2^-21 of a term where the fp32 operations round to 2^-24, and lose what lies 2^-30 below a row's largest value.  So plain
    // scores of fewer than 18000 rows keep the fp32 operations below 2048 keys; shaped ones, which are rounded besides, below 1000, where those of up to 64 values that do not make 250 tiles
    // of 128 rows keep them as well.
    const uint64_t seen = keys_of(chunk_rows);
    const bool many = all >= 18000 && (!shaped || chunk_rows > 128 || groups_of(chunk_rows) >= 250);
    wide = 2 * mean * group >= chunk_rows && (many || (all >= 8192 && seen >= (shaped ? 1000 : 2048)));
  }
  p.rows = wide ? chunk_rows : kAttentionRows;
  p.tiles = paged_attention_tiles(tokens, batch, group, p.rows);
  const uint64_t keys = keys_of(p.rows), groups = groups_of(p.rows);
  // One workgroup of eight wavefronts to a CU is best as long as there are no more than two for each CU: it has the CU's LDS for rows on
  // their way, and little time goes into beginnings and ends (64 sequences of up to 4096 keys, 8 heads of 128 in int8: 88 us, with
  // four wavefronts 97; 200 sequences of 700: 78 and 59).  Eight with heads wider than 128 do not have the registers.
  uint64_t splits = 1, step = kAttentionStep;
  p.waves = groups <= 512 && size <= 128 && keys > kAttentionStep / 2 ? 8 : 4;
  if (halves) {
    // What holds a workgroup of 4-bit integers up is its operations: as many wavefronts to a CU as registers allow, 12 (heads wider than 128: 8), in one workgroup where there is
    // no more than one to a CU and enough to do, else in several, whose beginnings and ends others fill.  (Us with one and with several, 8 heads of 128: 32 sequences of 4096 33 and 40,
    // 64 of up to 4096 54 and 48, 40 of up to 1000 22 and 14, 32 of up to 1000 13.2 and 15.1, 16 of 600 10.1 and 10.7, 4 of 3000 12.6 and 11.8; 12 heads, one of 4000 11.1 and 9.6;
    // 8 heads of 256, 32 of 4096 50 and 56, of 1000 22.8 and 21.7.)
    p.waves = groups <= 256 && ((groups >= 128 && keys > 512 && size <= 128) || (keys > 1024 && groups * keys > 256 * 384)) ? (size <= 128 ? 12 : 8) : 4;
  }
  if (!wide) step = p.waves * (float_cache ? 16 : 32);
  if (wide && float_cache) {
    // as many as run at the same time (one of 1024 tokens over 4096, 128 workgroups: two pieces 260 us, one 404; over 1024 77 and 116; 2 of 512 over 512 52 and 64)
    p.waves = chunk_rows / 32;
    step = p.waves * 16;
    uint64_t fit = groups == 0 ? 1 : 256 * 256 / chunk_rows / groups;
    // One more where that leaves many places free: of two or three pieces the tiles that see few keys, or are not there, make room for the others' (12 heads of 64, two and
    // one: 6 of up to 517 over up to 1201 67 us and 82, 3 of 1000 over 6000 401 and 471; three and two: one prompt of 1900 67 and 85, 3 of up to 600 over up to 2000 72 and 95,
    // but 5 of up to 512 over up to 1024, pieces of 350, 64 and 56; next to the line at 320 workgroups, chunks of one length over 1201: 300 85 and 91, 336 95 and 91, 360 96 and 91, 384 over 3000 207 and 204; six and five: one of 1024 over 4096 104 and 82; tiles of 256 rows, 20 of 64 over 1000, 144 and 120).
    if (chunk_rows == 128 && ((fit == 1 && groups <= 320) || (fit == 2 && groups <= 192)) && keys >= 512 * (fit + 1)) ++fit;
    // Of tiles of 256 rows a CU takes one, so a third round outweighs what two pieces of a window give: where ragged chunks, of which each makes half a tile more than its rows fill, would need one (window of 512,
    // 32 heads over 8 of 128: 14 of up to 91 over up to 4817 72 us, in two pieces 121; 32 over 16, 4 of up to 344 over up to 1800 78 and 111; with less to do in two pieces 0.92 to 0.95 of the time).
    if (chunk_rows == 256 && fit == 2 && keys < max_length && ((uint64_t)tokens * group * 2 + chunks * 256) * cache_heads > 280 * 256) fit = 1;
    splits = keys < 512 || fit < 1 ? 1 : fit < keys / 256 ? fit : keys / 256;
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
  p.groups = groups * p.splits;
  return p;
}

// Whether the longest sequences and the last rows of a chunk are taken first: where more workgroups than run at once wait for their turn (more than CUs, of wide tiles than two to a CU or one) and what
// one that begins late costs is more than the microsecond that every workgroup spends on the order.  That is so from so many keys on (random calls of 8 and 4 bits and float32, geometric means of the
// time without the order over that with it: single tokens over integers, ragged and uniform lengths, over 257 to 512 keys 0.97 and 0.95, over 513 to 1024 1.00 and 0.97, over 1025 to 2048 1.04 and
// 0.98, over more 1.05 and 0.99; chunks over 129 to 256 keys 0.98 and 0.96, over 257 to 512 0.98 and 0.98, over 513 to 1024 1.01 and 1.00, over more 1.03 and 1.00; float32 and wide tiles over
// up to 128 keys 1.00 and 0.96, over 129 to 256 1.01 and 0.98, over 257 to 512 1.03 and 1.01, over more 1.04 and 1.02), but not where a window of half the keys or less lets all rows see about as many (0.95 to
// 0.99 throughout), nor in pieces (ragged ones 1.00, from 0.80 to 1.42, uniform ones 0.98 to 0.99, of wide tiles 0.99; 2 chunks of up to 75 over up to 5758, 16 heads over 4 of 80: 58 us in the batch's order, 93).
inline bool attention_longest_first(const PagedAttentionPlan& p, unsigned tokens, unsigned batch, unsigned max_length, unsigned window, bool float_cache) {
  if (p.groups <= (p.rows == kAttentionRows ? 256 : 65536 / p.rows)) return false;
  if (p.splits > 1 || (window > 0 && window <= max_length / 2)) return false;
  return max_length > (float_cache || p.rows != kAttentionRows ? 256u : tokens > batch ? 512u : 1024u);
}

// Whether few lanes sum the pieces of a row one after the other, or a workgroup those of 64 values of one, which is for more pieces than kFewPieces and no more workgroups than kJoinGroups (8 bits and float32, 9 to
// 16 pieces: heads of 256, 160 to 320 rows 0.89 of the time in all, more rows 0.83, heads of 128 over 320 rows 0.90; up to 64 rows 1.00 to 1.05, 17 to 32 pieces of heads of 64 1.11).
constexpr unsigned kFewPieces = 8, kJoinGroups = 512;
inline bool attention_joins_few(unsigned splits, uint64_t rows, unsigned size) { return splits <= kFewPieces || rows * ((size + 63) / 64) > kJoinGroups; }

}  // namespace tfcc_rocm
