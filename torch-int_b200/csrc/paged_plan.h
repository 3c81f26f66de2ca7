// How a call of paged_attention is cut into CTAs: host arithmetic on sizes and bounds alone, without CUDA, so that it can
// be compiled and tested by itself.
#pragma once
#include <stdint.h>

namespace ti {

constexpr int PAGED_SMS = 148;
constexpr int STEP = 32;            // keys of a step of paged_rows_kernel: two groups of 16
constexpr int MAX_CLUSTER = 8;

// CTAs of paged_rows_kernel an SM holds: registers (147 per thread of 128-wide heads) and the queues' 16 KB a warp.
constexpr int rows_ctas_per_sm(int head_dim, int nt, int warps) {
  return (head_dim == 128 ? (nt == 1 ? 12 : 8) : (nt == 1 ? 16 : 12)) / warps;
}

// How the tile kernel (paged_attention_sm100.cu) cuts the work.
struct PagedTilePlan {
  int tokens_per_tile;  // of 128 rows: 128 / group
  int pairs;            // pairs of row tiles of the largest sequence
  int chunk;            // keys of a split, a multiple of 128
  int splits;
};

constexpr int TILE_ROWS = 128;  // rows of a row tile of paged_tiles_kernel
// Rows up to which a sequence is served by paged_rows_kernel, in tiles of 16 that each read the keys.  16 sequences of 2000
// keys, 32 query heads on 8 of 128: 8 new tokens (32 rows) 27 us so and 51 by paged_tiles_kernel; 12 (48 rows) 45 both;
// 48 rows of 32 key heads 144 and 106.
// Beside longer sequences half as many: 16 decoding sequences and a prompt take 82 us so, 88 with the empty tiles of 32 rows.
constexpr int FEW_ROWS = 32, FEW_BESIDE = 16;
constexpr int MIN_CHUNK = 256, MAX_CHUNK = 2048;  // keys of a split of paged_rows_kernel
constexpr int64_t MAX_PARTIAL_BYTES = 512ll << 20;
constexpr int64_t MAX_KEYS = (1 << 30) - 4096;  // a position plus a split stays within 31 bits

// How a call is cut.  Sequences with at most `few` rows per key head are served by paged_rows_kernel, the others by
// paged_tiles_kernel; a kernel is left out where the bounds show that no sequence needs it.
struct PagedPlan {
  bool rows, tiles;
  int few;
  int nt, warps;                         // rows kernel: 8-row tiles and warps of a CTA
  int row_tiles, chunk, row_splits;      // CTAs of a sequence, keys of a split
  bool cluster;                          // the splits of the rows kernel are a cluster
  PagedTilePlan tile;
  int splits;                            // most splits that go through the workspace: stride of the partial results
};

inline int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
inline int64_t div_up(int64_t x, int64_t m) { return (x + m - 1) / m; }

// `rows_only`, if not 0: every sequence is served by paged_rows_kernel, in at most so many splits.
inline PagedPlan make_plan(int64_t batch, int64_t tokens, int64_t group, int64_t kv_heads, int head_dim, int64_t max_query_len,
                           int64_t max_kv_len, int64_t rows_only = 0) {
  PagedPlan pl = {};
  const int64_t rows = max_query_len * group;
  pl.few = group > TILE_ROWS || rows_only > 0 ? 0x7FFFFFFF : FEW_ROWS;
  pl.tiles = rows > pl.few;
  if (pl.tiles) pl.few = FEW_BESIDE;
  // the shortest sequence brings at least the tokens that the others cannot hold
  const int64_t shortest = tokens - (batch - 1) * max_query_len;
  // (beside a prompt, tokens with more heads on a key head than `few` are the tile kernel's: no rows kernel is needed)
  pl.rows = !pl.tiles || (group <= pl.few && shortest * group <= pl.few);
  pl.splits = 1;
  // Bounds far above the lengths would ask for gigabytes of partial results that nobody writes (64 sequences bound to
  // 131072 keys with a prompt of 2048 tokens, 64 heads: 4.5 GB): fewer and longer splits there.
  int64_t most_splits = MAX_PARTIAL_BYTES / (tokens * group * kv_heads * (head_dim * 4 + 8));
  if (rows_only > 0 && rows_only < most_splits) most_splits = rows_only;
  if (pl.rows) {
    const int64_t most = rows < pl.few ? rows : pl.few;
    // Beside a prompt the sequences with few rows mostly have a single token: tiles of 8 rows where that is enough for its
    // heads, 16 otherwise and where every sequence may have more.
    const int64_t usual = pl.tiles && group <= 8 ? group : most;
    pl.nt = usual <= 8 ? 1 : 2;
    pl.row_tiles = static_cast<int>(div_up(most, 8 * pl.nt));
    // One CTA per unit where that fills the SMs, in pieces of at most MAX_CHUNK keys (sequences of unequal lengths:
    // 64 contexts of up to 8192 keys took 94 us in pieces of 1024 to 2048 keys, 102 in whole).  Otherwise as many pieces
    // as fill the SMs once (two contexts of 131072 keys: 82 us so, 110 with a third more pieces), of at least MIN_CHUNK
    // keys (one context of 2000 keys, 56 heads: 8.1 us in pieces of 288, 9.9 of 512).
    const int64_t units = batch * kv_heads * div_up(usual, 8 * pl.nt), slots = PAGED_SMS * rows_ctas_per_sm(head_dim, pl.nt, 4);
    int64_t chunk = units >= slots ? MAX_CHUNK : round_up(div_up(max_kv_len, slots / units), STEP);
    if (chunk < MIN_CHUNK) chunk = MIN_CHUNK;
    // Small calls are bound by the steps a warp takes one after another: where a CTA per SM leaves it at most two, its eight
    // warps beat several CTAs of four (16 contexts of 500 keys, 8 key heads: 5.5 us, 8.3 with four warps; 4 of 1000: 5.1 and
    // 6.8; two steps are better than a join for the narrow heads: one context of 500 keys 3.9 us whole, 4.3 in two parts).
    // But a cluster of eight such CTAs takes eight SMs of one GPC, and few of those are free at a time (two contexts of 2000
    // keys, 8 key heads: 9.4 us, 6.6 with four warps): more than four only where they are half the SMs at most.
    const int64_t alone = div_up(max_kv_len, units <= PAGED_SMS ? PAGED_SMS / units : 1);
    const int64_t chunk8 = alone > 256 || (head_dim < 128 && max_kv_len <= 512) ? 512 : 256, parts8 = div_up(max_kv_len, chunk8);
    const bool eight = !pl.tiles && units <= PAGED_SMS && alone <= 512 &&
                       (parts8 <= 4 || parts8 > MAX_CLUSTER || units * parts8 <= PAGED_SMS / 2);
    // Up to two units per SM: two CTAs of all the warps that fit, each unit in one piece (six of 128-wide heads: 32 contexts
    // of 1000 keys, 8 key heads, 15.8 -> 14.2 us, of up to 8000 keys 75 -> 61; eight of the others: 8 of 500, 32 x 64,
    // 6.2 -> 5.3).  The narrow heads also where that takes two rounds: the longest of unequal contexts then ends sooner
    // (16 of up to 2000, 32 x 80: 23.3 -> 20.6 us; 12 of up to 2000, 32 x 64: 19.2 -> 18.4), which is what equal ones lose
    // (29.7 -> 32.2; 12.7 both).  Of 128-wide heads equal ones lose more (336 units: 12.7 -> 16.3 us).
    const int64_t pieces = slots / units;
    const bool two = pl.nt == 1 && !pl.tiles && (head_dim == 128 ? pieces == 1 && units <= 2 * PAGED_SMS : pieces == 1 || pieces == 2);
    if (two) chunk = round_up(max_kv_len > 0 ? max_kv_len : 1, STEP);
    if (eight) chunk = chunk8;
    if (div_up(max_kv_len, chunk) > most_splits) chunk = round_up(div_up(max_kv_len, most_splits > 1 ? most_splits : 1), STEP);
    pl.chunk = static_cast<int>(chunk);
    pl.row_splits = static_cast<int>(max_kv_len > chunk ? div_up(max_kv_len, chunk) : 1);
    // Three warps to a CTA instead of four where the work then runs in fewer rounds, by more than each takes longer:
    // 8 sequences of 512 keys, 56 heads (448 units; 444 CTAs of four warps at a time, 592 of three): 21.0 -> 17.8 us.
    const int64_t slots3 = PAGED_SMS * rows_ctas_per_sm(head_dim, pl.nt, 3);
    const bool three = pl.nt == 1 && pl.row_splits == 1 && 4 * div_up(units, slots3) < 3 * div_up(units, slots);
    pl.warps = eight ? 8 : two ? (head_dim == 128 ? 6 : 8) : three ? 3 : 4;
    // a cluster holds its CTAs until the last one is done: only where all of them run at once
    pl.cluster = pl.row_splits > 1 && pl.row_splits <= MAX_CLUSTER && units * pl.row_splits <= slots;
    if (!pl.cluster) pl.splits = pl.row_splits;
  }
  if (pl.tiles) {
    pl.tile.tokens_per_tile = static_cast<int>(TILE_ROWS / group);
    pl.tile.pairs = static_cast<int>(div_up(max_query_len, 2 * pl.tile.tokens_per_tile));
    // The keys are split where that makes the last round of CTAs shorter: rounds of (1.8 us per key tile + 4 us of fixed
    // costs), as measured, against the partial results' way through memory (written and read at 5 TB/s, 6 us for the
    // joining kernel).  One prompt of 512 tokens behind 3488, 32 query heads: 64 items of 32 key tiles on 148 SMs take 65 us
    // whole, 48 in two parts, 52 in four; 16 items (8 query heads) 65 whole, 28 in four parts, 21.5 in nine; a chunk of 2048
    // behind 14336 tokens (256 items) 449 whole, 500 and 458.  Sequences with few rows run on the SMs left free, so their
    // share (at their bounds and 6.5 TB/s) counts as occupied SMs: the 512 tokens with 15 decoding sequences
    // beside them take 74 us whole and 80 in two parts.
    // The items are estimated from the number of tokens: of a batch that mixes a prompt with decoding sequences, the
    // bounds alone would count every sequence as a prompt.
    const int64_t by_tokens = div_up(tokens, 2 * pl.tile.tokens_per_tile), by_bounds = batch * pl.tile.pairs;
    const int64_t units = kv_heads * (by_tokens < by_bounds ? by_tokens : by_bounds), tiles = div_up(max_kv_len, 128);
    const double beside = pl.rows ? static_cast<double>((batch - 1) * max_kv_len * kv_heads) * head_dim * 2 / 6.5e6 : 0.0;
    double best = 0;
    for (int64_t n = 1; n <= 64 && (n == 1 || (n <= tiles && n <= most_splits)); ++n) {
      if (n > 1 && units * (n - 1) >= 4 * PAGED_SMS) break;  // four rounds and more: finer parts have nothing to fill
      const int64_t part = div_up(tiles, n);
      if (n > 1 && div_up(tiles, part) != n) continue;  // the same parts as a smaller n
      const double item = 1.8 * static_cast<double>(part) + 4.0, alone = static_cast<double>(div_up(units * n, PAGED_SMS)) * item;
      const double shared = static_cast<double>(units * n) * item / PAGED_SMS + beside;
      const double us = (alone > shared ? alone : shared) +
                        (n > 1 ? 6.0 + static_cast<double>(tokens * group * kv_heads * n) * head_dim * 8 / 5e6 : 0.0);
      if (n == 1 || us < best) {
        best = us;
        pl.tile.chunk = static_cast<int>(part > 0 ? part * 128 : 128);
        pl.tile.splits = static_cast<int>(n);
      }
    }
    if (pl.tile.splits > pl.splits) pl.splits = pl.tile.splits;
  }
  return pl;
}

inline int64_t partial_bytes(const PagedPlan& pl, int64_t tokens, int64_t q_heads, int64_t head_dim) {
  return pl.splits == 1 ? 0 : tokens * q_heads * pl.splits * (head_dim * 4 + 8);
}

// paged_tiles_kernel keeps its scores relative to an fp32 number of about |scale_log2| * 1.5 * 2^23, whose spacing moves
// the largest exponent, meant to be 7, by up to |scale_log2|: at 4 it stays within 3 .. 11 of the 15 that fp16 holds, at
// 12 it would pass them.  Steeper factors (a unit of q . k is then worth more than 2^4) are left to paged_rows_kernel,
// whose exponents cannot pass 15; it needs no larger workspace for them than the sizes alone ask for.  Eight prompts of 512, 56
// heads x 128: 316 us so, 64 by paged_tiles_kernel with an ordinary factor.
constexpr float MAX_TILE_SCALE = 4.f;

inline PagedPlan make_plan_for_scale(int64_t batch, int64_t tokens, int64_t group, int64_t kv_heads, int head_dim,
                                     int64_t max_query_len, int64_t max_kv_len, float scale_log2) {
  const PagedPlan pl = make_plan(batch, tokens, group, kv_heads, head_dim, max_query_len, max_kv_len);
  if (!pl.tiles || (scale_log2 >= -MAX_TILE_SCALE && scale_log2 <= MAX_TILE_SCALE)) return pl;
  return make_plan(batch, tokens, group, kv_heads, head_dim, max_query_len, max_kv_len, pl.splits);
}

// The launch of paged_combine_kernel, which joins the partial results of a plan with splits > 1.
struct PagedJoin {
  bool by_token;   // a row per block of the call, not of the longest sequence
  bool many;       // four warps to a row, not one
  int64_t blocks;  // in x
};

inline PagedJoin plan_join(const PagedPlan& pl, int64_t batch, int64_t tokens, int64_t q_heads, int64_t group, int64_t max_query_len) {
  PagedJoin j;
  // only the rows of few-row sequences have partial results where the tile kernel does not split
  const int64_t few_tokens = pl.few / group;
  const int64_t longest = pl.tiles && pl.tile.splits == 1 && few_tokens < max_query_len ? few_tokens : max_query_len;
  // A row per block of the call where most rows of a longest sequence each would be empty (a prompt of 512 tokens in a
  // batch of 16: 226 us with a block for every row that the bounds allow).
  j.by_token = longest * batch > 2 * tokens && batch <= 1024 && tokens * q_heads <= 0x7FFFFFFF;
  j.many = pl.splits > 8;
  const int64_t rows = (j.by_token ? tokens : longest) * q_heads;
  j.blocks = j.many ? rows : div_up(rows, 4);
  return j;
}

}  // namespace ti
