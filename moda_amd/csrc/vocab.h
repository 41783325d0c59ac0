// Argument blocks of the two ends of a language model: rows of an embedding by tokens and their gradient (embed_kernel.hip), the
// cross entropy of rows over a vocabulary and its gradients (vocab_loss_kernel.hip, product.h).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace moda {

// Tokens or targets, int32 or int64.  What they hold is known to the device alone: a number outside 0 .. vocab - 1, or the ignored
// one, is no word.
struct Words {
  const void* at;
  int64_t n, vocab, ignored;  // (ignored: -1 where nothing is besides what is outside)
  int wide;                   // int64
  __device__ __forceinline__ int of(int64_t i) const {  // the word, or -1
    const int64_t t = wide ? ((const int64_t*)at)[i] : (int64_t)((const int32_t*)at)[i];
    return (uint64_t)t < (uint64_t)vocab && t != ignored ? (int)t : -1;
  }
};

// ---------------------------------------------------------------------------------------------------------------------
// embedding
// ---------------------------------------------------------------------------------------------------------------------
struct EmbedArgs {
  Words words;
  const char* weight;  // forward: [vocab][width]; backward: dy [n][width]
  char* y;             // forward: [n][width]; backward: the weight's gradient [vocab][width]
  int64_t ld_in, ld_out;
  int64_t width;
  float scale;
  int lane_shift;  // 2^lane_shift lanes share a row
  // backward: words and places in the order of words, where a word's places are in it, the partial sums of long runs
  const uint32_t *keys, *places;
  const int2* range;
  float* parts;
  int64_t part_ld;
  int chunks;
  int cleared;  // ranges of words that are not there are empty (else whatever their memory held)
  unsigned chunk_blocks;
};

// The order of words: passes over digits of their number, lowest first, each stable.  A block of kSortThreads * rounds tokens counts its
// digits; a second launch places them.
constexpr int kDigitBits = 9, kDigits = 1 << kDigitBits, kSortThreads = 1024, kMostSortBlocks = 128;
constexpr int kFewRounds = 4, kFewTokens = kSortThreads * kFewRounds;  // as many one workgroup sorts by itself
struct SortArgs {
  Words words;
  const uint32_t *keys, *places;  // NULL in the first pass: the words themselves
  uint32_t *keys_out, *places_out;
  uint32_t* counts;  // [blocks][kDigits]
  int2* range;       // [vocab]: first place and end of the words that there are
  int rounds, blocks, shift;
};

// Rows of a run that are added up in one go; a word of more has its run cut at multiples of this (its parts are joined by a second launch).
constexpr int kRunRows = 32;

struct EmbedGradPlan {
  int passes, rounds, blocks;
  int64_t chunks, part_ld;  // pieces of kRunRows sorted places; floats of a part
  size_t keys[2], places[2], counts, range, parts, bytes;
};
inline EmbedGradPlan plan_embed_grad(int64_t n, int64_t vocab, int64_t width) {
  EmbedGradPlan p = {};
  int bits = 1;  // of the numbers 0 .. vocab, the last of which stands for no word
  while (bits < 32 && (vocab >> bits) != 0) bits++;
  p.passes = (bits + kDigitBits - 1) / kDigitBits;
  p.rounds = (int)((n + (int64_t)kSortThreads * kMostSortBlocks - 1) / ((int64_t)kSortThreads * kMostSortBlocks));
  if (p.rounds < 1) p.rounds = 1;
  p.blocks = (int)((n + (int64_t)kSortThreads * p.rounds - 1) / ((int64_t)kSortThreads * p.rounds));
  p.chunks = (n + kRunRows - 1) / kRunRows;
  p.part_ld = (width + 3) / 4 * 4;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t from = at;
    at += (bytes + 255) / 256 * 256;
    return from;
  };
  for (int i = 0; i < 2; i++) {
    p.keys[i] = take(n * sizeof(uint32_t));
    p.places[i] = take(n * sizeof(uint32_t));
  }
  p.counts = take((size_t)p.blocks * kDigits * sizeof(uint32_t));
  p.range = take((size_t)vocab * sizeof(int2));
  p.parts = take((size_t)p.chunks * 2 * p.part_ld * sizeof(float));
  p.bytes = at;
  return p;
}

// ---------------------------------------------------------------------------------------------------------------------
// cross entropy over a vocabulary
// ---------------------------------------------------------------------------------------------------------------------

// What the device alone knows of a call: how many rows have a target, and by what the two products that read the gradient of the logits
// are multiplied.
struct LossHead {
  int live;
  int splits;  // of the words where the gradient of the rows is added up in fp32 (SplitRule)
  float down;
};

// What choose_tiling's estimate needs where the device chooses the splits (vocab_loss_kernel.hip: gather_rows_kernel).
struct SplitRule {
  int tile_p, tiles_f, steps, at_once, most;  // a tile's rows, tiles of columns, steps of 64 words, workgroups; splits that there is room for at all rows
  float step_us, end_us, split_us;            // of a step, an item, a split of one row
};

// Rows with a target, one behind the other: their numbers, targets, factors and log sums, and the rows themselves as the products read
// them (`planes` of 16-bit elements whose sum a row is, each [rows][x_ld], zeros behind a row's end).
struct GatherArgs {
  Words words;
  const char* x;
  int64_t ld_x, width;
  LossHead* head;
  int *row_of, *target;
  uint16_t* rows;
  int64_t rows_ld, rows_plane;
  // of 1024 targets each, where there are many: rows with a target, the largest upstream gradient among them (bits of a float)
  int *counts, *largest;
  // forward: zeros for the rows without
  float *loss, *lse_out;
  // backward
  const float *d_loss, *lse_in;
  int64_t d_loss_stride;  // 0: one for all
  float *factor, *lse;
  SplitRule rule;
  char* dx;  // zeros for the rows without (or NULL)
  int64_t ld_dx;
  float up;  // the gradient of the logits is kept this many times as large
  int mean, vec_x, vec_dx;
};

struct LayArgs {  // rows of a matrix as the products read them
  const char* x;
  int64_t ld_x, width, rows;
  uint16_t* to;
  int64_t to_ld, to_plane;
  int vec;
};

// out[p][f] = sum_k P(p, k) F(f, k) and what is done with it (vocab_loss_kernel.hip).
struct ProductArgs {
  const uint16_t *f, *p;
  int64_t f_ld, p_ld, f_plane, p_plane;
  int f_count, p_count, k_count;  // of which live rows are known to the device
  const LossHead* head;           // NULL: every row counts
  int splits;                     // of the summation axis
  float c;                        // logits in base 2
  Words words;                    // targets where there is no head
  const int *target, *row_of;
  int first_word, rows;
  float2* stats;  // [tiles of words][rows]: largest logit, sum of the exponentials from there
  float* target_logit;
  int64_t stats_ld;
  const float *factor, *lse;
  uint16_t* dz;
  int64_t dz_ld, dz_plane;
  float* acc;  // [splits][rows][acc_ld] in fp32 (kGradRows: the live rows), or NULL: the result itself to out
  int64_t acc_ld, acc_split;
  int add;
  char* out;
  int64_t out_ld;
  int out_vec, out_by_eight;  // four, eight neighbouring results may be stored as one
  float scale;
};

struct JoinStatsArgs {
  const float2* stats;  // of one piece of the vocabulary
  const float* target_logit;
  int64_t stats_ld, tiles;
  float2* carry;  // [rows]: of the pieces before it, then with it (or NULL: one piece is all)
  int first, last;
  const LossHead* head;
  Words words;
  const int* row_of;
  float *loss, *lse;
};

struct JoinSumsArgs {
  const float* acc;
  int64_t acc_ld, acc_split, rows, width;
  int splits;
  const LossHead* head;
  int by_head;  // rows are the live ones, and go to row_of
  const int* row_of;
  char* out;
  int64_t out_ld;
  int out_vec;
  float scale;
};

struct LossTotalArgs {
  const float* rows;
  float* total;
  Words words;
  const LossHead* head;
  int mean;
};

// Tiles of a product, f x p: 256 x 256, 128 x 128, for few rows 128 x 32, for small products 64 x 64.
enum ProductTile { kTileLarge, kTileMedium, kTileRows, kTileSmall };
struct Tiling {
  ProductTile tile;
  int splits;
};
inline int tile_f(ProductTile t) { return t == kTileLarge ? 256 : t == kTileSmall ? 64 : 128; }
inline int tile_p(ProductTile t) { return t == kTileLarge ? 256 : t == kTileMedium ? 128 : t == kTileSmall ? 64 : 32; }

// The tile whose launch takes the least time by this estimate: what the busiest workgroup does -- its tiles' steps of 64 of the summation axis, and
// a start and end of each -- and where the axis is split, a launch more and the sums' way to memory and back.  Measured (8192 x 32000 x 2048,
// bf16): a step of the large tile 1.65 us, of two medium ones on a compute unit 1.04 (of one 0.85), of two for few rows 0.51, of three
// small ones 0.7; ends 2.5 to 4 us.
// 1638 rows, 50257 words, width 768: 146 us by large tiles, 160 by medium ones (estimated 143, 155); 80 rows, width 512: 15.4 medium, 18.6 few.
struct TileTimes {
  ProductTile tile;
  double at_once, step_us, alone_us, end_us;
};
constexpr TileTimes kTileTimes[4] = {
    {kTileLarge, 256, 1.65, 1.65, 4}, {kTileMedium, 512, 1.04, 0.85, 3}, {kTileRows, 512, 0.51, 0.45, 2.5}, {kTileSmall, 768, 0.7, 0.45, 2.5}};
inline Tiling choose_tiling(int64_t p, int64_t f, int64_t steps, bool may_split, bool may_few) {
  Tiling best = {kTileMedium, 1};
  double least = 1e30;
  for (const auto& k : kTileTimes) {
    if (k.tile == kTileRows && !may_few) continue;
    const int64_t tiles = ((p + tile_p(k.tile) - 1) / tile_p(k.tile)) * ((f + tile_f(k.tile) - 1) / tile_f(k.tile));
    for (int s = 1; s <= 64; s *= 2) {
      if (s > 1 && (!may_split || steps < 4 * s)) break;
      const double items = (double)tiles * s, rounds = (double)((int64_t)((items + k.at_once - 1) / k.at_once));
      const double us = rounds * ((double)((steps + s - 1) / s) * (items <= 256 ? k.alone_us : k.step_us) + k.end_us) +
                        (s > 1 ? 4 + (double)s * p * f * 8 / 5e6 : 0);
      if (us < least) {
        least = us;
        best = {k.tile, s};
      }
    }
  }
  return best;
}

struct LossPlan {
  bool direct;       // rows read where they are: few of them, 16 bits, on the grid
  bool copy_weight;  // the weight is laid out anew, piece by piece
  int planes;
  int64_t rows_ld, weight_ld, k;  // columns of the products' operands
  int64_t piece, pieces;          // words at once
  int64_t dz_ld;
  Tiling logits, grad_rows, grad_weight;
  int64_t stat_tiles, acc_ld;  // stat_tiles: of a piece
  bool acc_rows;  // the gradient of the rows is added up in fp32, split by the rows that have a target (else not split, however few they are)
  size_t head, row_of, target, factor, lse, target_logit, counts, largest, stats, carry, rows, weight, dz, dx_acc, dw_acc, losses, bytes;
};

constexpr int64_t kGatherBlock = 8, kCountBlock = 1024, kScanMost = 4096;

// Rows that are scored where they are, those without a target too: forward, bf16, 512 rows in place against 513 gathered, all with a target: 23
// against 27 us (4099 words, width 1000), 54 against 64 (50257, 768), 453 against 600 (131072, 4096; a row of tiles more).  Where few have one the gather is
// the better, by more the larger the product is: nine in ten without: 22.5 against 20, 53 against 30, 447 against 230.
constexpr int64_t kDirectRows = 512;

// grid16: x lies on the 16-byte grid (its rows may be read in place); weight16: the weight does
inline LossPlan plan_loss(int64_t n, int64_t vocab, int64_t width, bool fp32, bool grid16, bool weight16, bool backward, bool want_dx, bool want_dw,
                          bool reduce) {
  LossPlan p = {};
  p.planes = fp32 ? 3 : 1;
  p.copy_weight = fp32 || !weight16;
  p.direct = !backward && !fp32 && grid16 && weight16 && n <= kDirectRows;
  p.rows_ld = (width + 63) / 64 * 64;
  p.weight_ld = p.copy_weight ? p.rows_ld : 0;
  p.k = p.copy_weight ? p.rows_ld : width;
  // pieces: what a pass keeps of one (a copy of its weights, the gradient of its logits) stays within a GiB each
  const int64_t budget = 1ll << 30;
  int64_t most = vocab < 1 << 21 ? vocab : 1 << 21;  // (rows of the logits' gradient are reached by 32-bit offsets)
  const int64_t tiles_p = (n + 31) / 32, by_grid = (1ll << 22) / (tiles_p > 0 ? tiles_p : 1) * 128 / 256 * 256;
  if (most > by_grid) most = by_grid > 256 ? by_grid : 256;
  const auto within = [&](int64_t bytes_a_word) {
    const int64_t words = budget / bytes_a_word / 256 * 256;
    most = most < words ? most : words > 256 ? words : 256;
  };
  if (p.copy_weight) within(p.rows_ld * 2 * p.planes);
  if (backward) within((n > 0 ? n : 1) * 2 * p.planes);
  p.pieces = (vocab + most - 1) / most;
  p.piece = p.pieces == 1 ? vocab : ((vocab + p.pieces - 1) / p.pieces + 255) / 256 * 256;
  p.pieces = (vocab + p.piece - 1) / p.piece;
  p.dz_ld = (p.piece + 63) / 64 * 64;
  const int pairs = fp32 ? 6 : 1;
  p.logits = choose_tiling(n, p.piece, (p.k + 63) / 64 * pairs, false, true);
  p.stat_tiles = (p.piece + tile_f(p.logits.tile) - 1) / tile_f(p.logits.tile);
  p.acc_ld = p.rows_ld;
  p.grad_rows = choose_tiling(n, width, (p.piece + 63) / 64 * pairs, true, true);
  p.grad_weight = choose_tiling(p.piece, width, (n + 63) / 64 * pairs, true, false);
  p.acc_rows = p.pieces > 1 || p.grad_rows.splits > 1;
  size_t at = 0;
  auto take = [&](bool needed, int64_t bytes) {
    const size_t from = at;
    if (needed) at += ((size_t)bytes + 255) / 256 * 256;
    return from;
  };
  const bool gathers = !p.direct;
  p.head = take(gathers, sizeof(LossHead));
  p.row_of = take(gathers, n * 4);
  p.target = take(gathers, n * 4);
  p.factor = take(backward, n * 4);
  p.lse = take(backward, n * 4);
  p.counts = take(gathers && n > kScanMost, (n + kCountBlock - 1) / kCountBlock * 4);
  p.largest = take(gathers && n > kScanMost, (n + kCountBlock - 1) / kCountBlock * 4);
  p.rows = take(gathers, n * p.rows_ld * 2 * p.planes);
  p.weight = take(p.copy_weight, p.piece * p.rows_ld * 2 * p.planes);
  p.target_logit = take(!backward, n * 4);
  p.stats = take(!backward, p.stat_tiles * n * 8);  // (of a piece, which by_grid bounds: 2 GiB at most)
  p.carry = take(!backward && p.pieces > 1, n * 8);
  p.losses = take(!backward && reduce, n * 4);
  p.dz = take(backward, n * p.dz_ld * 2 * p.planes);
  p.dx_acc = take(backward && want_dx && p.acc_rows, p.grad_rows.splits * n * p.acc_ld * 4);
  p.dw_acc = take(backward && want_dw && p.grad_weight.splits > 1, p.grad_weight.splits * p.piece * p.acc_ld * 4);
  p.bytes = at;
  return p;
}

}  // namespace moda
