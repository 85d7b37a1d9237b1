// Launch descriptors of the paged key/value cache: the step plan, the append, the attention over
// pages and the page bookkeeping, shared by their kernels and the C-ABI layer.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "va_kernels.h"

namespace va {

constexpr int kPagedMaxSeqs = 4096;  // sequences of a step
constexpr int kPageMin = 16, kPageMax = 256;

// Work items of a step: rows (token, query head of the group) of one sequence and key/value head,
// flattened token by token. Up to kPagedFewRows of them are one tile whose waves share the keys out;
// more are tiles of kPagedTileRows, a strip of 32 per wave (in short steps tiles of kPagedFewRows, see below).
constexpr int kPagedFewRows = 32;
constexpr int kPagedTileRows = 128;
constexpr int kPagedChunkKeys = 64;  // key ranges are split at multiples of this
// The attention's work-groups: 8 waves, one work-group per CU, for steps with prompts (more rows than
// sequences) of up to this many tiles x heads, by the sizes that the host knows; 4 waves, two per CU,
// for the others. us with 4 / 8 waves: 2 x 2048 tokens, 12/2 heads (388 tiles) 51 / 42; 4096 tokens
// (386) 88 / 72; 8 x 300 on 700 (240) 27.5 / 26; two chunks of 512 beside 62 answers, 28/4 heads (492) 60 /
// 59; 2 x 1024 on 500 (456) 46.5 / 47.5; 3 x 1024 (684) 62 / 67; 4 x 1024 (912) 78 / 82; four chunks of
// 2048 623 / 680; 64 answers of 64 to 8192 tokens 30.4 / 32.0, 16 of 1500 12.1 / 12.8, four of 512 7.9
// / 7.5. Steps of few prompt tiles over ranges that are split take 4 waves too, and twice the parts:
// two work-groups of a CU wait for different barriers. us, 8 waves and 256 parts / 4 and 512, 28/4
// heads: 16 trees of 24 on 4000 75 / 53, 8 of 48 to 64 on 28,672 to 32,768 305 / 268, 512 new tokens on
// 8192 98 / 86, on 4096 55 / 55, 1024 new ones (the table's bound 228) on 4096 106 / 106, 8 x 300 on
// 700, 12/2 heads (240) 29 / 39.
// Sequences of a few tiles each, as long as each other, that are more items than CUs, take 4 waves: with 8 the
// last ones begin when the first have ended. us, 8 / 4: 36 trees of 24 on 500, 28/4 heads (288 items) 29.4 / 21.4, 40
// on 1200 52 / 40, 100 on 1500, 12/2 heads (400) 64 / 50; 32 on 64 to 8192, 28/4 heads (256) 40 / 45; prompts of
// kPagedLongTiles tiles and more differ in their tiles' ranges (above).
constexpr int kPagedWideTiles = 512, kPagedSplitTiles = 200, kPagedWidePlaces = 256, kPagedLongTiles = 4;
// Parts that a step's keys are split into, by kind of tile, the shortest part (but a range's last) and
// the longest table row that is never split. us at 384 / 512 / 1024 few-row parts: 64 answers of 64 to
// 8192 tokens, 12/2 heads 34 / 30 / 32, four of 65,536, 28/4 heads 103 / 97 / 100; shortest few-row part
// 128 / 256 / 512: one answer of 8192 9.0 / 9.8 / 11.5, 16 of 1500 13.4 / 12.1 / 12.6. At 256 / 512
// prompt parts: two chunks of 512 beside 62 answers 57 / 76, 128 new tokens on 32,768 80 / 94. Four answers
// of 512, table rows of 576: split 8.5, whole 7.9 and a launch less.
// Prompt tiles that are as many as the card has places (tiles x heads) are split where they are longer
// than the average one, into up to kPagedMostParts parts: 64 trees of 24 tokens on 64 to 8192, 28/4
// heads (512 items) 162 -> 59 us and 3 more to merge, 16 chunks of 64 to 2048 on 64 to 16,384 349 ->
// 220. Where answers follow, which fill the places that shorter items leave, at twice the average: two
// chunks of 512 beside 62 answers 58 us, 67 at the average. Steps of prompts of one length are not
// split by it. (What passes kPagedManyParts, few-row tiles go without, so that the room for items is
// the same.)
constexpr int kPagedFewParts = 512, kPagedManyParts = 256, kPagedMostParts = 512;
// Prompt parts are shorter than kPagedManyKeys, down to kPagedFewKeys, while that makes no more than
// kPagedShortItems of them (us with the merge, 512 / shorter: 300 new tokens on 700, 12/2 heads 19.6 /
// 16.5; with 384 items 512 on 1536 23.3 / 27.3, two of 64 on 8000 25.3 / 28.0).
constexpr int kPagedFewKeys = 256, kPagedManyKeys = 512, kPagedShortItems = 192;
constexpr int kPagedWholeKeys = 1024;
// Short steps: prompt tiles over table rows that are not split are of kPagedFewRows rows too, whose waves share
// the keys out, where that makes no more items than there are CUs (8 waves each), or up to twice as many (4
// waves, two work-groups per CU) of sequences of kPagedNarrowTiles such tiles or more. us, 128 rows / 32: four
// trees of 16 on 512, 12/2 heads 14.6 / 10.6, 28/4 15.4 / 10.6; 32 of 16 on 800 19.6 / 17.3; 128 new tokens on
// 800 19.5 / 12.3; two prompts of 512 (388 items) 14.1 / 11.7, one of 900 19.7 / 14.1, 8 x 64 on 600, 28/4 heads
// (480) 17.8 / 16.1. Sequences of fewer tiles, which read their keys as often as more work-groups hold them:
// 48 trees of 16 on 500 (384) 15.2 / 18.7, 24 x 32 on 900 (336) 21.3 / 23.1. (4 waves for up to 256 items: 8.6
// for 9.3 at 64 new tokens on 200, 13.5 for 12.4 at 16 x 8 on 900.)
constexpr int kPagedNarrowItems = 256, kPagedNarrowTiles = 8;
constexpr int kPagedPadRows = 64;     // padding rows that one item zeroes

// A step's plan, int32 words: cu (n_seqs + 1) row offsets of the sequences, the sequence (-1: padding)
// and the position of every row, the counts of items and merge records, the items, the records.
constexpr int kPagedItemWords = 12, kPagedMergeWords = 8;
struct PagedLayout {
  int64_t seq, pos, counts, items, merges, words;  // offsets; cu lies at 0
  int64_t max_items, max_merges, max_part_rows;
  int many_parts;  // parts of prompt tiles at most, and
  int many_base;   // where there are fewer of them than that, and no few-row tiles
  bool wide, narrow;
};
inline int64_t up4(int64_t x) { return (x + 3) & ~int64_t(3); }
// Bounds: a sequence with rows makes one tile, and one more per full kPagedTileRows (kPagedFewRows if narrow). A kind's parts have
// at least its total (tiles times the longest of the sequence) / its number of parts keys, so the
// tiles of a sequence of n > 1 parts stand for more than n - 1 >= n / 2 of them each, and all split
// tiles have at most twice as many parts; each part holds at most the kind's rows, and a row is in at
// most max_keys / kPagedFewKeys + 1 parts. A merge record takes 8 rows, or one of more than 8 parts (of 32
// in a prompt tile), which are then as many as the tile's rows by 4 (by 16) and more.
inline PagedLayout paged_layout(int64_t n_seqs, int64_t n_tokens, int64_t hq, int64_t hkv,
                                int64_t max_keys) {
  PagedLayout l;
  const bool split = max_keys > kPagedWholeKeys, prompts = n_tokens > n_seqs;
  const int64_t rows = n_tokens * hq, seqs = n_seqs < n_tokens ? n_seqs : n_tokens;
  const int64_t short_tiles = n_tokens * (hq / hkv) / kPagedFewRows, short_items = (seqs + short_tiles) * hkv;
  const bool fits = short_items <= kPagedNarrowItems;
  l.narrow = prompts && !split &&
             (fits || (short_items <= 2 * kPagedNarrowItems && short_tiles >= kPagedNarrowTiles * seqs));
  const int64_t tiles = seqs + (l.narrow ? short_tiles : n_tokens * (hq / hkv) / kPagedTileRows);
  const bool few = prompts && split && tiles * hkv <= kPagedSplitTiles;
  const int64_t each = seqs == 0 ? 0 : (n_tokens * (hq / hkv) + seqs * kPagedTileRows - 1) / (seqs * kPagedTileRows);
  const bool placed = seqs * each * hkv <= kPagedWidePlaces || each >= kPagedLongTiles;
  l.wide = prompts && !few && (l.narrow ? fits : tiles * hkv <= kPagedWideTiles && placed);
  const int64_t fit = n_tokens * (hq / hkv) / (kPagedFewRows + 1);  // (prompt tiles, of more rows each)
  const int64_t its = (fit < tiles ? fit : tiles) * hkv;
  const int64_t many = few || its > kPagedMostParts ? kPagedMostParts : its < kPagedManyParts ? kPagedManyParts : its;
  l.many_parts = (int)many;
  l.many_base = few ? kPagedMostParts : kPagedManyParts;
  l.max_items = tiles * hkv + (split ? kPagedFewParts + kPagedManyParts : 0) +
                (n_tokens + kPagedPadRows - 1) / kPagedPadRows;
  const int64_t merges = kPagedFewParts * (kPagedFewRows / 8) + many * (kPagedTileRows / 8);
  l.max_merges = !split ? 0 : rows < merges ? rows : merges;
  const int64_t by_row = rows * (max_keys / kPagedFewKeys + 1);
  const int64_t by_part = 2 * (kPagedFewParts * kPagedFewRows + many * kPagedTileRows);
  l.max_part_rows = !split ? 0 : by_row < by_part ? by_row : by_part;
  l.seq = up4(n_seqs + 1);
  l.pos = l.seq + up4(n_tokens);
  l.counts = l.pos + up4(n_tokens);
  l.items = l.counts + 4;
  l.merges = l.items + l.max_items * kPagedItemWords;
  l.words = l.merges + l.max_merges * kPagedMergeWords;
  return l;
}
// Partial results of split key ranges: O (rows, 128) fp32, then {maximum, sum} of every row.
inline int64_t paged_workspace(const PagedLayout& l) {
  return l.max_part_rows * (kHeadDim + 2) * 4;
}

struct PagedPlanArgs {
  const int32_t* q_lengths;
  const int32_t* kv_lengths;
  int n_seqs;
  int n_tokens;
  int hq, hkv;
  int max_keys;  // rows that a table row can name
  int32_t* plan;
  PagedLayout layout;
  hipStream_t stream;
  const int32_t* parents;  // null: no tree
  int32_t* tree;
};

// Pages of one layer. 8-bit pages have a byte per row beside them, the exponent of its power of two.
struct PagedPool {
  const int32_t* table;
  int table_width;
  int n_pages;
  int page_shift;               // log2 of page_size
  uint32_t k_stride, v_stride;  // bytes from page to page
  uint8_t* k_exp;               // null: 16-bit pages
  uint8_t* v_exp;
  uint32_t k_exp_stride, v_exp_stride;
};

// Rows of 8-bit pages are e4m3 numbers (up to 448 = 1.75 * 2^8) times 2^(byte - 127), the smallest such
// power that brings a row's largest finite number to 448 or less, from 2^-100 on (what is smaller than
// 448 * 2^-100 loses digits; 16-bit floats end far above).
constexpr int kExpBias = 127, kExpMin = 27;

// A step's tree: eight words per row, bit i of which says that token i of the row's sequence (of its new
// ones) lies on the row's path, itself included; then the position of every row, -1 for padding. The new
// tokens of a sequence of more than kTreeTokens are a chain and their words are not read.
constexpr int kTreeTokens = 256, kTreeWords = kTreeTokens / 32;
constexpr int64_t tree_positions(int64_t n_tokens) { return n_tokens * kTreeWords; }
inline int64_t tree_words(int64_t n_tokens) { return tree_positions(n_tokens) + up4(n_tokens); }

struct PagedAttnArgs {
  const void* q;
  const void* k;
  const void* v;
  PagedPool pool;
  const int32_t* plan;
  PagedLayout layout;
  int n_seqs;
  int n_tokens;
  int hq, hkv;
  float scale;
  int dtype;
  void* out;
  float* workspace;
  hipStream_t stream;
  const int32_t* tree;  // null: the new tokens of every sequence are a chain
};

struct PagedAppendArgs {
  const void* q;
  const void* k;
  const void* v;
  const float* cos;
  const float* sin;
  int64_t cos_batch_stride, cos_seq_stride, cos_token_stride;
  int64_t cos_rows;  // 0: positions are not bounded by the tables
  const int32_t* seq;  // plan: sequence and place of every row
  const int32_t* pos;
  const int32_t* rot;  // the position that it is rotated by
  PagedPool pool;
  void* q_out;
  void* k_pages;
  void* v_pages;
  int n_seqs, n_tokens;
  int heads, kv_heads;
  int in_dtype, out_dtype;
  hipStream_t stream;
};

// Page bookkeeping: outer x n_pages x (kv_heads, page_size) rows of row_chunks times 16 bytes (kHeadDim
// 16-bit elements, or 8-bit ones with an exponent byte per row in `exps`).
struct PagesArgs {
  void* pages;
  uint8_t* exps;  // null: 16-bit pages
  int row_chunks;
  int64_t outer;
  int n_pages, kv_heads;
  int page_shift;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* refs;
  const int32_t* parents;      // remap only; null: every row is its own parent
  const int32_t* new_lengths;  // remap only; null: as long as the parent
  int n_slots, width;
  int32_t* table_out;
  int32_t* lengths_out;  // remap only
  int32_t* refs_out;
  int32_t* result;  // remap: shortfall; compact: live pages
  int32_t* scratch;
  hipStream_t stream;
};
inline int64_t pages_scratch_words(int64_t n_slots, int64_t n_pages) {
  return 3 * n_pages + 5 * n_slots + 16;
}

struct PagesGrowthArgs {
  const int32_t* lengths;
  const int32_t* q_lengths;
  int n_slots;
  int64_t n_tokens;
  int32_t* new_lengths;
  int32_t* excess;
  hipStream_t stream;
};

// Rows of an accepted path: moved together behind the sequence's cached rows.
struct PagedAcceptArgs {
  const int32_t* plan;
  PagedLayout layout;
  const int32_t* tree;  // null: chains, nothing moves
  const int32_t* table;
  int n_seqs, n_tokens, width, page_shift;
  void* pages;
  uint8_t* exps;
  int row_chunks;
  int64_t outer;
  int n_pages, kv_heads;
  const int32_t* lengths;
  const int32_t* accepted;
  int32_t* lengths_out;
  hipStream_t stream;
};

hipError_t launch_paged_plan(const PagedPlanArgs& a);
hipError_t launch_paged_accept(const PagedAcceptArgs& a);
hipError_t launch_paged_attention(const PagedAttnArgs& a);
hipError_t launch_paged_append(const PagedAppendArgs& a);
hipError_t launch_pages_growth(const PagesGrowthArgs& a);
hipError_t launch_pages_remap(const PagesArgs& a);
hipError_t launch_pages_compact(const PagesArgs& a);

}  // namespace va
