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
// more are tiles of kPagedTileRows, a strip of 32 per wave.
constexpr int kPagedFewRows = 32;
constexpr int kPagedTileRows = 128;
constexpr int kPagedChunkKeys = 64;  // key ranges are split at multiples of this
// The attention's work-groups: 8 waves, one work-group per CU, for steps with prompts (more rows than
// sequences) of up to this many tiles x heads, by the sizes that the host knows; 4 waves, two per CU,
// for the others. us with 4 / 8 waves: 2 x 2048 tokens, 12/2 heads (388 tiles) 51 / 42; 4096 tokens
// (386) 88 / 72; 8 x 300 on 700 (240) 27.5 / 26; two chunks of 512 beside 62 answers, 28/4 heads (492) 60 /
// 59; 2 x 1024 on 500 (456) 46.5 / 47.5; 3 x 1024 (684) 62 / 67; 4 x 1024 (912) 78 / 82; four chunks of
// 2048 623 / 680; 64 answers of 64 to 8192 tokens 30.4 / 32.0, 16 of 1500 12.1 / 12.8, four of 512 7.9 / 7.5.
constexpr int kPagedWideTiles = 512;
// Parts that a step's keys are split into, by kind of tile, the shortest part (but a range's last) and
// the longest table row that is never split. us at 384 / 512 / 1024 few-row parts: 64 answers of 64 to
// 8192 tokens, 12/2 heads 34 / 30 / 32, four of 65,536, 28/4 heads 103 / 97 / 100; shortest few-row part
// 128 / 256 / 512: one answer of 8192 9.0 / 9.8 / 11.5, 16 of 1500 13.4 / 12.1 / 12.6. At 256 / 512
// prompt parts: two chunks of 512 beside 62 answers 57 / 76, 128 new tokens on 32,768 80 / 94; shortest
// prompt part 256 / 512 / 704: 300 new tokens on 1000 16.8 / 17.7 / 20.4, two of 64 on 8000 26.9 / 27.0 /
// 27.8, where 256 would make twice the parts and room for the merge. Four answers of 512, table rows of
// 576: split 8.5, whole 7.9 and a launch less.
constexpr int kPagedFewParts = 512, kPagedManyParts = 256;
constexpr int kPagedFewKeys = 256, kPagedManyKeys = 512;
constexpr int kPagedWholeKeys = 1024;
constexpr int kPagedPadRows = 64;     // padding rows that one item zeroes

// A step's plan, int32 words: cu (n_seqs + 1) row offsets of the sequences, the sequence (-1: padding)
// and the position of every row, the counts of items and merge records, the items, the records.
constexpr int kPagedItemWords = 12, kPagedMergeWords = 8;
struct PagedLayout {
  int64_t seq, pos, counts, items, merges, words;  // offsets; cu lies at 0
  int64_t max_items, max_merges, max_part_rows;
  bool wide;
};
inline int64_t up4(int64_t x) { return (x + 3) & ~int64_t(3); }
// Bounds: a sequence with rows makes one tile, and one more per full kPagedTileRows. A kind's parts have
// at least its total (tiles times the longest of the sequence) / its number of parts keys, so the
// tiles of a sequence of n > 1 parts stand for more than n - 1 >= n / 2 of them each, and all split
// tiles have at most twice as many parts; each part holds at most the kind's rows, and a row is in at
// most max_keys / kPagedFewKeys + 1 parts. A merge record takes 8 rows of a sequence of up to 8 parts,
// or one row of one of more.
inline PagedLayout paged_layout(int64_t n_seqs, int64_t n_tokens, int64_t hq, int64_t hkv,
                                int64_t max_keys) {
  PagedLayout l;
  const int64_t tiles = (n_seqs < n_tokens ? n_seqs : n_tokens) + n_tokens * (hq / hkv) / kPagedTileRows;
  const bool split = max_keys > kPagedWholeKeys;
  const int64_t rows = n_tokens * hq;
  l.wide = n_tokens > n_seqs && tiles * hkv <= kPagedWideTiles;
  l.max_items = tiles * hkv + (split ? kPagedFewParts + kPagedManyParts : 0) +
                (n_tokens + kPagedPadRows - 1) / kPagedPadRows;
  const int64_t merges = kPagedFewParts * (kPagedFewRows / 8) + kPagedManyParts * (kPagedTileRows / 8);
  l.max_merges = !split ? 0 : rows < merges ? rows : merges;
  const int64_t by_row = rows * (max_keys / kPagedFewKeys + 1);
  const int64_t by_part = 2 * (kPagedFewParts * kPagedFewRows + kPagedManyParts * kPagedTileRows);
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
};

// Pages of one layer.
struct PagedPool {
  const int32_t* table;
  int table_width;
  int n_pages;
  int page_shift;               // log2 of page_size
  uint32_t k_stride, v_stride;  // bytes from page to page
};

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
};

struct PagedAppendArgs {
  const void* q;
  const void* k;
  const void* v;
  const float* cos;
  const float* sin;
  int64_t cos_batch_stride, cos_seq_stride, cos_token_stride;
  int64_t cos_rows;  // 0: positions are not bounded by the tables
  const int32_t* seq;  // plan: sequence and position of every row
  const int32_t* pos;
  PagedPool pool;
  void* q_out;
  void* k_pages;
  void* v_pages;
  int n_seqs, n_tokens;
  int heads, kv_heads;
  int in_dtype, out_dtype;
  hipStream_t stream;
};

// Page bookkeeping: outer x n_pages x (kv_heads, page_size) rows of kHeadDim 16-bit elements.
struct PagesArgs {
  void* pages;
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

hipError_t launch_paged_plan(const PagedPlanArgs& a);
hipError_t launch_paged_attention(const PagedAttnArgs& a);
hipError_t launch_paged_append(const PagedAppendArgs& a);
hipError_t launch_pages_growth(const PagesGrowthArgs& a);
hipError_t launch_pages_remap(const PagesArgs& a);
hipError_t launch_pages_compact(const PagesArgs& a);

}  // namespace va
