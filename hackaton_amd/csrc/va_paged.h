// Launch descriptors of the paged key/value cache: the step plan, the append, the attention over
// pages and the page bookkeeping, shared by their kernels and the C-ABI layer.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace va {

constexpr int kPagedMaxSeqs = 8192;  // sequences of a step
constexpr int kPageMin = 16, kPageMax = 256;

// A step's plan, int32 words: cu (n_seqs + 1) row offsets of the sequences, then the sequence (-1:
// padding) and the position of every row.
struct PagedLayout {
  int64_t seq, pos, words;  // cu lies at 0
};
inline PagedLayout paged_layout(int64_t n_seqs, int64_t n_tokens) {
  PagedLayout l;
  const int64_t rows = (n_tokens + 3) & ~int64_t(3);
  l.seq = (n_seqs + 1 + 3) & ~int64_t(3);
  l.pos = l.seq + rows;
  l.words = l.pos + rows;
  return l;
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
  int64_t k_stride, v_stride;  // elements from page to page
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
  void* workspace;
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
  int n_tokens;
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
  return 3 * n_pages + 2 * n_slots + 16;
}

hipError_t launch_paged_plan(const PagedPlanArgs& a);
hipError_t launch_paged_attention(const PagedAttnArgs& a);
hipError_t launch_paged_append(const PagedAppendArgs& a);
hipError_t launch_pages_remap(const PagesArgs& a);
hipError_t launch_pages_compact(const PagesArgs& a);

}  // namespace va
