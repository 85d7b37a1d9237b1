// C-ABI entry points of the paged key/value cache: argument validation, then the kernel launchers.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "../../include/varlen_attn.h"
#include "va_api_internal.h"
#include "va_kernels.h"
#include "va_paged.h"

namespace {

int launched(hipError_t e, const char* what) {
  return e == hipSuccess ? VA_OK : va::fail((int)e, "%s launch: %s", what, hipGetErrorString(e));
}

int check_buffers(std::initializer_list<const void*> ptrs, const char* what) {
  for (const void* p : ptrs) {
    if (p == nullptr) return va::fail(VA_EINVAL, "%s: NULL buffer", what);
    if (((uintptr_t)p & 15u) != 0)
      return va::fail(VA_EINVAL, "%s: buffer not 16-byte aligned", what);
  }
  return VA_OK;
}

int check_words(std::initializer_list<const void*> ptrs, const char* what) {  // int32 arrays
  for (const void* p : ptrs) {
    if (p == nullptr) return va::fail(VA_EINVAL, "%s: NULL buffer", what);
    if (((uintptr_t)p & 3u) != 0) return va::fail(VA_EINVAL, "%s: buffer not 4-byte aligned", what);
  }
  return VA_OK;
}

int check_page_size(int32_t page_size, const char* what) {
  if (page_size < va::kPageMin || page_size > va::kPageMax || (page_size & (page_size - 1)) != 0)
    return va::fail(VA_ESHAPE, "%s: page_size=%d must be a power of two from %d to %d", what,
                    page_size, va::kPageMin, va::kPageMax);
  return VA_OK;
}

int shift_of(int32_t page_size) { return __builtin_ctz((unsigned)page_size); }

int check_step(const va_paged_step* s, const char* what) {
  if (s == nullptr) return va::fail(VA_EINVAL, "%s: step is NULL", what);
  if (s->n_seqs < 0 || s->n_seqs > va::kPagedMaxSeqs)
    return va::fail(VA_ESHAPE, "%s: n_seqs=%d (at most %d)", what, s->n_seqs, va::kPagedMaxSeqs);
  if (s->hq <= 0 || s->hkv <= 0 || s->hq % s->hkv != 0 || s->hq > 4096)
    return va::fail(VA_ESHAPE, "%s: Hq=%d must be a positive multiple of Hkv=%d, at most 4096", what,
                    s->hq, s->hkv);
  if (s->n_tokens < 0 || s->n_tokens > INT32_MAX / 2 || s->n_tokens * s->hq > INT32_MAX / 2)
    return va::fail(VA_ESHAPE, "%s: n_tokens=%lld out of range", what, (long long)s->n_tokens);
  const int rc = check_page_size(s->page_size, what);
  if (rc) return rc;
  if (s->table_width < 0 || (int64_t)s->table_width * s->page_size > INT32_MAX / 2)
    return va::fail(VA_ESHAPE, "%s: table_width=%d x page_size=%d out of range", what,
                    s->table_width, s->page_size);
  return VA_OK;
}

va::PagedLayout layout_of(const va_paged_step& s) {
  return va::paged_layout(s.n_seqs, s.n_tokens, s.hq, s.hkv, (int64_t)s.table_width * s.page_size);
}

// Pages of one layer, keys and values, and the step's table and plan.
int check_pool(const va_paged_step& s, const va_paged_pages& p, const char* what) {
  const bool bytes = p.dtype == VA_E4M3;
  if (p.n_pages < 0) return va::fail(VA_ESHAPE, "%s: n_pages=%d", what, p.n_pages);
  for (int64_t stride : {p.k_stride, p.v_stride})
    if (stride % (bytes ? 16 : 8) != 0 || stride < (int64_t)s.hkv * s.page_size * va::kHeadDim)
      return va::fail(VA_EINVAL, "%s: page strides must be multiples of %d and cover a page", what,
                      bytes ? 16 : 8);
    else if (stride > (int64_t)(UINT32_MAX / 2))
      return va::fail(VA_ESHAPE, "%s: page strides of 4 GiB or more", what);
  int rc = VA_OK;
  if (p.n_pages > 0 && (rc = check_buffers({p.k_pages, p.v_pages}, what))) return rc;
  if (bytes) {
    for (int64_t stride : {p.k_exp_stride, p.v_exp_stride})
      if (stride < (int64_t)s.hkv * s.page_size || stride > INT32_MAX)
        return va::fail(VA_EINVAL, "%s: exponent strides must cover a page", what);
    if (p.n_pages > 0 && (p.k_exps == nullptr || p.v_exps == nullptr))
      return va::fail(VA_EINVAL, "%s: NULL exponents", what);
  }
  if (s.n_tokens > 0 && (rc = check_buffers({s.plan}, what))) return rc;
  if (s.n_seqs > 0 && s.table_width > 0) rc = check_words({s.page_table}, what);
  return rc;
}

va::PagedPool pool_of(const va_paged_step& s, const va_paged_pages& p) {
  const bool bytes = p.dtype == VA_E4M3;
  const int64_t size = bytes ? 1 : 2;
  return va::PagedPool{s.page_table, s.table_width, p.n_pages, shift_of(s.page_size),
                       (uint32_t)(size * p.k_stride), (uint32_t)(size * p.v_stride),
                       bytes ? p.k_exps : nullptr, bytes ? p.v_exps : nullptr,
                       bytes ? (uint32_t)p.k_exp_stride : 0, bytes ? (uint32_t)p.v_exp_stride : 0};
}

int append_checked(const va_paged_step* step, const int32_t* tree, const void* q, const void* k,
                   const void* v, const float* cos, const float* sin, int64_t cos_batch_stride,
                   int64_t cos_seq_stride, int64_t cos_token_stride, int64_t cos_rows, void* q_out,
                   const va_paged_pages& pages, int32_t head_dim, int32_t in_dtype,
                   int32_t out_dtype, void* stream, const char* what) {
  if (head_dim != va::kHeadDim)
    return va::fail(VA_ESHAPE, "%s: head_dim=%d, built for %d", what, head_dim, va::kHeadDim);
  int rc = check_step(step, what);
  if (rc) return rc;
  const va_paged_step& s = *step;
  if (in_dtype < VA_F16 || in_dtype > VA_F32 || (out_dtype != VA_F16 && out_dtype != VA_BF16) ||
      (pages.dtype != out_dtype && pages.dtype != VA_E4M3))
    return va::fail(VA_EDTYPE, "%s: dtype", what);
  for (int64_t stride : {cos_batch_stride, cos_seq_stride, cos_token_stride})
    if (stride < 0 || stride % 4 != 0)
      return va::fail(VA_EINVAL, "%s: cos/sin strides must be non-negative multiples of 4", what);
  if (cos_rows < 0) return va::fail(VA_EINVAL, "%s: cos_rows", what);
  if ((rc = check_pool(s, pages, what))) return rc;
  if (s.n_tokens == 0) return VA_OK;
  if ((rc = check_buffers({q, k, v, cos, sin, q_out}, what))) return rc;
  if (tree != nullptr && (rc = check_buffers({tree}, what))) return rc;
  const va::PagedLayout layout = layout_of(s);
  const int32_t* pos = s.plan + layout.pos;
  va::PagedAppendArgs a{q, k, v, cos, sin, cos_batch_stride, cos_seq_stride, cos_token_stride,
                        cos_rows, s.plan + layout.seq, pos,
                        tree == nullptr ? pos : tree + va::tree_positions(s.n_tokens),
                        pool_of(s, pages), q_out, pages.k_pages, pages.v_pages, s.n_seqs,
                        (int)s.n_tokens, s.hq, s.hkv, in_dtype, out_dtype, (hipStream_t)stream};
  return launched(va::launch_paged_append(a), what);
}

int attention_checked(const va_paged_step* step, const int32_t* tree, const void* q,
                      const va_paged_pages& pages, int32_t head_dim, float scale, int32_t dtype,
                      void* out, void* workspace, int64_t workspace_bytes, void* stream,
                      const char* what) {
  if (head_dim != va::kHeadDim)
    return va::fail(VA_ESHAPE, "%s: head_dim=%d, built for %d", what, head_dim, va::kHeadDim);
  int rc = check_step(step, what);
  if (rc) return rc;
  const va_paged_step& s = *step;
  if ((dtype != VA_F16 && dtype != VA_BF16) || (pages.dtype != dtype && pages.dtype != VA_E4M3))
    return va::fail(VA_EDTYPE, "%s: dtype %d: attention runs on VA_F16 or VA_BF16", what, dtype);
  if (!std::isfinite(scale) || scale <= 0.f)
    return va::fail(VA_EINVAL, "%s: scale must be finite and positive", what);
  if ((rc = check_pool(s, pages, what))) return rc;
  if (s.n_tokens == 0) return VA_OK;
  const va::PagedLayout layout = layout_of(s);
  const int64_t need = va::paged_workspace(layout);
  if (workspace_bytes < need)
    return va::fail(VA_ECAPACITY, "%s: workspace %lld bytes, need %lld", what,
                    (long long)workspace_bytes, (long long)need);
  if ((rc = check_buffers({q, out}, what))) return rc;
  if (need > 0 && (rc = check_buffers({workspace}, what))) return rc;
  if (tree != nullptr && (rc = check_buffers({tree}, what))) return rc;
  va::PagedAttnArgs a{q, pages.k_pages, pages.v_pages, pool_of(s, pages), s.plan, layout,
                      s.n_seqs, (int)s.n_tokens, s.hq, s.hkv, scale, dtype, out, (float*)workspace,
                      (hipStream_t)stream, tree};
  return launched(va::launch_paged_attention(a), what);
}

// (the 16-bit entry points' pages)
va_paged_pages pages16(const void* k, const void* v, int64_t k_stride, int64_t v_stride,
                       int32_t n_pages, int32_t dtype) {
  return va_paged_pages{const_cast<void*>(k), const_cast<void*>(v), nullptr, nullptr, k_stride,
                        v_stride, 0, 0, n_pages, dtype};
}

}  // namespace

extern "C" int va_paged_plan_words(const va_paged_step* step, int64_t* words) {
  const int rc = check_step(step, "va_paged_plan_words");
  if (rc) return rc;
  if (words == nullptr) return va::fail(VA_EINVAL, "va_paged_plan_words: NULL output");
  *words = layout_of(*step).words;
  return VA_OK;
}

namespace {

int plan_checked(const va_paged_step* step, const int32_t* q_lengths, const int32_t* kv_lengths,
                 int64_t plan_words, const int32_t* parents, int32_t* tree, int64_t tree_words,
                 bool with_tree, void* stream, const char* what) {
  int rc = check_step(step, what);
  if (rc) return rc;
  const va_paged_step& s = *step;
  if (s.n_tokens == 0) return VA_OK;
  const va::PagedLayout layout = layout_of(s);
  if (plan_words < layout.words)
    return va::fail(VA_ECAPACITY, "%s: %lld words, need %lld", what, (long long)plan_words,
                    (long long)layout.words);
  if (with_tree && tree_words < va::tree_words(s.n_tokens))
    return va::fail(VA_ECAPACITY, "%s: %lld words of a tree, need %lld", what, (long long)tree_words,
                    (long long)va::tree_words(s.n_tokens));
  if ((rc = check_buffers({s.plan}, what))) return rc;
  if (s.n_seqs > 0 && (rc = check_words({q_lengths, kv_lengths}, what))) return rc;
  if (with_tree && ((rc = check_buffers({tree}, what)) || (rc = check_words({parents}, what)))) return rc;
  va::PagedPlanArgs a{q_lengths, kv_lengths, s.n_seqs, (int)s.n_tokens, s.hq, s.hkv,
                      s.table_width * s.page_size, s.plan, layout, (hipStream_t)stream,
                      with_tree ? parents : nullptr, with_tree ? tree : nullptr};
  return launched(va::launch_paged_plan(a), what);
}

}  // namespace

extern "C" int va_paged_plan(const va_paged_step* step, const int32_t* q_lengths,
                             const int32_t* kv_lengths, int64_t plan_words, void* stream) {
  return plan_checked(step, q_lengths, kv_lengths, plan_words, nullptr, nullptr, 0, false, stream,
                      "va_paged_plan");
}

extern "C" int va_paged_plan_tree(const va_paged_step* step, const int32_t* q_lengths,
                                  const int32_t* kv_lengths, int64_t plan_words,
                                  const int32_t* parents, int32_t* tree, int64_t tree_words,
                                  void* stream) {
  return plan_checked(step, q_lengths, kv_lengths, plan_words, parents, tree, tree_words, true, stream,
                      "va_paged_plan_tree");
}

extern "C" int va_paged_append(const va_paged_step* step, const void* q, const void* k,
                               const void* v, const float* cos, const float* sin,
                               int64_t cos_batch_stride, int64_t cos_seq_stride,
                               int64_t cos_token_stride, int64_t cos_rows, void* q_out,
                               void* k_pages, void* v_pages, int64_t k_stride, int64_t v_stride,
                               int32_t n_pages, int32_t head_dim, int32_t in_dtype,
                               int32_t out_dtype, void* stream) {
  return append_checked(step, nullptr, q, k, v, cos, sin, cos_batch_stride, cos_seq_stride,
                        cos_token_stride, cos_rows, q_out,
                        pages16(k_pages, v_pages, k_stride, v_stride, n_pages, out_dtype), head_dim,
                        in_dtype, out_dtype, stream, "va_paged_append");
}

extern "C" int va_paged_append_pages(const va_paged_step* step, const int32_t* tree, const void* q,
                                     const void* k, const void* v, const float* cos,
                                     const float* sin, int64_t cos_batch_stride,
                                     int64_t cos_seq_stride, int64_t cos_token_stride,
                                     int64_t cos_rows, void* q_out, const va_paged_pages* pages,
                                     int32_t head_dim, int32_t in_dtype, int32_t out_dtype,
                                     void* stream) {
  const char* what = "va_paged_append_pages";
  if (pages == nullptr) return va::fail(VA_EINVAL, "%s: pages is NULL", what);
  return append_checked(step, tree, q, k, v, cos, sin, cos_batch_stride, cos_seq_stride,
                        cos_token_stride, cos_rows, q_out, *pages, head_dim, in_dtype, out_dtype,
                        stream, what);
}

extern "C" int va_paged_attention_workspace(const va_paged_step* step, int64_t* bytes) {
  const int rc = check_step(step, "va_paged_attention_workspace");
  if (rc) return rc;
  if (bytes == nullptr) return va::fail(VA_EINVAL, "va_paged_attention_workspace: NULL output");
  *bytes = va::paged_workspace(layout_of(*step));
  return VA_OK;
}

extern "C" int va_paged_attention(const va_paged_step* step, const void* q, const void* k_pages,
                                  const void* v_pages, int64_t k_stride, int64_t v_stride,
                                  int32_t n_pages, int32_t head_dim, float scale, int32_t dtype,
                                  void* out, void* workspace, int64_t workspace_bytes,
                                  void* stream) {
  return attention_checked(step, nullptr, q,
                           pages16(k_pages, v_pages, k_stride, v_stride, n_pages, dtype), head_dim,
                           scale, dtype, out, workspace, workspace_bytes, stream,
                           "va_paged_attention");
}

extern "C" int va_paged_attention_pages(const va_paged_step* step, const int32_t* tree,
                                        const void* q, const va_paged_pages* pages,
                                        int32_t head_dim, float scale, int32_t dtype, void* out,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "va_paged_attention_pages";
  if (pages == nullptr) return va::fail(VA_EINVAL, "%s: pages is NULL", what);
  return attention_checked(step, tree, q, *pages, head_dim, scale, dtype, out, workspace,
                           workspace_bytes, stream, what);
}

extern "C" int va_paged_tree_words(const va_paged_step* step, int64_t* words) {
  const int rc = check_step(step, "va_paged_tree_words");
  if (rc) return rc;
  if (words == nullptr) return va::fail(VA_EINVAL, "va_paged_tree_words: NULL output");
  *words = va::tree_words(step->n_tokens);
  return VA_OK;
}

namespace {

int check_pages(const void* pages, int64_t outer, int32_t n_pages, int32_t kv_heads,
                int32_t page_size, int32_t head_dim, int32_t n_slots, int32_t table_width,
                int64_t scratch_words, const char* what) {
  if (head_dim != va::kHeadDim)
    return va::fail(VA_ESHAPE, "%s: head_dim=%d, built for %d", what, head_dim, va::kHeadDim);
  int rc = check_page_size(page_size, what);
  if (rc) return rc;
  if (outer < 0 || outer > (1 << 20) || n_pages < 0 || n_pages > (1 << 28) || kv_heads <= 0 ||
      kv_heads > 4096 || n_slots < 0 || n_slots > (1 << 20) || table_width < 0 ||
      (int64_t)table_width * page_size > INT32_MAX / 2)
    return va::fail(VA_ESHAPE, "%s: outer=%lld n_pages=%d kv_heads=%d n_slots=%d table_width=%d",
                    what, (long long)outer, n_pages, kv_heads, n_slots, table_width);
  if (scratch_words < va::pages_scratch_words(n_slots, n_pages))
    return va::fail(VA_ECAPACITY, "%s: scratch of %lld words, need %lld", what,
                    (long long)scratch_words, (long long)va::pages_scratch_words(n_slots, n_pages));
  return n_pages > 0 && outer > 0 ? check_buffers({pages}, what) : VA_OK;
}

}  // namespace

extern "C" int va_pages_scratch_words(int32_t n_slots, int32_t n_pages, int64_t* words) {
  if (n_slots < 0 || n_pages < 0) return va::fail(VA_ESHAPE, "va_pages_scratch_words: sizes");
  if (words == nullptr) return va::fail(VA_EINVAL, "va_pages_scratch_words: NULL output");
  *words = va::pages_scratch_words(n_slots, n_pages);
  return VA_OK;
}

extern "C" int va_pages_growth(const int32_t* lengths, const int32_t* q_lengths, int32_t n_slots,
                               int64_t n_tokens, int32_t* new_lengths, int32_t* excess,
                               void* stream) {
  const char* what = "va_pages_growth";
  if (n_slots < 0 || n_slots > (1 << 20) || n_tokens < 0)
    return va::fail(VA_ESHAPE, "%s: n_slots=%d n_tokens=%lld", what, n_slots, (long long)n_tokens);
  if (n_slots == 0) return VA_OK;
  const int rc = check_words({lengths, q_lengths, new_lengths, excess}, what);
  if (rc) return rc;
  va::PagesGrowthArgs a{lengths, q_lengths, n_slots, n_tokens, new_lengths, excess,
                        (hipStream_t)stream};
  return launched(va::launch_pages_growth(a), what);
}

namespace {

int remap_checked(void* pages, uint8_t* exps, bool bytes, int64_t outer, int32_t n_pages,
                  int32_t kv_heads, int32_t page_size, int32_t head_dim, const int32_t* table,
                  const int32_t* lengths, const int32_t* refs, const int32_t* parents,
                  const int32_t* new_lengths, int32_t n_slots, int32_t table_width,
                  int32_t* table_out, int32_t* lengths_out, int32_t* refs_out, int32_t* shortfall,
                  int32_t* scratch, int64_t scratch_words, void* stream, const char* what) {
  int rc = check_pages(pages, outer, n_pages, kv_heads, page_size, head_dim, n_slots, table_width,
                       scratch_words, what);
  if (rc) return rc;
  if (bytes && n_pages > 0 && outer > 0 && (rc = check_buffers({exps}, what))) return rc;
  if ((rc = check_words({shortfall, scratch}, what))) return rc;
  if (n_slots > 0 && (rc = check_words({lengths, lengths_out}, what))) return rc;
  for (const int32_t* p : {parents, new_lengths})
    if (n_slots > 0 && p != nullptr && (rc = check_words({p}, what))) return rc;
  if (n_slots > 0 && table_width > 0 && (rc = check_words({table, table_out}, what))) return rc;
  if (n_pages > 0 && (rc = check_words({refs, refs_out}, what))) return rc;
  if ((table != nullptr && table == table_out) || (lengths != nullptr && lengths == lengths_out) ||
      (refs != nullptr && refs == refs_out))
    return va::fail(VA_EINVAL, "%s: outputs may not be the inputs", what);
  va::PagesArgs a{pages, bytes ? exps : nullptr, va::kHeadDim / (bytes ? 16 : 8), outer, n_pages,
                  kv_heads, shift_of(page_size), table, lengths, refs, parents, new_lengths,
                  n_slots, table_width, table_out, lengths_out, refs_out, shortfall, scratch,
                  (hipStream_t)stream};
  return launched(va::launch_pages_remap(a), what);
}

int compact_checked(void* pages, uint8_t* exps, bool bytes, int64_t outer, int32_t n_pages,
                    int32_t kv_heads, int32_t page_size, int32_t head_dim, const int32_t* table,
                    const int32_t* lengths, const int32_t* refs, int32_t n_slots,
                    int32_t table_width, int32_t* table_out, int32_t* refs_out, int32_t* live,
                    int32_t* scratch, int64_t scratch_words, void* stream, const char* what) {
  int rc = check_pages(pages, outer, n_pages, kv_heads, page_size, head_dim, n_slots, table_width,
                       scratch_words, what);
  if (rc) return rc;
  if (bytes && n_pages > 0 && outer > 0 && (rc = check_buffers({exps}, what))) return rc;
  if ((rc = check_words({live, scratch}, what))) return rc;
  if (n_slots > 0 && (rc = check_words({lengths}, what))) return rc;
  if (n_slots > 0 && table_width > 0 && (rc = check_words({table, table_out}, what))) return rc;
  if (n_pages > 0 && (rc = check_words({refs, refs_out}, what))) return rc;
  if ((table != nullptr && table == table_out) || (refs != nullptr && refs == refs_out))
    return va::fail(VA_EINVAL, "%s: outputs may not be the inputs", what);
  va::PagesArgs a{pages, bytes ? exps : nullptr, va::kHeadDim / (bytes ? 16 : 8), outer, n_pages,
                  kv_heads, shift_of(page_size), table, lengths, refs, nullptr, nullptr, n_slots,
                  table_width, table_out, nullptr, refs_out, live, scratch, (hipStream_t)stream};
  return launched(va::launch_pages_compact(a), what);
}

}  // namespace

extern "C" int va_pages_remap(void* pages, int64_t outer, int32_t n_pages, int32_t kv_heads,
                              int32_t page_size, int32_t head_dim, const int32_t* table,
                              const int32_t* lengths, const int32_t* refs, const int32_t* parents,
                              const int32_t* new_lengths, int32_t n_slots, int32_t table_width,
                              int32_t* table_out, int32_t* lengths_out, int32_t* refs_out,
                              int32_t* shortfall, int32_t* scratch, int64_t scratch_words,
                              void* stream) {
  return remap_checked(pages, nullptr, false, outer, n_pages, kv_heads, page_size, head_dim, table,
                       lengths, refs, parents, new_lengths, n_slots, table_width, table_out,
                       lengths_out, refs_out, shortfall, scratch, scratch_words, stream,
                       "va_pages_remap");
}

extern "C" int va_pages_remap8(void* pages, uint8_t* exps, int64_t outer, int32_t n_pages,
                               int32_t kv_heads, int32_t page_size, int32_t head_dim,
                               const int32_t* table, const int32_t* lengths, const int32_t* refs,
                               const int32_t* parents, const int32_t* new_lengths, int32_t n_slots,
                               int32_t table_width, int32_t* table_out, int32_t* lengths_out,
                               int32_t* refs_out, int32_t* shortfall, int32_t* scratch,
                               int64_t scratch_words, void* stream) {
  return remap_checked(pages, exps, true, outer, n_pages, kv_heads, page_size, head_dim, table,
                       lengths, refs, parents, new_lengths, n_slots, table_width, table_out,
                       lengths_out, refs_out, shortfall, scratch, scratch_words, stream,
                       "va_pages_remap8");
}

extern "C" int va_pages_compact(void* pages, int64_t outer, int32_t n_pages, int32_t kv_heads,
                                int32_t page_size, int32_t head_dim, const int32_t* table,
                                const int32_t* lengths, const int32_t* refs, int32_t n_slots,
                                int32_t table_width, int32_t* table_out, int32_t* refs_out,
                                int32_t* live, int32_t* scratch, int64_t scratch_words,
                                void* stream) {
  return compact_checked(pages, nullptr, false, outer, n_pages, kv_heads, page_size, head_dim,
                         table, lengths, refs, n_slots, table_width, table_out, refs_out, live,
                         scratch, scratch_words, stream, "va_pages_compact");
}

extern "C" int va_pages_compact8(void* pages, uint8_t* exps, int64_t outer, int32_t n_pages,
                                 int32_t kv_heads, int32_t page_size, int32_t head_dim,
                                 const int32_t* table, const int32_t* lengths, const int32_t* refs,
                                 int32_t n_slots, int32_t table_width, int32_t* table_out,
                                 int32_t* refs_out, int32_t* live, int32_t* scratch,
                                 int64_t scratch_words, void* stream) {
  return compact_checked(pages, exps, true, outer, n_pages, kv_heads, page_size, head_dim, table,
                         lengths, refs, n_slots, table_width, table_out, refs_out, live, scratch,
                         scratch_words, stream, "va_pages_compact8");
}

extern "C" int va_paged_accept(const va_paged_step* step, const int32_t* tree, void* pages,
                               uint8_t* exps, int64_t outer, int32_t n_pages, int32_t kv_heads,
                               int32_t head_dim, const int32_t* lengths, const int32_t* accepted,
                               int32_t* lengths_out, void* stream) {
  const char* what = "va_paged_accept";
  int rc = check_step(step, what);
  if (rc) return rc;
  const va_paged_step& s = *step;
  if ((rc = check_pages(pages, outer, n_pages, kv_heads, s.page_size, head_dim, s.n_seqs,
                        s.table_width, INT64_MAX, what)))
    return rc;
  if (exps != nullptr && (rc = check_buffers({exps}, what))) return rc;
  if (s.n_seqs == 0) return VA_OK;
  if ((rc = check_words({lengths, accepted, lengths_out}, what))) return rc;
  if (s.table_width > 0 && (rc = check_words({s.page_table}, what))) return rc;
  if (s.n_tokens > 0 && (rc = check_buffers({s.plan}, what))) return rc;
  if (tree != nullptr && (rc = check_buffers({tree}, what))) return rc;
  va::PagedAcceptArgs a{s.plan, layout_of(s), tree, s.page_table, s.n_seqs, (int)s.n_tokens,
                        s.table_width, shift_of(s.page_size), pages, exps,
                        va::kHeadDim / (exps == nullptr ? 8 : 16), outer, n_pages, kv_heads,
                        lengths, accepted, lengths_out, (hipStream_t)stream};
  return launched(va::launch_paged_accept(a), what);
}
