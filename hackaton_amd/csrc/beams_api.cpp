// C-ABI entry points of beam search's selection: argument validation, then the kernel launcher.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/varlen_attn.h"
#include "va_api_internal.h"
#include "va_beams.h"

namespace {

int check_sizes(int64_t groups, int32_t beams, int32_t vocab, const char* what) {
  if (beams < 1 || beams > va::kBeamsMost)
    return va::fail(VA_ESHAPE, "%s: beams=%d (1 to %d)", what, beams, va::kBeamsMost);
  if (vocab < 1 || vocab > va::kBeamsVocab)
    return va::fail(VA_ESHAPE, "%s: vocab=%d (1 to %d)", what, vocab, va::kBeamsVocab);
  if (groups < 0 || groups > va::kBeamsRows / beams)
    return va::fail(VA_ESHAPE, "%s: groups=%lld of %d beams (at most %d rows)", what, (long long)groups, beams,
                    va::kBeamsRows);
  return VA_OK;
}

}  // namespace

extern "C" int va_select_beams_workspace(int64_t groups, int32_t beams, int32_t vocab, int64_t* bytes) {
  const char* what = "va_select_beams_workspace";
  const int rc = check_sizes(groups, beams, vocab, what);
  if (rc) return rc;
  if (bytes == nullptr) return va::fail(VA_EINVAL, "%s: NULL output", what);
  *bytes = 4 * va::beams_layout(groups * beams, beams, vocab).words;
  return VA_OK;
}

extern "C" int va_select_beams(const void* logits, int32_t dtype, int64_t row_stride, int64_t groups,
                               int32_t beams, int32_t vocab, const float* scores,
                               const uint8_t* ended, int32_t end_token, int32_t count,
                               float* scores_out, int32_t* parents_out, int32_t* tokens_out,
                               void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "va_select_beams";
  int rc = check_sizes(groups, beams, vocab, what);
  if (rc) return rc;
  if (dtype < VA_F16 || dtype > VA_F32) return va::fail(VA_EDTYPE, "%s: dtype %d", what, dtype);
  if (count < 1 || count > va::kBeamsCount || count > (int64_t)beams * vocab)
    return va::fail(VA_ESHAPE, "%s: count=%d (1 to %d, and no more than beams x vocab)", what, count,
                    va::kBeamsCount);
  if (ended != nullptr && (end_token < 0 || end_token >= vocab))
    return va::fail(VA_EINVAL, "%s: end_token=%d of %d", what, end_token, vocab);
  if (row_stride < vocab && groups * beams > 1)
    return va::fail(VA_EINVAL, "%s: row_stride=%lld, rows of %d", what, (long long)row_stride, vocab);
  if (groups == 0) return VA_OK;
  const va::BeamsLayout layout = va::beams_layout(groups * beams, beams, vocab);
  if (workspace_bytes < 4 * layout.words)
    return va::fail(VA_ECAPACITY, "%s: workspace %lld bytes, need %lld", what,
                    (long long)workspace_bytes, (long long)(4 * layout.words));
  for (const void* p : {logits, (const void*)scores, (const void*)scores_out,
                        (const void*)parents_out, (const void*)tokens_out, (const void*)workspace})
    if (p == nullptr) return va::fail(VA_EINVAL, "%s: NULL buffer", what);
  if (((uintptr_t)logits & (dtype == VA_F32 ? 3u : 1u)) != 0 || ((uintptr_t)scores & 3u) != 0 ||
      ((uintptr_t)scores_out & 3u) != 0 || ((uintptr_t)parents_out & 3u) != 0 ||
      ((uintptr_t)tokens_out & 3u) != 0 || ((uintptr_t)workspace & 15u) != 0)
    return va::fail(VA_EINVAL, "%s: buffer not aligned to its elements (workspace: 16 bytes)", what);
  va::BeamsArgs a{logits, dtype, row_stride, (int)groups, beams, vocab, scores, ended, end_token, count,
                  layout, (float*)workspace, scores_out, parents_out, tokens_out, (hipStream_t)stream};
  const hipError_t e = va::launch_select_beams(a);
  return e == hipSuccess ? VA_OK : va::fail((int)e, "%s launch: %s", what, hipGetErrorString(e));
}
