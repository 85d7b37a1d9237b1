// Attention of a step's new tokens over a paged key/value cache: the plan kernel that places every
// row, and the attention.
#include "../../include/varlen_attn.h"
#include "va_common.h"
#include "va_kernels.h"
#include "va_paged.h"
#include "va_scan.h"

namespace va {

namespace {

constexpr int PT = 1024;                    // threads of a planning work-group
constexpr int SPT = kPagedMaxSeqs / PT;     // sequences per thread
constexpr int kPlanRowsPerGroup = 4 * PT;   // rows that a planning work-group places

// Every work-group sums the lengths by itself (at most 64 KB of them) and places its own rows: one
// launch, nothing handed from one work-group to another.
__global__ __launch_bounds__(PT) void paged_plan_kernel(PagedPlanArgs a) {
  __shared__ int s_cu[kPagedMaxSeqs + 1];
  __shared__ long long s_scan[PT / 64];
  const int tid = threadIdx.x;
  int q[SPT];
  long long sum = 0;
#pragma unroll
  for (int i = 0; i < SPT; ++i) {
    const int s = tid * SPT + i;
    q[i] = s < a.n_seqs ? max(a.q_lengths[s], 0) : 0;
    sum += q[i];
  }
  long long total;
  long long at = block_exclusive_sum<PT / 64>(sum, s_scan, total);
#pragma unroll
  for (int i = 0; i < SPT; ++i) {
    const int s = tid * SPT + i;
    if (s <= a.n_seqs) s_cu[s] = (int)min(at, (long long)a.n_tokens);
    at += q[i];
  }
  if (tid == PT - 1 && a.n_seqs == kPagedMaxSeqs)
    s_cu[kPagedMaxSeqs] = (int)min(total, (long long)a.n_tokens);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int s = tid; s <= a.n_seqs; s += PT) a.plan[s] = s_cu[s];
  const int rows = s_cu[a.n_seqs];
  const int end = min((int)(blockIdx.x + 1) * kPlanRowsPerGroup, a.n_tokens);
  for (int n = blockIdx.x * kPlanRowsPerGroup + tid; n < end; n += PT) {
    int seq = -1, pos = -1;
    if (n < rows) {
      int lo = 0, hi = a.n_seqs - 1;  // last sequence that starts at or before row n
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_cu[mid] <= n) lo = mid;
        else hi = mid - 1;
      }
      seq = lo;
      const int kv = min(max(a.kv_lengths[lo], 0), a.max_keys);
      pos = kv - max(a.q_lengths[lo], 0) + (n - s_cu[lo]);
    }
    a.plan[a.layout.seq + n] = seq;
    a.plan[a.layout.pos + n] = pos;
  }
}

// One wave per row and query head, 16 lanes per key, four keys at a time: each 16-lane group keeps
// the running maximum and sum of its keys, the groups meet at the end.
template <class E>
__global__ __launch_bounds__(256) void paged_row_kernel(PagedAttnArgs a) {
  constexpr int D = kHeadDim;
  const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (item >= (long)a.n_tokens * a.hq) return;
  const int row = (int)(item / a.hq), h = (int)(item % a.hq), lane = threadIdx.x & 63;
  const int kvh = h / (a.hq / a.hkv), grp = lane >> 4, d0 = 8 * (lane & 15);
  const int seq = a.plan[a.layout.seq + row];
  const int keys = seq < 0 ? 0 : a.plan[a.layout.pos + row] + 1;
  const int ps = 1 << a.pool.page_shift;
  const uint16_t* k = (const uint16_t*)a.k;
  const uint16_t* v = (const uint16_t*)a.v;
  float q[8], o[8];
  const u32x4 qv = gload16((const uint16_t*)a.q + item * D + d0);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    q[e] = E::to_f32(half_of(qv, e)) * a.scale * kLog2e;
    o[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int t = grp; t < keys; t += 4) {
    const int page = a.pool.table[(long)seq * a.pool.table_width + (t >> a.pool.page_shift)];
    u32x4 kv = u32x4{0u, 0u, 0u, 0u}, vv = kv;
    if (page >= 0 && page < a.pool.n_pages) {
      const long in = ((long)kvh * ps + (t & (ps - 1))) * D + d0;
      kv = gload16(k + page * a.pool.k_stride + in);
      vv = gload16(v + page * a.pool.v_stride + in);
    }
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(q[e], E::to_f32(half_of(kv, e)), s);
    s = sum_rows16(s);
    const float m_new = fmaxf(m, s);
    const float m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = fast_exp2(m - m_use), p = fast_exp2(s - m_use);
    m = m_new;
    l = l * alpha + p;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = fmaf(o[e], alpha, p * E::to_f32(half_of(vv, e)));
  }
#pragma unroll
  for (int off = 16; off < 64; off <<= 1) {
    const float m_b = __shfl_xor(m, off), m_tot = fmaxf(m, m_b);
    const float m_use = m_tot == -INFINITY ? 0.f : m_tot;
    const float ca = fast_exp2(m - m_use), cb = fast_exp2(m_b - m_use);
    m = m_tot;
    l = l * ca + __shfl_xor(l, off) * cb;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = o[e] * ca + __shfl_xor(o[e], off) * cb;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (grp == 0)
    gstore16((uint16_t*)a.out + item * D + d0,
             pack8<E>(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv, o[4] * inv, o[5] * inv,
                      o[6] * inv, o[7] * inv));
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs& a) {
  const int groups = max(1, (a.n_tokens + kPlanRowsPerGroup - 1) / kPlanRowsPerGroup);
  hipLaunchKernelGGL(paged_plan_kernel, dim3(groups), dim3(PT), 0, a.stream, a);
  return hipGetLastError();
}

hipError_t launch_paged_attention(const PagedAttnArgs& a) {
  const unsigned groups = (unsigned)(((long)a.n_tokens * a.hq + 3) / 4);
  if (a.dtype == 0) hipLaunchKernelGGL(paged_row_kernel<F16>, dim3(groups), dim3(256), 0, a.stream, a);
  else hipLaunchKernelGGL(paged_row_kernel<BF16>, dim3(groups), dim3(256), 0, a.stream, a);
  return hipGetLastError();
}

}  // namespace va
