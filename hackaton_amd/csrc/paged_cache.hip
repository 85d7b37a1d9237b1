// Page bookkeeping of a paged key/value cache: the next step's page tables (sequences forked, cut,
// freed and grown; pages shared by count) and the move of live pages to the front of the pool.
// Everything is read and decided on the device, so a program that knows its lengths only there
// needs no host read, and a captured step follows them.
#include <climits>

#include "va_common.h"
#include "va_kernels.h"
#include "va_paged.h"
#include "va_scan.h"

namespace va {

namespace {

constexpr int T = 256;        // threads of the wide kernels
constexpr int ST = 1024;      // threads of the one work-group that hands out pages
constexpr int kCopyGroups = 2048;  // work-groups that copy rows (eight per CU)

// scratch words: per page the count without part-filled last pages, the lowest row that ends in the
// page (INT_MAX: none; kTaken: handed out in this call) and the pages handed out, in order; per row
// its first entry in that list and the rows that copy their last page; then the totals.
constexpr int kTaken = -1;
enum { kNeed = 0, kCopies = 1, kFailed = 2 };
struct Scratch {
  int32_t *count, *keeper, *list, *start, *copies, *totals;
};
__device__ inline Scratch scratch_of(const PagesArgs& a) {
  int32_t* p = a.scratch;
  return Scratch{p, p + a.n_pages, p + 2 * (long)a.n_pages, p + 3 * (long)a.n_pages,
                 p + 3 * (long)a.n_pages + a.n_slots, p + 3 * (long)a.n_pages + 2 * (long)a.n_slots};
}

__device__ inline int pages_of(const PagesArgs& a, int tokens) {
  return (int)(((long)tokens + (1 << a.page_shift) - 1) >> a.page_shift);
}
__device__ inline int clamp_length(const PagesArgs& a, int tokens) {
  return (int)min((long)max(tokens, 0), (long)a.width << a.page_shift);
}
__device__ inline bool is_page(const PagesArgs& a, int page) { return page >= 0 && page < a.n_pages; }

// What row `slot` keeps of its parent, and what it becomes.
struct Slot {
  int parent, kept, wanted, kept_pages, wanted_pages;
  bool part;  // the last kept page is part-filled
};
__device__ inline Slot slot_of(const PagesArgs& a, int slot) {
  Slot r;
  const int p = a.parents == nullptr ? slot : a.parents[slot];
  r.parent = p >= 0 && p < a.n_slots ? p : -1;
  const int had = r.parent < 0 ? 0 : clamp_length(a, a.lengths[r.parent]);
  r.wanted = a.new_lengths == nullptr ? had : max(a.new_lengths[slot], 0);
  r.kept = min(had, r.wanted);
  r.kept_pages = pages_of(a, r.kept);
  r.wanted_pages = pages_of(a, r.wanted);
  r.part = (r.kept & ((1 << a.page_shift) - 1)) != 0;
  return r;
}

__global__ __launch_bounds__(T) void remap_clear_kernel(PagesArgs a) {
  const Scratch sc = scratch_of(a);
  const int p = blockIdx.x * T + threadIdx.x;
  if (p >= a.n_pages) return;
  sc.count[p] = a.refs[p];
  sc.keeper[p] = INT_MAX;
}

// One work-group per row: its old pages are given back, the pages it keeps counted (whole adds and a
// minimum, so their order does not matter) and written to its new table row.
__global__ __launch_bounds__(T) void remap_rows_kernel(PagesArgs a) {
  const Scratch sc = scratch_of(a);
  const int slot = blockIdx.x;
  const Slot s = slot_of(a, slot);
  const int old_pages = pages_of(a, clamp_length(a, a.lengths[slot]));
  const int32_t* mine = a.table + (long)slot * a.width;
  const int32_t* from = a.table + (long)max(s.parent, 0) * a.width;
  for (int j = threadIdx.x; j < a.width; j += T) {
    const bool keep = j < s.kept_pages, tail = keep && s.part && j == s.kept_pages - 1;
    const int page = keep ? from[j] : -1;
    a.table_out[(long)slot * a.width + j] = page;
    if (s.parent == slot && keep && !tail) continue;  // held before and after
    if (j < old_pages && is_page(a, mine[j])) atomicAdd(&sc.count[mine[j]], -1);
    if (!keep || !is_page(a, page)) continue;
    if (tail) atomicMin(&sc.keeper[page], slot);
    else atomicAdd(&sc.count[page], 1);
  }
}

// Whether row `slot` gets a copy of its last kept page: another row or the program holds it too.
__device__ inline int has_copy(const PagesArgs& a, const Scratch& sc, int slot, const Slot& s) {
  if (!s.part) return 0;
  const int last = a.table_out[(long)slot * a.width + s.kept_pages - 1];
  return is_page(a, last) && !(sc.count[last] <= 0 && sc.keeper[last] == slot);
}

// One work-group hands out the free pages: how many every row needs, then the free pages in
// ascending order until all are served.
__global__ __launch_bounds__(ST) void remap_hand_out_kernel(PagesArgs a) {
  __shared__ long long s_scan[ST / 64];
  const Scratch sc = scratch_of(a);
  const int tid = threadIdx.x;
  long long need = 0, copies = 0, beyond = 0;  // totals so far
  for (int base = 0; base < a.n_slots; base += ST) {
    const int slot = base + tid;
    long long mine = 0, copy = 0, over = 0;
    if (slot < a.n_slots) {
      const Slot s = slot_of(a, slot);
      copy = has_copy(a, sc, slot, s);
      mine = copy + s.wanted_pages - s.kept_pages;
      over = max(0, s.wanted_pages - a.width);
    }
    long long all;
    const long long before = block_exclusive_sum<ST / 64>(mine, s_scan, all);
    if (slot < a.n_slots) sc.start[slot] = (int)min(need + before, (long long)INT_MAX);
    need += all;
    const long long place = block_exclusive_sum<ST / 64>(copy, s_scan, all);
    if (copy) sc.copies[copies + place] = slot;
    copies += all;
    block_exclusive_sum<ST / 64>(over, s_scan, all);
    beyond += all;
  }
  long long found = 0;
  for (int base = 0; base < a.n_pages && found < need; base += ST) {
    const int page = base + tid;
    const bool is_free = page < a.n_pages && sc.count[page] <= 0 && sc.keeper[page] == INT_MAX;
    long long all;
    const long long at = found + block_exclusive_sum<ST / 64>((long long)is_free, s_scan, all);
    if (is_free && at < need) {
      sc.list[at] = page;
      sc.keeper[page] = kTaken;
    }
    found += all;
  }
  if (tid == 0) {
    const long long lacking = max(0LL, need - found) + beyond;
    sc.totals[kNeed] = (int)min(need, (long long)INT_MAX);
    sc.totals[kCopies] = (int)copies;
    sc.totals[kFailed] = lacking != 0;
    a.result[0] = (int)min(lacking, (long long)INT_MAX);
  }
}

// The last step: work-groups below n_slots write the rows' new pages, the next ones the counts, the
// others copy the part-filled pages. Where the pages did not suffice everything stays as it was.
__global__ __launch_bounds__(T) void remap_finish_kernel(PagesArgs a, int count_groups) {
  const Scratch sc = scratch_of(a);
  const bool failed = sc.totals[kFailed] != 0;
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < a.n_slots) {
    const int slot = blockIdx.x;
    int32_t* out = a.table_out + (long)slot * a.width;
    if (failed) {
      for (int j = tid; j < a.width; j += T) out[j] = a.table[(long)slot * a.width + j];
      if (tid == 0) a.lengths_out[slot] = a.lengths[slot];
      return;
    }
    const Slot s = slot_of(a, slot);
    const int copy = has_copy(a, sc, slot, s);
    const int32_t* list = sc.list + sc.start[slot];
    for (int j = s.kept_pages + tid; j < s.wanted_pages; j += T) out[j] = list[copy + j - s.kept_pages];
    if (tid == 0) a.lengths_out[slot] = s.wanted;
    __syncthreads();  // every thread has read the row's last kept page
    if (tid == 0 && copy) out[s.kept_pages - 1] = list[0];
    return;
  }
  if ((int)blockIdx.x < a.n_slots + count_groups) {
    const int p = (blockIdx.x - a.n_slots) * T + tid;
    if (p >= a.n_pages) return;
    const int held = sc.keeper[p] == kTaken || (sc.keeper[p] != INT_MAX && sc.count[p] <= 0);
    a.refs_out[p] = failed ? a.refs[p] : held ? 1 : max(sc.count[p], 0);
    return;
  }
  if (failed) return;
  const long units = (long)sc.totals[kCopies] * a.outer;
  const int ps = 1 << a.page_shift, row_chunks = kHeadDim / 8;
  const long page_chunks = (long)a.kv_heads * ps * row_chunks;
  u32x4* pages = (u32x4*)a.pages;
  for (long u = blockIdx.x - a.n_slots - count_groups; u < units; u += kCopyGroups) {
    const int slot = sc.copies[u / a.outer];
    const long o = u % a.outer;
    const Slot s = slot_of(a, slot);
    const int src = a.table[(long)s.parent * a.width + s.kept_pages - 1];
    const int dst = sc.list[sc.start[slot]];
    const int run = (s.kept & (ps - 1)) * row_chunks;  // 16-byte chunks of a head
    const u32x4* from = pages + (o * a.n_pages + src) * page_chunks;
    u32x4* to = pages + (o * a.n_pages + dst) * page_chunks;
    for (int i = tid; i < run * a.kv_heads; i += T) {
      const int at = i / run * (ps * row_chunks) + i % run;
      to[at] = from[at];
    }
  }
}

// ------------------------------------------------------------------------------------------------
// compaction: scratch words are place (where every page goes), from (where it comes from) and the
// movers' list; totals hold their number and the live pages.
// ------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(ST) void compact_plan_kernel(PagesArgs a) {
  __shared__ int s_scan[ST / 64];
  const Scratch sc = scratch_of(a);
  int32_t *place = sc.count, *from = sc.keeper, *movers = sc.list;
  const int tid = threadIdx.x;
  int n_live = 0, all;
  for (int base = 0; base < a.n_pages; base += ST) {
    const int p = base + tid;
    block_exclusive_sum<ST / 64>((int)(p < a.n_pages && a.refs[p] > 0), s_scan, all);
    n_live += all;
  }
  // live pages past n_live, in order; then the free pages below it take them in the same order
  int moves = 0, holes = 0;
  for (int base = 0; base < a.n_pages; base += ST) {
    const int p = base + tid;
    const bool moves_out = p < a.n_pages && p >= n_live && a.refs[p] > 0;
    const int at = block_exclusive_sum<ST / 64>((int)moves_out, s_scan, all);
    if (moves_out) movers[moves + at] = p;
    moves += all;
  }
  __syncthreads();
  for (int base = 0; base < a.n_pages; base += ST) {
    const int p = base + tid;
    const bool hole = p < n_live && a.refs[p] <= 0;
    const int at = block_exclusive_sum<ST / 64>((int)hole, s_scan, all);
    if (hole) {
      const int src = movers[holes + at];
      place[src] = p;
      from[p] = src;
    } else if (p < a.n_pages) {
      from[p] = p;
      if (p < n_live) place[p] = p;
    }
    holes += all;
  }
  if (tid == 0) {
    sc.totals[0] = moves;
    a.result[0] = n_live;
  }
}

__global__ __launch_bounds__(T) void compact_move_kernel(PagesArgs a, int count_groups) {
  const Scratch sc = scratch_of(a);
  const int32_t *place = sc.count, *from = sc.keeper, *movers = sc.list;
  const int n_live = a.result[0], tid = threadIdx.x;
  if ((int)blockIdx.x < a.n_slots) {
    const long row = (long)blockIdx.x * a.width;
    const int used = pages_of(a, clamp_length(a, a.lengths[blockIdx.x]));
    for (int j = tid; j < a.width; j += T) {
      const int page = j < used ? a.table[row + j] : -1;
      a.table_out[row + j] = is_page(a, page) && a.refs[page] > 0 ? place[page] : -1;
    }
    return;
  }
  if ((int)blockIdx.x < a.n_slots + count_groups) {
    const int p = (blockIdx.x - a.n_slots) * T + tid;
    if (p < a.n_pages) a.refs_out[p] = p < n_live ? a.refs[from[p]] : 0;
    return;
  }
  const long page_chunks = (long)a.kv_heads * (kHeadDim / 8) << a.page_shift;
  u32x4* pages = (u32x4*)a.pages;
  const long units = (long)sc.totals[0] * a.outer;
  for (long u = blockIdx.x - a.n_slots - count_groups; u < units; u += kCopyGroups) {
    const int src = movers[u / a.outer];
    const long layer = u % a.outer * a.n_pages;
    const u32x4* x = pages + (layer + src) * page_chunks;
    u32x4* y = pages + (layer + place[src]) * page_chunks;
    for (long i = tid; i < page_chunks; i += T) y[i] = x[i];
  }
}

}  // namespace

hipError_t launch_pages_remap(const PagesArgs& a) {
  const int count_groups = (a.n_pages + T - 1) / T;
  if (count_groups > 0)
    hipLaunchKernelGGL(remap_clear_kernel, dim3(count_groups), dim3(T), 0, a.stream, a);
  if (a.n_slots > 0)
    hipLaunchKernelGGL(remap_rows_kernel, dim3(a.n_slots), dim3(T), 0, a.stream, a);
  hipLaunchKernelGGL(remap_hand_out_kernel, dim3(1), dim3(ST), 0, a.stream, a);
  hipLaunchKernelGGL(remap_finish_kernel, dim3(a.n_slots + count_groups + kCopyGroups), dim3(T), 0,
                     a.stream, a, count_groups);
  return hipGetLastError();
}

hipError_t launch_pages_compact(const PagesArgs& a) {
  const int count_groups = (a.n_pages + T - 1) / T;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(ST), 0, a.stream, a);
  hipLaunchKernelGGL(compact_move_kernel, dim3(a.n_slots + count_groups + kCopyGroups), dim3(T), 0,
                     a.stream, a, count_groups);
  return hipGetLastError();
}

}  // namespace va
