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
constexpr int ST = 1024;      // threads of the one work-group that counts and hands out pages
constexpr int SW = ST / 64;
constexpr int PER = 4;        // pages per thread and step
constexpr int kCopyGroups = 2048;  // work-groups that copy rows (eight per CU)
constexpr int kLdsPages = 16384;   // pages whose counts fit in LDS (128 KB) beside 1024 rows

// scratch words: per page the count without part-filled last pages, the lowest row that ends in the
// page (INT_MAX: none; kTaken: handed out in this call) and the pages handed out, in order; per row
// its parent, what it keeps and becomes, its first entry in that list (kCopied: the row copies its last
// kept page into it) and the rows that copy; then the totals.
constexpr int kTaken = -1, kCopied = 1 << 30;
enum { kCopies = 0, kFailed = 1 };
struct Scratch {
  int32_t *count, *keeper, *list, *parent, *kept, *wanted, *start, *copies, *totals;
};
__device__ inline Scratch scratch_of(const PagesArgs& a) {
  int32_t* p = a.scratch;
  const long pages = a.n_pages, slots = a.n_slots;
  int32_t* rows = p + 3 * pages;
  return Scratch{p, p + pages, p + 2 * pages, rows, rows + slots, rows + 2 * slots, rows + 3 * slots,
                 rows + 4 * slots, rows + 5 * slots};
}

__device__ inline int pages_of(const PagesArgs& a, int tokens) {
  return (int)(((long)tokens + (1 << a.page_shift) - 1) >> a.page_shift);
}
__device__ inline int clamp_length(const PagesArgs& a, int tokens) {
  return (int)min((long)max(tokens, 0), (long)a.width << a.page_shift);
}
__device__ inline bool is_page(const PagesArgs& a, int page) { return page >= 0 && page < a.n_pages; }

// What a row keeps of its parent, and what it becomes.
struct Slot {
  int parent, kept, wanted, kept_pages, wanted_pages;
  bool part;  // the last kept page is part-filled
};
__device__ inline Slot slot_from(const PagesArgs& a, int parent, int kept, int wanted) {
  return Slot{parent, kept, wanted, pages_of(a, kept), pages_of(a, wanted),
              (kept & ((1 << a.page_shift) - 1)) != 0};
}
__device__ inline Slot slot_of(const PagesArgs& a, int slot) {
  const int p = a.parents == nullptr ? slot : a.parents[slot];
  const int parent = p >= 0 && p < a.n_slots ? p : -1;
  const int had = parent < 0 ? 0 : clamp_length(a, a.lengths[parent]);
  const int wanted = a.new_lengths == nullptr ? had : max(a.new_lengths[slot], 0);
  return slot_from(a, parent, min(had, wanted), wanted);
}
// The part-filled last page that a row keeps, or a number that is no page.
__device__ inline int last_page(const PagesArgs& a, const Slot& s) {
  return s.part ? a.table[(long)s.parent * a.width + s.kept_pages - 1] : -1;
}

// Row `slot` gives back its old pages and holds the ones it keeps, entries first, first + step, ...:
// whole adds and a minimum, so their order does not matter.
__device__ inline void count_row(const PagesArgs& a, int slot, const Slot& s, int old_pages, int first,
                                 int step, int32_t* count, int32_t* keeper) {
  const int32_t* mine = a.table + (long)slot * a.width;
  const int32_t* from = a.table + (long)max(s.parent, 0) * a.width;
  const int whole = s.kept_pages - s.part;
  // (its own whole pages are held before and after)
  for (int j = first + (s.parent == slot ? whole : 0); j < max(old_pages, s.kept_pages); j += step) {
    if (j < old_pages && is_page(a, mine[j])) atomicAdd(&count[mine[j]], -1);
    if (j >= s.kept_pages || !is_page(a, from[j])) continue;
    if (j >= whole) atomicMin(&keeper[from[j]], slot);
    else atomicAdd(&count[from[j]], 1);
  }
}

// out[p] = value(p) for all pages, by one work-group: four at a time where `out` is 16-byte aligned.
template <class Value>
__device__ inline void for_pages(const PagesArgs& a, int32_t* out, Value value) {
  const bool wide = ((uintptr_t)out & 15) == 0;
  for (int p = 4 * threadIdx.x; p < a.n_pages; p += 4 * ST) {
    if (wide && p + 4 <= a.n_pages) {
      *reinterpret_cast<int4*>(out + p) = int4{value(p), value(p + 1), value(p + 2), value(p + 3)};
    } else {
      for (int i = p; i < min(p + 4, a.n_pages); ++i) out[i] = value(i);
    }
  }
}

// One work-group hands out the free pages: how many every row needs, then the free pages in ascending
// order until all are served. info(slot, last) gives a row and its part-filled last page.
template <class Info>
__device__ inline void hand_out(const PagesArgs& a, const Scratch& sc, int32_t* count, int32_t* keeper,
                                int* s_scan, Info info) {
  const int tid = threadIdx.x;
  long long need = 0, beyond = 0;
  int first = 0, copies = 0;  // so far (`first` wraps only where the total passes the pages)
  for (int base = 0; base < a.n_slots; base += ST) {
    const int slot = base + tid;
    // pages, copies; pages and pages beyond the table row in pieces whose sums stay in 32 bits
    int x[6] = {}, total[6];
    if (slot < a.n_slots) {
      int last;
      const Slot s = info(slot, last);
      x[1] = is_page(a, last) && !(count[last] <= 0 && keeper[last] == slot);
      x[0] = x[1] + s.wanted_pages - s.kept_pages;
      const int over = max(0, s.wanted_pages - a.width);
      x[2] = x[0] & 0x7fff;
      x[3] = x[0] >> 15;
      x[4] = over & 0x7fff;
      x[5] = over >> 15;
      sc.parent[slot] = s.parent;
      sc.kept[slot] = s.kept;
      sc.wanted[slot] = s.wanted;
    }
    const int copy = x[1];
    block_exclusive_sums<SW>(x, total, s_scan);
    if (slot < a.n_slots) sc.start[slot] = ((first + x[0]) & (kCopied - 1)) | (copy ? kCopied : 0);
    if (copy) sc.copies[copies + x[1]] = slot;
    first += total[0];
    copies += total[1];
    need += ((long long)total[3] << 15) + total[2];
    beyond += ((long long)total[5] << 15) + total[4];
  }
  long long found = 0;
  for (int base = 0; base < a.n_pages && found < need; base += PER * ST) {
    bool is_free[PER];
    int at[PER], total;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int page = base + i * ST + tid;
      is_free[i] = page < a.n_pages && count[page] <= 0 && keeper[page] == INT_MAX;
    }
    block_places<SW>(is_free, at, total, s_scan);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (is_free[i] && found + at[i] < need) {
        sc.list[found + at[i]] = base + i * ST + tid;
        keeper[base + i * ST + tid] = kTaken;
      }
    found += total;
  }
  const long long lacking = max(0LL, need - found) + beyond;
  if (tid == 0) {
    sc.totals[kCopies] = copies;
    sc.totals[kFailed] = lacking != 0;
    a.result[0] = (int)min(lacking, (long long)INT_MAX);
  }
  // the counts of the next step, or of this one again
  __syncthreads();
  for_pages(a, a.refs_out, [&](int p) {
    const int k = keeper[p], c = count[p];
    return lacking != 0 ? a.refs[p] : k == kTaken || (k != INT_MAX && c <= 0) ? 1 : max(c, 0);
  });
}

// Pools of up to kLdsPages pages and up to 1024 rows: one work-group counts in LDS and hands out. What
// the rows are is read once, beside the counts.
__global__ __launch_bounds__(ST) void remap_small_kernel(PagesArgs a) {
  __shared__ __attribute__((aligned(16))) int32_t s_count[kLdsPages], s_keeper[kLdsPages];
  __shared__ int s_parent[ST], s_kept[ST], s_wanted[ST], s_last[ST], s_old[ST];
  __shared__ int s_scan[6 * SW];
  const int tid = threadIdx.x;
  if (tid < a.n_slots) {
    const Slot s = slot_of(a, tid);
    s_parent[tid] = s.parent;
    s_kept[tid] = s.kept;
    s_wanted[tid] = s.wanted;
    s_last[tid] = last_page(a, s);
    s_old[tid] = pages_of(a, clamp_length(a, a.lengths[tid]));
  }
  const bool wide = ((uintptr_t)a.refs & 15) == 0;
#pragma unroll 4
  for (int p = 4 * tid; p < a.n_pages; p += 4 * ST) {
    int4 r;
    if (wide && p + 4 <= a.n_pages) {
      r = *reinterpret_cast<const int4*>(a.refs + p);
    } else {
      int* const one[4] = {&r.x, &r.y, &r.z, &r.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) *one[i] = p + i < a.n_pages ? a.refs[p + i] : 0;
    }
    *reinterpret_cast<int4*>(s_count + p) = r;  // (kLdsPages is a multiple of 4)
    *reinterpret_cast<int4*>(s_keeper + p) = int4{INT_MAX, INT_MAX, INT_MAX, INT_MAX};
  }
  __syncthreads();
  // 16 lanes per row: rows that go on as themselves only have their last page to look at
  for (int slot = tid >> 4; slot < a.n_slots; slot += ST / 16)
    count_row(a, slot, slot_from(a, s_parent[slot], s_kept[slot], s_wanted[slot]), s_old[slot], tid & 15,
              16, s_count, s_keeper);
  __syncthreads();
  hand_out(a, scratch_of(a), s_count, s_keeper, s_scan, [&](int slot, int& last) {
    last = s_last[slot];
    return slot_from(a, s_parent[slot], s_kept[slot], s_wanted[slot]);
  });
}

__global__ __launch_bounds__(T) void remap_clear_kernel(PagesArgs a) {
  const Scratch sc = scratch_of(a);
  const int p = blockIdx.x * T + threadIdx.x;
  if (p >= a.n_pages) return;
  sc.count[p] = a.refs[p];
  sc.keeper[p] = INT_MAX;
}
__global__ __launch_bounds__(T) void remap_rows_kernel(PagesArgs a) {
  const Scratch sc = scratch_of(a);
  const int slot = blockIdx.x;
  count_row(a, slot, slot_of(a, slot), pages_of(a, clamp_length(a, a.lengths[slot])), threadIdx.x, T,
            sc.count, sc.keeper);
}
__global__ __launch_bounds__(ST) void remap_hand_out_kernel(PagesArgs a) {
  __shared__ int s_scan[6 * SW];
  const Scratch sc = scratch_of(a);
  hand_out(a, sc, sc.count, sc.keeper, s_scan, [&](int slot, int& last) {
    const Slot s = slot_of(a, slot);
    last = last_page(a, s);
    return s;
  });
}

// A step's lengths: every row's with its new tokens, unless those pass the step's rows all together. (A
// few KB at most: bounded by its launch, 2 us, in place of a clamp, a sum and an addition.)
__global__ __launch_bounds__(ST) void growth_kernel(PagesGrowthArgs a) {
  __shared__ int s_scan[3 * SW];
  long long sum = 0;
  for (int i = threadIdx.x; i < a.n_slots; i += ST) sum += max(a.q_lengths[i], 0);
  // (pieces of 20 bits: 1024 threads of them stay in 32)
  int x[3] = {(int)(sum & 0xfffff), (int)(sum >> 20 & 0xfffff), (int)(sum >> 40)}, total[3];
  block_exclusive_sums<SW>(x, total, s_scan);
  const long long excess =
      ((long long)total[2] << 40) + ((long long)total[1] << 20) + total[0] - a.n_tokens;
  for (int i = threadIdx.x; i < a.n_slots; i += ST) {
    const int q = excess > 0 ? 0 : max(a.q_lengths[i], 0);
    a.new_lengths[i] = (int)min((long long)a.lengths[i] + q, (long long)INT_MAX);
  }
  if (threadIdx.x == 0 && excess > 0)
    a.excess[0] = max(a.excess[0], (int)min(excess, (long long)INT_MAX));
}

// The last step: work-groups below n_slots write the rows, the others copy the part-filled pages. Where
// the pages did not suffice everything stays as it was.
__global__ __launch_bounds__(T) void remap_finish_kernel(PagesArgs a) {
  const Scratch sc = scratch_of(a);
  const bool failed = sc.totals[kFailed] != 0;
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < a.n_slots) {
    const int slot = blockIdx.x;
    const Slot s = slot_from(a, sc.parent[slot], sc.kept[slot], sc.wanted[slot]);
    const int32_t* from = a.table + (long)(failed ? slot : max(s.parent, 0)) * a.width;
    const int given = sc.start[slot], copy = (given & kCopied) != 0;
    // page j of the row is list[j] for the copied last page and the ones that it grows by
    const int32_t* list = sc.list + (long)(given & (kCopied - 1)) - (s.kept_pages - copy);
    for (int j = tid; j < a.width; j += T) {
      int page = -1;
      if (failed || j < s.kept_pages - copy) page = from[j];
      else if (j < s.wanted_pages) page = list[j];
      a.table_out[(long)slot * a.width + j] = page;
    }
    if (tid == 0) a.lengths_out[slot] = failed ? a.lengths[slot] : s.wanted;
    return;
  }
  if (failed) return;
  const long units = (long)sc.totals[kCopies] * a.outer;
  const int ps = 1 << a.page_shift, row_chunks = a.row_chunks;
  const long page_chunks = (long)a.kv_heads * ps * row_chunks;
  u32x4* pages = (u32x4*)a.pages;
  for (long u = blockIdx.x - a.n_slots; u < units; u += kCopyGroups) {
    const int slot = sc.copies[u / a.outer];
    const long o = u % a.outer;
    const Slot s = slot_from(a, sc.parent[slot], sc.kept[slot], sc.wanted[slot]);
    const int src = last_page(a, s), dst = sc.list[sc.start[slot] & (kCopied - 1)];
    const int run = (s.kept & (ps - 1)) * row_chunks;  // 16-byte chunks of a head
    const u32x4* from = pages + (o * a.n_pages + src) * page_chunks;
    u32x4* to = pages + (o * a.n_pages + dst) * page_chunks;
    for (int i = tid; i < run * a.kv_heads; i += T) {
      const int at = i / run * (ps * row_chunks) + i % run;
      to[at] = from[at];
    }
    if (a.exps != nullptr) {  // (a byte per row)
      const int rows = s.kept & (ps - 1);
      const uint8_t* x = a.exps + (o * a.n_pages + src) * a.kv_heads * ps;
      uint8_t* y = a.exps + (o * a.n_pages + dst) * a.kv_heads * ps;
      for (int i = tid; i < rows * a.kv_heads; i += T) {
        const int at = i / rows * ps + i % rows;
        y[at] = x[at];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------
// compaction: scratch words are the pages that move, the free pages that take them (in the same order),
// for a page that moves its new place and for a page that is taken where its rows come from.
// ------------------------------------------------------------------------------------------------
struct Moves {
  int32_t *movers, *holes, *other, *totals;
};
__device__ inline Moves moves_of(const PagesArgs& a) {
  const Scratch sc = scratch_of(a);
  return Moves{sc.count, sc.keeper, sc.list, sc.totals};
}

__global__ __launch_bounds__(ST) void compact_plan_kernel(PagesArgs a) {
  __shared__ int s_scan[PER * SW];
  const Moves mv = moves_of(a);
  const int tid = threadIdx.x;
  int live[1] = {0}, all[1];
#pragma unroll 4
  for (int p = tid; p < a.n_pages; p += ST) live[0] += a.refs[p] > 0;
  block_exclusive_sums<SW>(live, all, s_scan);
  const int n_live = all[0];
  int holes = 0;
  for (int base = 0; base < a.n_pages; base += PER * ST) {
    bool wanted[PER];
    int at[PER], total;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int p = base + i * ST + tid;
      wanted[i] = p < a.n_pages && (a.refs[p] > 0) != (p < n_live);
    }
    // (free pages below n_live, then live pages from n_live on: a step that has both has them in this
    // order, and the holes' total is known when the movers begin)
    block_places<SW>(wanted, at, total, s_scan);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (wanted[i]) {
        const int p = base + i * ST + tid;
        if (p < n_live) mv.holes[holes + at[i]] = p;
        else mv.movers[holes + at[i]] = p;  // shifted by all holes, taken back below
      }
    holes += total;
  }
  const int moves = holes / 2;  // as many pages move as are taken
  __syncthreads();
  for (int k = tid; k < moves; k += ST) {
    const int src = mv.movers[moves + k], dst = mv.holes[k];
    mv.other[src] = dst;
    mv.other[dst] = src;
  }
  if (tid == 0) {
    mv.totals[0] = moves;
    a.result[0] = n_live;
  }
}

__global__ __launch_bounds__(T) void compact_move_kernel(PagesArgs a, int count_groups) {
  const Moves mv = moves_of(a);
  const int n_live = a.result[0], moves = mv.totals[0], tid = threadIdx.x;
  if ((int)blockIdx.x < a.n_slots) {
    const long row = (long)blockIdx.x * a.width;
    const int used = pages_of(a, clamp_length(a, a.lengths[blockIdx.x]));
    for (int j = tid; j < a.width; j += T) {
      const int page = j < used ? a.table[row + j] : -1;
      const bool held = is_page(a, page) && a.refs[page] > 0;
      a.table_out[row + j] = !held ? -1 : page < n_live ? page : mv.other[page];
    }
    return;
  }
  if ((int)blockIdx.x < a.n_slots + count_groups) {
    const int p = (blockIdx.x - a.n_slots) * T + tid;
    if (p >= a.n_pages) return;
    const int own = a.refs[p];
    a.refs_out[p] = p >= n_live ? 0 : own > 0 ? own : a.refs[mv.other[p]];
    return;
  }
  const long page_chunks = (long)a.kv_heads * a.row_chunks << a.page_shift;
  const long page_exps = (long)a.kv_heads << a.page_shift;  // (a multiple of 16)
  u32x4* pages = (u32x4*)a.pages;
  const long units = (long)moves * a.outer;
  for (long u = blockIdx.x - a.n_slots - count_groups; u < units; u += kCopyGroups) {
    const int src = mv.movers[moves + u / a.outer];
    const long layer = u % a.outer * a.n_pages;
    const u32x4* x = pages + (layer + src) * page_chunks;
    u32x4* y = pages + (layer + mv.other[src]) * page_chunks;
    for (long i = tid; i < page_chunks; i += T) y[i] = x[i];
    if (a.exps != nullptr) {
      const u32x4* from = reinterpret_cast<const u32x4*>(a.exps + (layer + src) * page_exps);
      u32x4* to = reinterpret_cast<u32x4*>(a.exps + (layer + mv.other[src]) * page_exps);
      for (long i = tid; i < page_exps / 16; i += T) to[i] = from[i];
    }
  }
}

// ------------------------------------------------------------------------------------------------
// accepted paths: a work-group per sequence and (layer, keys or values). Token path[i] of the sequence's
// new ones goes to place i behind the cached rows; path[i] >= i and ascending, so that rows read together
// may be written together once all of them are in registers, front to back. Bounded by its launch for
// the paths that drafted trees have (tens of rows of a few hundred bytes).
// ------------------------------------------------------------------------------------------------
constexpr int kAcceptLoads = 4;  // 16-byte pieces per thread between two barriers
__global__ __launch_bounds__(T) void accept_kernel(PagedAcceptArgs a) {
  __shared__ int s_path[kTreeTokens], s_page_of[2][kTreeTokens];
  const int s = blockIdx.y, tid = threadIdx.x;
  const long o = blockIdx.x;
  int first = 0, count = 0;
  if (a.n_tokens > 0) {
    first = min(max(a.plan[s], 0), a.n_tokens);
    count = max(min(a.plan[s + 1], a.n_tokens) - first, 0);
  }
  const int last = a.accepted[s];
  const bool some = last >= 0 && last < count;
  const bool chain = a.tree == nullptr || count > kTreeTokens;
  int kept = !some ? 0 : last + 1, moved = 0;  // rows that stay; of them, those that are in place
  if (some && !chain) {
    const uint32_t* words = reinterpret_cast<const uint32_t*>(a.tree) + (long)(first + last) * kTreeWords;
    int before = 0;
    kept = 0;
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) {
      const uint32_t x = words[w];
      const int mine = tid >> 5;
      if (w < mine) before += __builtin_popcount(x);
      if (w == mine) before += __builtin_popcount(x & ((1u << (tid & 31)) - 1));
      kept += __builtin_popcount(x);
    }
    if (words[tid >> 5] >> (tid & 31) & 1) s_path[before] = tid;
    // (a token is in place where all before it are on the path)
    moved = kept;
    for (int w = kTreeWords - 1; w >= 0; --w)
      if (~words[w] != 0) moved = min(kept, 32 * w + __builtin_ctz(~words[w]));
  }
  // The place of the first new token as the plan has it: where the rows lie. (`lengths` may count tokens that
  // the step had no rows for, or that pass the table row.)
  const int pos0 = count > 0 ? a.plan[a.layout.pos + first] : 0;
  if (tid == 0 && o == 0) a.lengths_out[s] = count > 0 ? max(pos0 + kept, 0) : a.lengths[s];
  if (!some || chain || moved >= kept || o >= a.outer) return;  // (the same in all threads)
  __syncthreads();
  const int ps = 1 << a.page_shift;
  if (tid < kept) {  // pages of the path's rows and of their new places
    const int32_t* row = a.table + (long)s * a.width;
    const int from = pos0 + s_path[tid], to = pos0 + tid;
    const int x = from >= 0 && from >> a.page_shift < a.width ? row[from >> a.page_shift] : -1;
    const int y = to >= 0 && to >> a.page_shift < a.width ? row[to >> a.page_shift] : -1;
    s_page_of[0][tid] = x < a.n_pages ? x : -1;
    s_page_of[1][tid] = y < a.n_pages ? y : -1;
  }
  __syncthreads();
  u32x4* const pages = (u32x4*)a.pages + o * a.n_pages * a.kv_heads * ps * a.row_chunks;
  const int per_row = a.kv_heads * a.row_chunks, pieces = (kept - moved) * per_row;
  // piece i: chunk i % row_chunks of head i / row_chunks % kv_heads of the (i / per_row)-th row that moves
  auto at = [&](int i, int side) -> long {
    const int r = moved + i / per_row, in = i % per_row, page = s_page_of[side][r];
    const int place = pos0 + (side == 0 ? s_path[r] : r);
    if (page < 0) return -1;
    return (((long)page * a.kv_heads + in / a.row_chunks) * ps + (place & (ps - 1))) * a.row_chunks +
           in % a.row_chunks;
  };
  for (int base = 0; base < pieces; base += kAcceptLoads * T) {
    u32x4 x[kAcceptLoads];
    bool have[kAcceptLoads];
#pragma unroll
    for (int l = 0; l < kAcceptLoads; ++l) {
      const int i = base + l * T + tid;
      const long from = i < pieces ? at(i, 0) : -1;
      have[l] = from >= 0;
      if (have[l]) x[l] = pages[from];
    }
    __syncthreads();
#pragma unroll
    for (int l = 0; l < kAcceptLoads; ++l) {
      const long to = have[l] ? at(base + l * T + tid, 1) : -1;
      if (to >= 0) pages[to] = x[l];
    }
    __syncthreads();
  }
  if (a.exps == nullptr) return;
  uint8_t* const exps = a.exps + o * a.n_pages * a.kv_heads * ps;
  const int bytes = (kept - moved) * a.kv_heads;
  auto exp_at = [&](int i, int side) -> long {
    const int r = moved + i / a.kv_heads, page = s_page_of[side][r];
    const int place = pos0 + (side == 0 ? s_path[r] : r);
    return page < 0 ? -1 : ((long)page * a.kv_heads + i % a.kv_heads) * ps + (place & (ps - 1));
  };
  for (int base = 0; base < bytes; base += T) {
    const int i = base + tid;
    const long from = i < bytes ? exp_at(i, 0) : -1;
    const uint8_t x = from >= 0 ? exps[from] : 0;
    __syncthreads();
    const long to = from >= 0 ? exp_at(i, 1) : -1;
    if (to >= 0) exps[to] = x;
    __syncthreads();
  }
}

}  // namespace

hipError_t launch_paged_accept(const PagedAcceptArgs& a) {
  const bool moves = a.tree != nullptr && a.outer > 0 && a.n_pages > 0;
  hipLaunchKernelGGL(accept_kernel, dim3(moves ? (unsigned)a.outer : 1, a.n_seqs), dim3(T), 0, a.stream, a);
  return hipGetLastError();
}

hipError_t launch_pages_growth(const PagesGrowthArgs& a) {
  hipLaunchKernelGGL(growth_kernel, dim3(1), dim3(ST), 0, a.stream, a);
  return hipGetLastError();
}

hipError_t launch_pages_remap(const PagesArgs& a) {
  if (a.n_pages <= kLdsPages && a.n_slots <= ST) {
    hipLaunchKernelGGL(remap_small_kernel, dim3(1), dim3(ST), 0, a.stream, a);
  } else {
    if (a.n_pages > 0)
      hipLaunchKernelGGL(remap_clear_kernel, dim3((a.n_pages + T - 1) / T), dim3(T), 0, a.stream, a);
    if (a.n_slots > 0)
      hipLaunchKernelGGL(remap_rows_kernel, dim3(a.n_slots), dim3(T), 0, a.stream, a);
    hipLaunchKernelGGL(remap_hand_out_kernel, dim3(1), dim3(ST), 0, a.stream, a);
  }
  hipLaunchKernelGGL(remap_finish_kernel, dim3(a.n_slots + kCopyGroups), dim3(T), 0, a.stream, a);
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
