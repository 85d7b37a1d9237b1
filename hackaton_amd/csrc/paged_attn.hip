// Attention of a step's new tokens over a paged key/value cache: the plan kernel that places every
// row and splits the work, the attention, and the merge of split key ranges.
//
// An item is a tile of rows x a range of keys of one sequence and key/value head. Rows are (token, query
// head of the group) pairs, so all query heads of a group read a key once. Scores and the running
// maximum, sum and output of every row stay in fp32; weights are rounded to 16 bits for the product
// with the values on v_mfma_f32_32x32x16, and their sum is taken over the rounded ones.
//
//   few rows (up to 32: single and drafted tokens)   the waves share the keys out, each with a K and a V
//       tile of 32 keys of its own in LDS, no barrier until the waves meet at the end;
//   many rows (prompt chunks)   128 rows, a strip of 32 per wave or pair of waves, 64-key tiles in LDS
//       stages that all waves read: two stages and four waves, or four stages and eight waves, where the
//       two waves of a strip take half of a tile's keys each and meet at the end.
//
// Both copy pages straight from memory into LDS (16 rows of a page per wave and step, so a page border
// never falls into a copy), rows past the end of the range as zeros: what earlier sequences left in a
// page is not read (in 8-bit pages it may be, see below). S^T = K Q^T has one row's scores in a lane and its half-wave partner; O^T += V^T
// P^T reads V^T from the row-major tile with transposed LDS reads. A tile's rows are stored in groups of
// 4 (1 KB, one copy instruction) 1088 bytes apart, chunk c of row r at c ^ (r & 3), so that both reads
// touch all banks.
//
// 8-bit pages: an e4m3 number times a power of two is a 16-bit number exactly (four significant bits), in fp16 but
// for its range: past 65504 it is infinite, and below 2^-14 it is rounded to a multiple of 2^-24 (rows of
// numbers around 10^-4 lose digits of their smaller ones, rows around 10^-6 keep a few steps). So
// rows are turned into 16-bit ones on the way, two numbers and their power by one instruction, and the
// products are those of 16-bit pages. Copies go through registers: a wave turns its share of a tile into
// LDS rows while the next tile's loads are in flight. Few rows take keys as the matrix operand straight
// from memory (a lane holds a key's numbers in memory's order, the queries follow it) and only the values,
// which the product needs transposed, through LDS.
// Few rows load whole tiles of 32 keys and their exponents without bounds: bytes behind the range's end, of page 0
// where there is no page, and one tile more behind the last. All lie in the pool (a pool without pages takes
// another path), and none counts: the scores of keys behind the end are replaced by the mask, codes of missing pages
// by zeros, values behind the end read as zeros by the descriptor, and an exponent byte of 255 stands for a
// finite power, so that zero times it is zero.
//
// Trees of new tokens: the tiles that reach past the cached rows read, for every row, the bits of the
// tokens on its path (tree_paths) instead of comparing places.
#include <climits>

#include "../../include/varlen_attn.h"
#include "va_common.h"
#include "va_kernels.h"
#include "va_paged.h"
#include "va_scan.h"

namespace va {

namespace {

// ------------------------------------------------------------------------------------------------
// plan
// ------------------------------------------------------------------------------------------------
constexpr int PT = 256;                     // threads of a planning work-group
constexpr int kPlanRowsPerGroup = 4 * PT;   // rows that a planning work-group places
constexpr int kPlanWriters = 64;            // work-groups that write items (and as many for the merges)

enum { kFew = 0, kMany = 1, kPad = 2, kNone = 3 };  // kinds of items

struct Item {
  int token0, seq, pos0, head;        // the sequence's first row and its position; key/value head | kind << 16
  int row, row_end, key, key_end;     // flattened rows of the sequence and keys
  int part_row;                       // first workspace row of a split range's part, -1: whole
  int pad[3];
};
static_assert(sizeof(Item) == 4 * kPagedItemWords, "item words");

struct Merge {
  int token0, head, row, rows;        // 1 to 8 flattened rows
  int part_row, stride, parts;        // workspace row of the first one in the first part; rows per part;
                                      // parts (0: the rows' only item has written them)
  int spread;                         // one row, whose parts are shared out
};
static_assert(sizeof(Merge) == 4 * kPagedMergeWords, "merge words");

// Tiles of a sequence with `rows` rows, and the keys that the row before `end` sees (pos0: the position
// of the first one).
__device__ inline int tiles_of(int rows, bool narrow) {
  return narrow                  ? (rows + kPagedFewRows - 1) / kPagedFewRows
         : rows <= kPagedFewRows ? (rows > 0)
                                 : (rows + kPagedTileRows - 1) / kPagedTileRows;
}
__device__ inline int keys_of(int pos0, int end, int group) { return max(pos0 + (end - 1) / group + 1, 0); }
// The last of n ascending numbers at or below x (the first one is).
__device__ inline int last_at_most(const int* v, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (v[mid] <= x) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// ------------------------------------------------------------------------------------------------
// trees
// ------------------------------------------------------------------------------------------------
// The paths of a sequence's new tokens by doubling (after round r a token knows the 2^r next ones on
// its way to the root, and the one behind them), a work-group per sequence. Bounded by the latency of
// its first loads and the rounds' barriers.
static_assert(PT == kTreeTokens && PT <= 256, "a thread per token; eight bits of a sequence's number");
struct TreeLds {
  uint32_t path[PT][kTreeWords + 1];
  int next[PT];
};
__device__ inline void tree_paths(const PagedPlanArgs& a, TreeLds& lds, int first, int count, int pos0) {
  const int tid = threadIdx.x;
  int32_t* positions = a.tree + tree_positions(a.n_tokens);
  if (count <= 0) return;  // (the same in all threads)
  if (count > kTreeTokens) {
    for (int j = tid; j < count; j += PT) positions[first + j] = pos0 + j;
    return;
  }
  uint32_t path[kTreeWords];
#pragma unroll
  for (int w = 0; w < kTreeWords; ++w) path[w] = tid >> 5 == w ? 1u << (tid & 31) : 0u;
  int next = tid < count ? a.parents[first + tid] : -1;
  if (next < 0 || next >= tid) next = -1;
  while (__syncthreads_or(next >= 0)) {  // (at most 8 rounds: a parent comes before its token)
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) lds.path[tid][w] = path[w];
    lds.next[tid] = next;
    __syncthreads();
    if (next >= 0) {
#pragma unroll
      for (int w = 0; w < kTreeWords; ++w) path[w] |= lds.path[next][w];
      next = lds.next[next];
    }
  }
  if (tid >= count) return;
  int depth = -1;
#pragma unroll
  for (int w = 0; w < kTreeWords; ++w) depth += __builtin_popcount(path[w]);
  u32x4* words = reinterpret_cast<u32x4*>(a.tree + (long)(first + tid) * kTreeWords);
  words[0] = u32x4{path[0], path[1], path[2], path[3]};
  words[1] = u32x4{path[4], path[5], path[6], path[7]};
  positions[first + tid] = pos0 + depth;
}

// x / by for x >= 0, by > 0. (The division of 64 bits is a hundred instructions, in the one wave of a
// SIMD.)
__device__ inline long long quotient(long long x, long long by) {
  return ((x | by) >> 32) == 0 ? (long long)((uint32_t)x / (uint32_t)by) : x / by;
}

// Two tiles of a sequence read the same keys: on one XCD, the second finds them in its L2. Their items lie hkv apart
// where ranges are not split; in every 16 items of such, the bit that tells them apart changes places with the
// ones above it, which puts them 8 apart. hkv: 1, 2 or 4. (Steps of prompts alone: 32 trees of 24 on 3000, 28/4
// heads 71 -> 64 us, 64 on 64 to 8192, 12/2 heads 50.4 -> 48.2, the plan 0.2 to 0.5 more.)
__device__ inline int paired_tile(int i, int hkv) {
  const int p = hkv >> 1;  // the bit's place: 0, 1, 2
  return (i & ~15) | (i & (hkv - 1)) | (i >> 3 & 1) << p | (i & 7) >> p << (p + 1);
}

// Rows of a merge record: one where few rows have many parts, which are then shared out in it. (16
// trees of 32 tokens on 500 to 16,000, up to 26 parts: 11 us with one row each.)
__device__ inline int merged_rows(bool few, int parts) { return parts <= (few ? 8 : 32) ? 8 : 1; }

// The first `writers` work-groups write the items, as many the merge records, the others place the rows.
// Each sums the lengths by itself (at most 32 KB of them): one launch, nothing handed from one
// work-group to another.
//
// The keys of all tiles of a sequence are split at the same places, into parts of at most `chunk` keys,
// equal but for the last: chunk is the total over the tiles of a kind and all heads (each tile with its
// sequence's longest) divided by the kind's number of parts, so a step of few long tiles fills the card
// with about that many parts, and one of many tiles splits only what is longer than its share.
// Prompt tiles come first, the last (longest) ones of a sequence before its first. Work-group i runs on
// XCD i mod 8: with a multiple of 8 items per tile, the tiles that read the same keys run on one XCD
// and find them in its L2, so the parts are rounded down to that where there are enough of them
// (128 new tokens on 32,768, 28/4 heads: 9 parts per tile and head 85 us, 8 parts 80 us).
// With a tree and one sequence per thread, `n_seqs` more work-groups take a sequence's paths each (64
// answers of 24 drafted tokens: 4 us in a launch of their own).
template <int SPT, bool TREE>  // sequences per thread
__global__ __launch_bounds__(PT) void paged_plan_kernel(PagedPlanArgs a, int writers, int placers) {
  constexpr int S = PT * SPT;
  // of every sequence: first row, its position, items before it (per kind), workspace rows and merge
  // records before it, parts, keys of a part
  __shared__ int s_cu[S + 1], s_pos0[S], s_many[S], s_few[S], s_part[S], s_merge[S], s_parts[S], s_chunk[S];
  __shared__ int s_scan[10 * PT / 64];
  __shared__ __attribute__((aligned(16))) uint32_t s_key[PT];
  __shared__ int s_at[PT], s_items[PT];  // (one sequence per thread: their order)
  const int tid = threadIdx.x, group = a.hq / a.hkv;
  const bool narrow = a.layout.narrow;
  // Row offsets need sums of q; the split shares need, per kind (many rows, few rows), the tiles and
  // their keys, here from the lengths as they are given (cut to n_tokens one by one), which is no less
  // than what the rows make. Sums that could pass 32 bits go in pieces of 15 and 19 bits: 4096 sequences
  // times 2^19 - 1 stay below 2^31, three pieces hold 2^57 (a sequence has up to 2^23 tiles of 2^30 keys).
  int q[SPT], sum[10] = {}, sums[10];
#pragma unroll
  for (int i = 0; i < SPT; ++i) {
    const int s = tid * SPT + i;
    const bool in = s < a.n_seqs;
    const int len = in ? max(a.q_lengths[s], 0) : 0;
    const int kv = in ? min(max(a.kv_lengths[s], 0), a.max_keys) : 0;
    s_pos0[s] = kv - len;
    q[i] = min(len, a.n_tokens);
    sum[0] += q[i] & 0x7fff;
    sum[1] += q[i] >> 15;
    const int rows = q[i] * group, kind = narrow || rows <= kPagedFewRows, t = tiles_of(rows, narrow);
    const long long keys = (long long)t * kv;
    sum[2 + kind] += t;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int b = 0; b < 3; ++b) sum[4 + 3 * k + b] += k == kind ? (int)(keys >> 19 * b) & 0x7ffff : 0;
  }
  block_exclusive_sums<PT / 64>(sum, sums, s_scan);
  long long at = ((long long)sum[1] << 15) + sum[0];
  int n_rows[SPT];  // flattened rows of a sequence
#pragma unroll
  for (int i = 0; i < SPT; ++i) {
    const int first = (int)min(at, (long long)a.n_tokens);
    at += q[i];
    s_cu[tid * SPT + i] = first;
    n_rows[i] = ((int)min(at, (long long)a.n_tokens) - first) * group;
  }
  if (tid == PT - 1) s_cu[S] = (int)min(at, (long long)a.n_tokens);
  if constexpr (TREE && SPT == 1) {
    if ((int)blockIdx.x >= 2 * writers + placers) {
      __shared__ TreeLds lds;
      __syncthreads();
      const int s = blockIdx.x - 2 * writers - placers;
      tree_paths(a, lds, s_cu[s], s_cu[s + 1] - s_cu[s], s_pos0[s]);
      return;
    }
  }
  if ((int)blockIdx.x >= 2 * writers) {
    __syncthreads();
    const int rows = s_cu[a.n_seqs], first = (blockIdx.x - 2 * writers) * kPlanRowsPerGroup;
    const int end = min(first + kPlanRowsPerGroup, a.n_tokens);
    for (int n = first + tid; n < end; n += PT) {
      int seq = -1, pos = -1;
      if (n < rows) {
        seq = last_at_most(s_cu, a.n_seqs, n);
        pos = s_pos0[seq] + (n - s_cu[seq]);
      }
      a.plan[a.layout.seq + n] = seq;
      a.plan[a.layout.pos + n] = pos;
      if (TREE && seq < 0) a.tree[tree_positions(a.n_tokens) + n] = -1;
    }
    return;
  }
  // (lengths that pass the rows are cut there, which may change a tile's kind: such a step is not split)
  const bool split =
      a.max_keys > kPagedWholeKeys && ((long long)sums[1] << 15) + sums[0] <= a.n_tokens;
  int chunks[2] = {INT_MAX / 2, INT_MAX / 2};
  // parts of prompt tiles that are as many as the card has places (few-row tiles behind them fill the
  // places that shorter ones leave)
  const long long its = (long long)sums[2] * a.hkv;
  const long long many = min(max(sums[3] == 0 ? its : its / 2, (long long)kPagedManyParts / 4),
                             (long long)a.layout.many_parts);
#pragma unroll
  for (int k = 0; k < 2 && split; ++k) {
    if (sums[2 + k] == 0) continue;  // (no such tile)
    const long long items = (long long)sums[2 + k] * a.hkv;
    const long long all = k == 1         ? kPagedFewParts - max(0LL, many - kPagedManyParts)
                          : sums[3] == 0 ? a.layout.many_base
                                         : kPagedManyParts;
    const long long parts = max(all - items, k == 0 ? many : all / 4);
    const long long keys =
        ((long long)sums[6 + 3 * k] << 38) + ((long long)sums[5 + 3 * k] << 19) + sums[4 + 3 * k];
    // (at most INT_MAX / 2, which no range is longer than: such a share splits nothing; a prompt of 2^20
    // tokens, 32/8 heads, makes 2^32. Rounded up and added to a range it stays below 2^31.)
    const long long least =
        k == 1 ? kPagedFewKeys
               : min(max(quotient(keys * a.hkv, kPagedShortItems), (long long)kPagedFewKeys),
                     (long long)kPagedManyKeys);
    const long long share =
        min(max(quotient(keys * a.hkv + parts - 1, parts), least), (long long)(INT_MAX / 2));
    chunks[k] = (int)((share + kPagedChunkKeys - 1) / kPagedChunkKeys * kPagedChunkKeys);
  }
  const int aligned = 8 / (a.hkv % 8 == 0 ? 8 : a.hkv % 4 == 0 ? 4 : a.hkv % 2 == 0 ? 2 : 1);
  int x[4] = {0, 0, 0, 0}, n[4];  // items of both kinds, workspace rows, merge records
  int own[SPT][4], longest_of[SPT];
#pragma unroll
  for (int i = 0; i < SPT; ++i) {
    const int s = tid * SPT + i, rows = n_rows[i], kind = narrow || rows <= kPagedFewRows;
    const int longest = rows > 0 ? keys_of(s_pos0[s], rows, group) : 0;
    int parts = max(1, (longest + chunks[kind] - 1) / chunks[kind]);
    if (kind == 0 && parts > aligned) parts -= parts % aligned;
    const int c =
        ((longest + parts - 1) / parts + kPagedChunkKeys - 1) / kPagedChunkKeys * kPagedChunkKeys;
    if (parts > 1) parts = (longest + c - 1) / c;
    s_parts[s] = parts;
    s_chunk[s] = max(c, 1);
    const int items = tiles_of(rows, narrow) * parts * a.hkv;
    longest_of[i] = kind == 0 ? longest : 0;
    own[i][0] = kind == 0 ? items : 0;
    own[i][1] = kind == 0 ? 0 : items;
    own[i][2] = parts > 1 ? rows * parts * a.hkv : 0;
    own[i][3] = parts > 1 ? (rows + merged_rows(kind, parts) - 1) / merged_rows(kind, parts) * a.hkv : 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] += own[i][k];
  }
  block_exclusive_sums<PT / 64>(x, n, s_scan);
#pragma unroll
  for (int i = 0; i < SPT; ++i) {
    const int s = tid * SPT + i;
    s_many[s] = x[0];
    if constexpr (SPT == 1) s_items[s] = own[i][0];
    s_few[s] = x[1];
    s_part[s] = x[2];
    s_merge[s] = x[3];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] += own[i][k];
  }
  __syncthreads();
  // Prompt tiles of unequal ranges, more than the card has places and nothing behind them: the
  // sequences with the longest ranges first, so that what starts last is short (64 trees on 64 to 8192
  // tokens 78 -> 58 us for 1 us here; up to PT sequences, by counting).
  bool sorted = false;
  if constexpr (SPT == 1) {
    sorted = n[0] > kPagedManyParts && n[1] == 0 && n[2] > 0;
    if (sorted) {
      // (by the range, then by number: all different)
      const uint32_t mine = (uint32_t)min(longest_of[0], (1 << 24) - 1) << 8 | (PT - 1 - tid);
      s_key[tid] = tid < a.n_seqs ? mine : 0;
      __syncthreads();
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < a.n_seqs; j += 4) {
        const u32x4 k = *reinterpret_cast<const u32x4*>(s_key + j);
        rank += (k[0] > mine) + (k[1] > mine) + (k[2] > mine) + (k[3] > mine);
      }
      if (tid < a.n_seqs) s_at[rank] = tid;
      __syncthreads();
      int y[1] = {tid < a.n_seqs ? s_items[s_at[tid]] : 0}, all[1];
      block_exclusive_sums<PT / 64>(y, all, s_scan);
      s_many[tid] = y[0];
      __syncthreads();
    }
  }
  Item* items = reinterpret_cast<Item*>(a.plan + a.layout.items);
  Merge* merges = reinterpret_cast<Merge*>(a.plan + a.layout.merges);
  const bool merging = (int)blockIdx.x >= writers;
  const int first = (blockIdx.x - (merging ? writers : 0)) * PT + tid, step = writers * PT;
  const int n_items = (int)min((long)n[0] + n[1], (long)a.layout.max_items);
  const bool paired = n[1] == 0 && (a.hkv == 1 || a.hkv == 2 || a.hkv == 4);
  for (int i = first; i < n_items && !merging; i += step) {
    const bool many = i < n[0];
    const int* before = many ? s_many : s_few;
    int j = many ? i : i - n[0], nth = last_at_most(before, a.n_seqs, many && paired ? j & ~15 : j);
    if (many && paired) {
      if ((j | 15) < n[0] && s_parts[SPT == 1 && sorted ? s_at[nth] : nth] == 1) j = paired_tile(j, a.hkv);
      nth = last_at_most(before, a.n_seqs, j);
    }
    const int s = SPT == 1 && many && sorted ? s_at[nth] : nth;
    const int rows = (s_cu[s + 1] - s_cu[s]) * group, parts = s_parts[s], chunk = s_chunk[s];
    const int in = j - before[nth], per_tile = parts * a.hkv;
    const int tile = tiles_of(rows, narrow) - 1 - in / per_tile;
    const int head = in % a.hkv, part = in % per_tile / a.hkv;
    Item it;
    it.token0 = s_cu[s];
    it.seq = s;
    it.pos0 = s_pos0[s];
    const int each = narrow ? kPagedFewRows : kPagedTileRows;
    it.row = tile * each;
    it.row_end = min(it.row + each, rows);
    const int all = keys_of(it.pos0, it.row_end, group);
    it.key = part * chunk;
    it.key_end = parts == 1 ? all : min(it.key + chunk, all);
    it.head = head | (it.key >= all && part > 0 ? kNone : many ? kMany : kFew) << 16;
    it.part_row = parts == 1 || all <= chunk ? -1 : s_part[s] + (head * parts + part) * rows + it.row;
    it.pad[0] = it.pad[1] = it.pad[2] = 0;
    items[i] = it;
  }
  const int n_merges = (int)min((long)n[3], (long)a.layout.max_merges);
  for (int i = first; i < n_merges && merging; i += step) {
    const int s = last_at_most(s_merge, a.n_seqs, i), in = i - s_merge[s];
    const int rows = (s_cu[s + 1] - s_cu[s]) * group, parts = s_parts[s], chunk = s_chunk[s];
    const int each = merged_rows(rows <= kPagedFewRows, parts), per_head = (rows + each - 1) / each;
    const int head = in / per_head, row = in % per_head * each;
    const int all = keys_of(s_pos0[s], min((row / kPagedTileRows + 1) * kPagedTileRows, rows), group);
    Merge m;
    m.token0 = s_cu[s];
    m.head = head;
    m.row = row;
    m.rows = min(each, rows - row);
    m.part_row = s_part[s] + head * parts * rows + row;
    m.stride = rows;
    m.parts = all <= chunk ? 0 : (all + chunk - 1) / chunk;
    m.spread = each == 1;
    merges[i] = m;
  }
  if (blockIdx.x > 0) return;
  for (int s = tid; s <= a.n_seqs; s += PT) a.plan[s] = s_cu[s];
  const int rows = s_cu[a.n_seqs], n_pad = (a.n_tokens - rows + kPagedPadRows - 1) / kPagedPadRows;
  for (int i = tid; i < n_pad; i += PT) {
    Item it{};
    it.head = kPad << 16;
    it.row = rows + i * kPagedPadRows;
    it.row_end = min(it.row + kPagedPadRows, a.n_tokens);
    if (n_items + i < a.layout.max_items) items[n_items + i] = it;
  }
  if (tid == 0) {
    a.plan[a.layout.counts] = (int)min((long)(n_items + n_pad), (long)a.layout.max_items);
    a.plan[a.layout.counts + 1] = n_merges;
  }
}

// Trees of steps of more sequences than a planning work-group of one each has threads (one launch more).
__global__ __launch_bounds__(PT) void paged_tree_kernel(PagedPlanArgs a) {
  __shared__ TreeLds lds;
  const int s = blockIdx.x, first = a.plan[s];
  tree_paths(a, lds, first, a.plan[s + 1] - first, a.plan[a.layout.pos + min(first, a.n_tokens - 1)]);
}

// ------------------------------------------------------------------------------------------------
// attention
// ------------------------------------------------------------------------------------------------
constexpr int D = kHeadDim;
constexpr int GRP = 4 * D + 32;  // halfs from one group of 4 rows to the next
constexpr int TILE = 16 * GRP;   // a 64-key K or V tile, or a 32-key tile of each
template <int W>  // waves of a work-group: 4 (two work-groups per CU) or 8 (one)
struct Shape {
  static constexpr int THREADS = 64 * W;
  static constexpr int STAGES = W / 2;        // prompt tiles: 64-key stages of K and V
  static constexpr int LDS = STAGES * 2 * TILE;  // halfs: one 32-key K and V tile per wave, as much
  static constexpr int HALVES = W / 4;        // prompt tiles: waves per strip, which share a tile's keys out
  static constexpr int BLOCKS = 2 / HALVES;   // 32-key blocks per wave and tile
  static constexpr int GROUPS = 16 / W;       // row groups that a wave copies per K or V tile
};
constexpr float kRescaleLog2 = 8.f;  // many rows: the maximum moves when a tile exceeds it by 2^8

// Read offsets (halfs) inside a tile. K (A operand of S^T): row perm32(l32), chunk 2 kk + hi. V^T: row
// 8 hi + 2 (src >> 2) + e (+ 16 c), chunk 8 (grp & 1) + 2 db + (sg >> 1): registers [8 c, 8 c + 8) of
// accumulator db then hold d = 16 db + 64 c + 8 hi + 0..7 of the lane's row.
struct Offsets {
  int k[2], v[2][2];
};
__device__ inline Offsets offsets_of(int lane) {
  Offsets o;
  const int l32 = lane & 31, hi = lane >> 5, src = lane & 15, grp = lane >> 4;
  const int r = perm32(l32);
#pragma unroll
  for (int p = 0; p < 2; ++p) o.k[p] = (r >> 2) * GRP + (r & 3) * D + 8 * ((2 * p + hi) ^ (r & 3));
  const int sg = (((src & 3) & 1) << 1) | ((src & 3) >> 1);
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int rr = 8 * hi + 2 * (src >> 2) + e;
      o.v[p][e] = (rr >> 2) * GRP + (rr & 3) * D +
                  8 * (8 * (grp & 1) + ((2 * p + (sg >> 1)) ^ (rr & 3))) + 4 * (sg & 1);
    }
  return o;
}
__device__ inline u32x4 read_k(const lds_u16* kb, const Offsets& o, int kk, int b) {
  return ld128(kb + o.k[kk & 1] + 32 * (kk >> 1) + 8 * b * GRP);
}
__device__ inline u32x4 read_v(const lds_u16* vb, const Offsets& o, int i) {  // i = (b, c, db)
  const lds_u16* p = vb + (8 * (i >> 3) + 4 * ((i >> 2) & 1)) * GRP + 32 * ((i & 3) >> 1);
  const u32x2 x = ldtr(p + o.v[i & 1][0]), y = ldtr(p + o.v[i & 1][1]);
  return u32x4{x[0], x[1], y[0], y[1]};
}

// Buffer descriptors and items in scalar registers (the loads that they come from are not always).
__device__ inline int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ inline u32x4 scalar_rsrc(const void* base, long bytes) {
  u32x4 r = make_rsrc4(base, bytes);
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (uint32_t)scalar((int)r[i]);
  return r;
}

struct State {
  f32x16 o[4];
  float m, l;  // the row's running maximum (log2 units) and this half-wave's share of its sum
};
__device__ inline void start(State& st) {
#pragma unroll
  for (int db = 0; db < 4; ++db) st.o[db] = f32x16{};
  st.m = -INFINITY;
  st.l = 0.f;
}

// S^T of one tile of 32 BLOCKS keys, each K operand read 4 ahead.
template <class E, int BLOCKS>
__device__ inline void scores(const lds_u16* kb, const Offsets& o, const u32x4 (&qf)[8], f32x16 (&s)[BLOCKS]) {
  constexpr int N = 8 * BLOCKS;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) s[b] = f32x16{};
  u32x4 ka[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) ka[i] = read_k(kb, o, i / BLOCKS, i % BLOCKS);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s[i % BLOCKS] = E::mfma(ka[i & 3], qf[i / BLOCKS], s[i % BLOCKS]);
    if (i + 4 < N) ka[i & 3] = read_k(kb, o, (i + 4) / BLOCKS, (i + 4) % BLOCKS);
  }
  if constexpr (BLOCKS == 2) {
    VA_SCHED(kSchedDsRead, 4);
#pragma unroll
    for (int i = 0; i < N - 4; ++i) {
      VA_SCHED(kSchedMfma, 1);
      VA_SCHED(kSchedDsRead, 1);
    }
    VA_SCHED(kSchedMfma, 4);
  }
}

// What a row sees of a tile's keys: those up to `lim` of the tile, or, with a tree, the ones whose bits are
// set in the words of its path. Key k of the cache is new token k - pos0; earlier keys are seen by all.
struct Chain {
  int lim;
  template <int BLOCKS>
  __device__ inline void hide(f32x16 (&s)[BLOCKS], int hi) const {
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (32 * b + reg_row(j, hi) > lim) s[b][j] = -INFINITY;
  }
};
struct Path {
  const uint32_t* words;  // the row's (null: the sequence's new tokens are a chain)
  int first;              // number of the tile's first key among the new tokens
  int lim;
  // keys o to o + 31 by number (o the same in all lanes)
  __device__ inline uint32_t bits(int o) const {
    if (o <= -32) return ~0u;
    if (o < 0) return words[0] << -o | ((1u << -o) - 1);
    const int w = o >> 5;
    const uint32_t lo = w < kTreeWords ? words[w] : 0u, up = w + 1 < kTreeWords ? words[w + 1] : 0u;
    return __builtin_amdgcn_alignbit(up, lo, o & 31);
  }
  template <int BLOCKS>
  __device__ inline void hide(f32x16 (&s)[BLOCKS], int hi) const {
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      const int n = lim - 32 * b;
      const uint32_t seen = words != nullptr ? bits(first + 32 * b)
                            : n >= 31        ? ~0u
                            : n < 0          ? 0u
                                             : (2u << n) - 1;
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (!(seen >> reg_row(j, hi) & 1)) s[b][j] = -INFINITY;
    }
  }
};
// How an item's rows see its keys.
template <bool TREE>
struct Sight {
  const uint32_t* words;  // of the lane's row
  int lim, pos0, from;    // the row's last key; the cached rows; tiles that end behind `from` are masked
  __device__ Sight(const PagedAttnArgs& a, const Item& it, int tok, int lim, int first_lim)
      : words(nullptr), lim(lim), pos0(it.pos0), from(first_lim) {
    if constexpr (TREE) {
      if (scalar_count(a, it.seq) <= kTreeTokens) {
        words = reinterpret_cast<const uint32_t*>(a.tree) + (long)(it.token0 + tok) * kTreeWords;
        from = it.pos0 - 1;
      }
    }
  }
  __device__ static inline int scalar_count(const PagedAttnArgs& a, int seq) {
    return __builtin_amdgcn_readfirstlane(a.plan[seq + 1] - a.plan[seq]);
  }
  __device__ inline auto of(int key) const {  // the tile from `key` on
    if constexpr (TREE) return Path{words, key - pos0, lim - key};
    else return Chain{lim - key};
  }
};

// Mask, running maximum and sum, weights of one tile. The maximum moves when some row's tile maximum
// exceeds its own by more than 2^margin.
template <class E, int BLOCKS, class Seen>
__device__ inline void soften(f32x16 (&s)[BLOCKS], bool mask, const Seen& seen, int hi, float scale_log2,
                              float margin, State& st, u32x4 (&pf)[BLOCKS][2]) {
  if (mask) seen.hide(s, hi);
  float mt = -INFINITY;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int j = 0; j < 16; ++j) mt = fmaxf(mt, s[b][j]);
  mt = max_with_other_half(mt) * scale_log2;
  if (__builtin_amdgcn_ballot_w64(mt > st.m + margin) != 0) {
    const float m_new = fmaxf(st.m, mt);
    const float alpha = fast_exp2(st.m - (m_new == -INFINITY ? 0.f : m_new));
    st.m = m_new;
    st.l *= alpha;
#pragma unroll
    for (int db = 0; db < 4; ++db) st.o[db] *= alpha;
  }
  const float m_use = st.m == -INFINITY ? 0.f : st.m;
  float rs = 0.f;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = fast_exp2(fmaf(s[b][8 * c + e], scale_log2, -m_use));
      pf[b][c] = pack8_tr<E>(p);
#pragma unroll
      for (int w = 0; w < 4; ++w) rs = E::sum2(pf[b][c][w], rs);
    }
  st.l += rs;
}

// O^T += V^T P^T; the first four V operands are in `va`, the others are read 4 ahead.
template <class E, int BLOCKS>
__device__ inline void weigh(const lds_u16* vb, const Offsets& o, const u32x4 (&pf)[BLOCKS][2],
                             u32x4 (&va)[4], State& st) {
  constexpr int N = 8 * BLOCKS;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    st.o[i & 3] = E::mfma(va[i & 3], pf[i >> 3][(i >> 2) & 1], st.o[i & 3]);
    if (i + 4 < N) va[i & 3] = read_v(vb, o, i + 4);
  }
}

// Where the rows of one key/value head lie, and buffer descriptors of up to 16 rows of a page: built by
// scalar instructions, of which each costs the wave as much as a vector one.
struct Head {
  uint64_t k, v;  // addresses of the head's rows in page 0
  uint32_t k_stride, v_stride, mask;
  int n_pages, end;  // the range's end
  __device__ Head(const PagedAttnArgs& a, const Item& it, int head, int row_bytes = D * 2)
      : k((uint64_t)a.k + ((uint64_t)(head << a.pool.page_shift) * row_bytes)),
        v((uint64_t)a.v + ((uint64_t)(head << a.pool.page_shift) * row_bytes)),
        k_stride(a.pool.k_stride), v_stride(a.pool.v_stride), mask((1u << a.pool.page_shift) - 1),
        n_pages(a.pool.n_pages), end(it.key_end) {}
  // The page of the row at `pos`; -1 where there is none, or the range has ended.
  __device__ inline int page(const int32_t* table, int shift, int pos) const {
    const int p = pos < end ? table[pos >> shift] : -1;
    return (uint32_t)p < (uint32_t)n_pages ? p : -1;
  }
  // 8-bit pages: where the row at `pos` of this page lies (of page 0 where there is none: what is read
  // there is not used), and its power of two, as a float, from the exponent byte. (Bytes that no row was
  // written with, behind a sequence's end, may be anything: 255 would be no number.)
  __device__ inline uint64_t row8(uint64_t base, uint32_t stride, int page, int pos) const {
    return base + (uint64_t)(uint32_t)max(page, 0) * stride + ((uint32_t)pos & mask) * D;
  }
  __device__ inline uint32_t exp8(const uint8_t* base, uint32_t stride, int head, int shift, int page, int pos) const {
    return base[(uint64_t)(uint32_t)max(page, 0) * stride + ((uint32_t)(head << shift) + ((uint32_t)pos & mask))];
  }
  // The rows from `pos` on: the page's, up to 16 and up to the range's end; the others read as zeros.
  template <int ROW = D * 2>
  __device__ inline void rows(int page, int pos, u32x4& rk, u32x4& rv) const {
    const uint32_t in = ((uint32_t)pos & mask) * ROW, p = (uint32_t)max(page, 0);
    const uint32_t bytes = page < 0 ? 0 : (uint32_t)min(end - pos, 16) * ROW;
    const uint64_t ak = k + (uint64_t)p * k_stride + in, av = v + (uint64_t)p * v_stride + in;
    rk = u32x4{(uint32_t)scalar((int)ak), (uint32_t)scalar((int)(ak >> 32)) & 0xffffu,
               (uint32_t)scalar((int)bytes), 0x00020000u};
    rv = u32x4{(uint32_t)scalar((int)av), (uint32_t)scalar((int)(av >> 32)) & 0xffffu,
               (uint32_t)scalar((int)bytes), 0x00020000u};
  }
};

// An item's rows: row r of the sequence is token r / group, query head r % group of the group.
// Divisions of small numbers by the group: exact in fp32 (rows below 2^13, half a unit to spare).
struct RowMap {
  int token, rest, group;  // of the item's first row
  float inv;
  __device__ RowMap(int row, int g) : token(row / g), rest(row % g), group(g), inv(1.f / (float)g) {}
  __device__ inline void at(int r, int& tok, int& h) const {
    const int x = r + rest, t = (int)(((float)x + 0.5f) * inv);
    tok = token + t;
    h = x - t * group;
  }
};

// The waves of a few-row tile meet.
template <class E, int W>
__device__ inline void join_waves(const PagedAttnArgs& a, const Item& it, const RowMap& map, int head,
                                  int n_rows, char* smem_raw, const State& st) {
  constexpr int NW = W;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5, group = map.group;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // fp32 rows of 132 words per wave, then their maxima and sums
  constexpr int LT = D + 4;
  float* xo = reinterpret_cast<float*>(smem_raw);
  float* xs = xo + NW * 32 * LT;
  static_assert((NW * 32 * LT + NW * 32 * 2) * 4 <= Shape<W>::LDS * 2, "the waves' rows fit in LDS");
  __syncthreads();  // every wave has read its tiles
  const float l_row = sum_with_other_half(st.l);
  if (l32 < n_rows) {
    float* row = xo + (wave * 32 + l32) * LT;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float* p = row + 16 * db + 64 * c + 8 * hi;
        *reinterpret_cast<f32x4*>(p) = f32x4{st.o[db][8 * c], st.o[db][8 * c + 1],
                                             st.o[db][8 * c + 2], st.o[db][8 * c + 3]};
        *reinterpret_cast<f32x4*>(p + 4) = f32x4{st.o[db][8 * c + 4], st.o[db][8 * c + 5],
                                                 st.o[db][8 * c + 6], st.o[db][8 * c + 7]};
      }
    if (hi == 0) {
      xs[2 * (wave * 32 + l32)] = st.m;
      xs[2 * (wave * 32 + l32) + 1] = l_row;
    }
  }
  __syncthreads();
  constexpr int PER = 32 * D / Shape<W>::THREADS;  // elements of a row per thread
  const int r = tid / (D / PER), d0 = PER * (tid % (D / PER));
  if (r >= n_rows) return;
  float m[NW], l = 0.f, m_all = -INFINITY;
#pragma unroll
  for (int w = 0; w < NW; ++w) m_all = fmaxf(m_all, m[w] = xs[2 * (w * 32 + r)]);
  const float m_use = m_all == -INFINITY ? 0.f : m_all;
  f32x4 o[PER / 4] = {};
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const float c = fast_exp2(m[w] - m_use);
    l += c * xs[2 * (w * 32 + r) + 1];
#pragma unroll
    for (int e = 0; e < PER / 4; ++e)
      o[e] += c * *reinterpret_cast<const f32x4*>(xo + (w * 32 + r) * LT + d0 + 4 * e);
  }
  if (it.part_row >= 0) {
    const long row = it.part_row + r;
#pragma unroll
    for (int e = 0; e < PER / 4; ++e)
      *reinterpret_cast<f32x4*>(a.workspace + row * D + d0 + 4 * e) = o[e];
    if (d0 == 0)
      *reinterpret_cast<f32x2*>(a.workspace + a.layout.max_part_rows * D + 2 * row) = f32x2{m_all, l};
    return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  int tok, h;
  map.at(r, tok, h);
  uint16_t* out = (uint16_t*)a.out + ((long)(it.token0 + tok) * a.hq + head * group + h) * D + d0;
#pragma unroll
  for (int e = 0; e < PER / 8; ++e)
    gstore16(out + 8 * e, pack8<E>(o[2 * e][0] * inv, o[2 * e][1] * inv, o[2 * e][2] * inv,
                                   o[2 * e][3] * inv, o[2 * e + 1][0] * inv, o[2 * e + 1][1] * inv,
                                   o[2 * e + 1][2] * inv, o[2 * e + 1][3] * inv));
}

template <class E, int W, bool TREE>
__device__ inline void few_rows(const PagedAttnArgs& a, const Item& it, lds_u16* smem, char* smem_raw) {
  constexpr int NW = W;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = it.head & 0xffff, group = a.hq / a.hkv, n_rows = it.row_end - it.row;
  const float scale_log2 = a.scale * kLog2e;
  const RowMap map(it.row, group);
  const Offsets off = offsets_of(lane);
  const int32_t* table = a.pool.table + (long)it.seq * a.pool.table_width;
  const int n_tiles = (it.key_end - it.key + 31) >> 5;

  // This wave's rows: all waves hold the same queries.
  u32x4 qf[8];
  int my_lim = -1, my_tok = map.token;
  {
    int tok, h;
    map.at(l32, tok, h);
    if (l32 < n_rows) my_lim = it.pos0 + tok, my_tok = tok;
    const uint16_t* q = (const uint16_t*)a.q + ((long)(it.token0 + tok) * a.hq + head * group + h) * D;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      qf[kk] = u32x4{0u, 0u, 0u, 0u};
      if (l32 < n_rows) qf[kk] = gload16(q + 16 * kk + 8 * hi);
    }
  }
  // Page numbers of this wave's next 32 tiles, two per tile (16 rows each): lane 2 i + h holds half h.
  const Head rows(a, it, head);
  auto load_pages = [&](int t) {
    return rows.page(table, a.pool.page_shift, it.key + 32 * (t + NW * (lane >> 1)) + 16 * (lane & 1));
  };
  const uint32_t kl = lds_addr(smem + wave * (TILE)), vl = lds_addr(smem + wave * TILE + TILE / 2);
  const lds_u16* kb = smem + wave * TILE;
  const lds_u16* vb = kb + TILE / 2;
  const int c_row = lane >> 4, coff = (c_row * D + 8 * ((lane & 15) ^ c_row)) * 2;
  auto copy = [&](const u32x4 (&from)[2], uint32_t dst) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        dma16_opaque(from[h], dst + (4 * h + j) * GRP * 2, coff + j * 4 * D * 2);
  };
  State st;
  start(st);
  int pages = 0, i = 0;  // i: this wave's tiles so far
  u32x4 rk[2], rv[2];
  auto locate = [&](int t, int n) {  // this wave's n-th tile, tile t of the item
    if ((n & 31) == 0) pages = load_pages(t);
#pragma unroll
    for (int h = 0; h < 2; ++h)
      rows.rows(__builtin_amdgcn_readlane(pages, 2 * (n & 31) + h), it.key + 32 * t + 16 * h, rk[h], rv[h]);
  };
  if (wave < n_tiles) {
    locate(wave, 0);
    copy(rk, kl);
    copy(rv, vl);
  }
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) settle(qf[kk]);
  const Sight<TREE> sight(a, it, my_tok, my_lim, it.pos0 + map.token);  // (the first row's last key)
  for (int t = wave; t < n_tiles; t += NW, ++i) {
    const bool more = t + NW < n_tiles;
    asm volatile("s_waitcnt vmcnt(8)" ::: "memory");  // this tile's K; its V (8 copies) may be in flight
    f32x16 s[1];
    scores<E, 1>(kb, off, qf, s);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K read: its place is free
    if (more) {
      locate(t + NW, i + 1);
      copy(rk, kl);
    }
    const int kv0 = it.key + 32 * t;
    u32x4 pf[1][2];
    soften<E, 1>(s, kv0 + 31 > sight.from, sight.of(kv0), hi, scale_log2, 0.f, st, pf);
    if (more) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");  // V; the next K in flight
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    u32x4 va[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) va[j] = read_v(vb, off, j);
    weigh<E, 1>(vb, off, pf, va, st);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // V read
    if (more) copy(rv, vl);
  }

  join_waves<E, W>(a, it, map, head, n_rows, smem_raw, st);
}

// 8-bit pages. Keys: lane (row, hi) of the operand loads its row's 16-byte pieces 2 i + hi, i = 0..3; piece
// i serves two products, whose k slots 8 hi + 0..7 are then numbers 16 (2 i + hi) + 8 half + 0..7 of a row,
// in the queries too. Values: 16 numbers of row 8 j + lane / 8 per lane and load, turned into 16-bit
// rows of the wave's own LDS tile. A tile's loads are issued when the registers of the one before are
// free: keys after its products, values after their rows are in LDS, so that 8 KB per wave are in
// flight but for the conversions.
template <class E>
__device__ inline u32x4 numbers8(uint32_t lo, uint32_t hi, float power) {
  return u32x4{E::from_e4m3(lo, power, false), E::from_e4m3(lo, power, true),
               E::from_e4m3(hi, power, false), E::from_e4m3(hi, power, true)};
}
__device__ inline float power_of(uint32_t byte) {
  return __builtin_bit_cast(float, min(byte, 254u) << 23);
}
__device__ inline float from_lane(int lane, float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_ds_bpermute(4 * lane, __builtin_bit_cast(int, x)));
}

template <class E, int W, bool TREE>
__device__ inline void few_rows8(const PagedAttnArgs& a, const Item& it, lds_u16* smem, char* smem_raw) {
  constexpr int NW = W;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = it.head & 0xffff, group = a.hq / a.hkv, n_rows = it.row_end - it.row;
  const int shift = a.pool.page_shift;
  const float scale_log2 = a.scale * kLog2e;
  const RowMap map(it.row, group);
  const Offsets off = offsets_of(lane);
  const int32_t* table = a.pool.table + (long)it.seq * a.pool.table_width;
  const int n_tiles = (it.key_end - it.key + 31) >> 5;

  u32x4 qf[8];
  int my_lim = -1, my_tok = map.token;
  {
    int tok, h;
    map.at(l32, tok, h);
    if (l32 < n_rows) my_lim = it.pos0 + tok, my_tok = tok;
    const uint16_t* q = (const uint16_t*)a.q + ((long)(it.token0 + tok) * a.hq + head * group + h) * D;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      qf[i] = u32x4{0u, 0u, 0u, 0u};
      if (l32 < n_rows) qf[i] = gload16(q + 16 * (2 * (i >> 1) + hi) + 8 * (i & 1));
    }
  }
  const Head rows(a, it, head, D);
  int pages = 0;
  auto load_pages = [&](int t) {
    return rows.page(table, shift, it.key + 32 * (t + NW * (lane >> 1)) + 16 * (lane & 1));
  };
  const int k_row = perm32(l32);
  lds_u16* const vt = smem + wave * (TILE / 2);
  // this lane's rows of the value tile: row 8 j + lane / 8, numbers 16 m .. 16 m + 15
  const int v_row = lane >> 3, m = lane & 7;
  const Sight<TREE> sight(a, it, my_tok, my_lim, it.pos0 + map.token);
  State st;
  start(st);

  u32x4 kr[4], vr[4];
  uint32_t ke = 0, ve = 0;
  int pg[2] = {-1, -1};  // pages of the tile whose keys are in flight, and of the one whose values are
  auto locate = [&](int t, int n) {  // this wave's n-th tile, tile t of the item
    if ((n & 31) == 0) pages = load_pages(t);
#pragma unroll
    for (int h = 0; h < 2; ++h) pg[h] = __builtin_amdgcn_readlane(pages, 2 * (n & 31) + h);
  };
  auto fetch_keys = [&](int t) {
    const int pos = it.key + 32 * t;
    const uint64_t p0 = rows.row8(rows.k, rows.k_stride, pg[0], pos);
    const uint64_t p1 = rows.row8(rows.k, rows.k_stride, pg[1], pos + 16);
    // (as device memory: loads of any memory return out of order with LDS reads, and all are waited for)
    typedef const __attribute__((address_space(1))) u32x4 device_u32x4;
    device_u32x4* p = (device_u32x4*)((k_row < 16 ? p0 : p1) + (uint64_t)((k_row & 15) * D + 16 * hi));
#pragma unroll
    for (int i = 0; i < 4; ++i) kr[i] = p[2 * i];
    ke = rows.exp8(a.pool.k_exp, a.pool.k_exp_stride, head, shift, k_row < 16 ? pg[0] : pg[1], pos + k_row);
  };
  auto fetch_values = [&](int t) {
    const int pos = it.key + 32 * t;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 rk, rv;
      rows.rows<D>(pg[h], pos + 16 * h, rk, rv);
      const brsrc r = __builtin_amdgcn_make_buffer_rsrc(
          (void*)((uint64_t)rv[0] | (uint64_t)rv[1] << 32), (short)0, (int)rv[2], 0x00020000);
#pragma unroll
      for (int j = 0; j < 2; ++j) vr[2 * h + j] = bload16(r, 16 * lane + 1024 * j);
    }
    ve = rows.exp8(a.pool.v_exp, a.pool.v_exp_stride, head, shift, l32 < 16 ? pg[0] : pg[1], pos + l32);
  };
  int i = 0;  // this wave's tiles so far
  if (wave < n_tiles) {
    locate(wave, 0);
    fetch_keys(wave);
    fetch_values(wave);
  }
  for (int t = wave; t < n_tiles; t += NW, ++i) {
    const int kv0 = it.key + 32 * t;
    f32x16 s[1] = {f32x16{}};
    {
      const float power = power_of(ke);
      if ((pg[0] | pg[1]) < 0) {  // (rows that no page holds are zeros; those behind the end are not seen)
        const bool gone = (k_row < 16 ? pg[0] : pg[1]) < 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) kr[j] = gone ? u32x4{0u, 0u, 0u, 0u} : kr[j];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        s[0] = E::mfma(numbers8<E>(kr[j >> 1][2 * (j & 1)], kr[j >> 1][2 * (j & 1) + 1], power), qf[j], s[0]);
    }
    // (behind the last tile too, where no page is: loads under a condition would all be waited for
    // before the next tile's first use; with keys loaded as device memory, eight answers of 700 11.6 ->
    // 11.0 us, four of 512 9.3 -> 9.0)
    locate(t + NW, i + 1);
    fetch_keys(t + NW);
    u32x4 pf[1][2];
    soften<E, 1>(s, kv0 + 31 > sight.from, sight.of(kv0), hi, scale_log2, 0.f, st, pf);
    const float power = power_of(ve);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = 8 * j + v_row;
      const float f = from_lane(r, power);
      lds_u16* row = vt + (r >> 2) * GRP + (r & 3) * D;
#pragma unroll
      for (int c = 0; c < 2; ++c)
        st128(row + 8 * ((2 * m + c) ^ (r & 3)), numbers8<E>(vr[j][2 * c], vr[j][2 * c + 1], f));
    }
    fetch_values(t + NW);
    u32x4 va[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) va[j] = read_v(vt, off, j);
    weigh<E, 1>(vt, off, pf, va, st);
  }
  join_waves<E, W>(a, it, map, head, n_rows, smem_raw, st);
}

template <class E, int W, bool P8, bool TREE>
__device__ inline void many_rows(const PagedAttnArgs& a, const Item& it, lds_u16* smem) {
  using S = Shape<W>;
  constexpr int KEYS = 64, STAGE = 2 * TILE, STAGES = S::STAGES, BLOCKS = S::BLOCKS, GROUPS = S::GROUPS;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hi = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), strip = wave & 3, half = wave >> 2;
  const int head = it.head & 0xffff, group = a.hq / a.hkv, n_rows = it.row_end - it.row;
  const float scale_log2 = a.scale * kLog2e;
  const RowMap map(it.row, group);
  const Offsets off = offsets_of(lane);
  const int32_t* table = a.pool.table + (long)it.seq * a.pool.table_width;
  const int n_tiles = (it.key_end - it.key + KEYS - 1) / KEYS;
  const int c_row = lane >> 4;

  // Copies, in tile order: wave w moves 4 GROUPS rows of K and of V, which lie in one page; the page
  // numbers of its next 64 tiles are in its lanes.
  const Head rows(a, it, head, P8 ? D : D * 2);
  int pages = 0, tc = 0;
  // 8-bit pages: a wave fetches 4 GROUPS rows of K and of V into registers (16 numbers of row 8 j +
  // lane / 8 per lane and load; the powers of K rows in lanes 0 to 15, of V rows in lanes 16 to 31) and
  // places them as 16-bit rows in their stage.
  constexpr int PIECES = 4 * GROUPS / 8;
  u32x4 kr[PIECES], vr[PIECES];
  uint32_t ex = 0;
  int tp = 0;  // tiles placed
  auto fetch_next = [&]() {
    const int pos = it.key + 4 * GROUPS * wave + KEYS * tc, shift = a.pool.page_shift;
    if ((tc & 63) == 0) pages = rows.page(table, shift, pos + KEYS * lane);
    const int page = __builtin_amdgcn_readlane(pages, tc & 63);
    u32x4 r[2];
    rows.template rows<D>(page, pos, r[0], r[1]);
    brsrc b[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      b[i] = __builtin_amdgcn_make_buffer_rsrc((void*)((uint64_t)r[i][0] | (uint64_t)r[i][1] << 32), (short)0,
                                               (int)r[i][2], 0x00020000);
#pragma unroll
    for (int j = 0; j < PIECES; ++j) kr[j] = bload16(b[0], 16 * lane + 1024 * j);
#pragma unroll
    for (int j = 0; j < PIECES; ++j) vr[j] = bload16(b[1], 16 * lane + 1024 * j);
    const bool is_v = lane & 16;
    ex = rows.exp8(is_v ? a.pool.v_exp : a.pool.k_exp, is_v ? a.pool.v_exp_stride : a.pool.k_exp_stride, head,
                   shift, page, pos + (lane & (4 * GROUPS - 1)));
    ++tc;
  };
  auto place_next = [&]() {
    const float power = power_of(ex);
    lds_u16* const stage = smem + (tp & (STAGES - 1)) * STAGE + GROUPS * wave * GRP;
    const int m = lane & 7;
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int r = 8 * j + (lane >> 3);
      const float fk = from_lane(r, power), fv = from_lane(16 + r, power);
      lds_u16* row = stage + (r >> 2) * GRP + (r & 3) * D;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        st128(row + 8 * ((2 * m + c) ^ (r & 3)), numbers8<E>(kr[j][2 * c], kr[j][2 * c + 1], fk));
        st128(row + TILE + 8 * ((2 * m + c) ^ (r & 3)), numbers8<E>(vr[j][2 * c], vr[j][2 * c + 1], fv));
      }
    }
    ++tp;
  };
  const int coff = (c_row * D + 8 * ((lane & 15) ^ c_row)) * 2;
  auto copy_next = [&]() {
    const int pos = it.key + 4 * GROUPS * wave + KEYS * tc;
    if ((tc & 63) == 0) pages = rows.page(table, a.pool.page_shift, pos + KEYS * lane);
    u32x4 rk, rv;
    rows.rows(__builtin_amdgcn_readlane(pages, tc & 63), pos, rk, rv);
    const uint32_t dst = lds_addr(smem + (tc & (STAGES - 1)) * STAGE + GROUPS * wave * GRP);
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) dma16_opaque(rk, dst + j * GRP * 2, coff + j * 4 * D * 2);
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) dma16_opaque(rv, dst + (TILE + j * GRP) * 2, coff + j * 4 * D * 2);
    ++tc;
  };

  // Q from stage 1 on (32 row groups), tile 0 into stage 0; every lane reads its row.
  const long q0 = ((long)(it.token0 + map.token) * a.hq + head * group) * D;  // the first row's token
  {
    const long span = (long)((map.rest + n_rows - 1) / group * a.hq + group) * D * 2;
    const u32x4 rq = scalar_rsrc((const uint16_t*)a.q + q0, span);
#pragma unroll
    for (int j = 0; j < 32 / W; ++j) {
      const int g = 32 / W * wave + j, r = 4 * g + c_row;
      int tok, h;
      map.at(r, tok, h);
      const int o = (((tok - map.token) * a.hq + h) * D + 8 * ((lane & 15) ^ c_row)) * 2;
      dma16_opaque(rq, lds_addr(smem + STAGE + g * GRP), r < n_rows ? o : 0x7fffff00);
    }
  }
  if constexpr (P8) {
    if (n_tiles > 0) {
      fetch_next();
      place_next();
    }
  } else {
    if (n_tiles > 0) copy_next();
  }
  wait_vmcnt<0>();
  __syncthreads();
  u32x4 qf[8];
  {
    const lds_u16* qt = smem + STAGE + (8 * strip + (l32 >> 2)) * GRP + (l32 & 3) * D;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk)
      qf[kk] = ld128(qt + 8 * ((2 * (kk & 1) + hi) ^ (l32 & 3)) + 32 * (kk >> 1));
  }
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) settle(qf[kk]);
  __syncthreads();  // every wave holds its rows before the second stage is written
  if constexpr (P8) {
    if (1 < n_tiles) fetch_next();
  } else {
#pragma unroll
    for (int t = 1; t < STAGES - 1; ++t)
      if (t < n_tiles) copy_next();
  }

  int my_tok, my_h;
  map.at(32 * strip + l32, my_tok, my_h);
  const int my_lim = it.pos0 + my_tok;
  const int left = n_rows - 32 * strip;  // rows of this strip
  const int first_lim = __builtin_amdgcn_readfirstlane(my_lim);
  const int last_lim = __builtin_amdgcn_readlane(my_lim, max(0, min(31, left - 1)));
  const Sight<TREE> sight(a, it, l32 < left ? my_tok : map.token, my_lim, first_lim);
  const int key0 = it.key + 32 * BLOCKS * half;  // this wave's keys of the first tile
  const int n_live = left <= 0 || last_lim < key0 ? 0 : min((last_lim - key0) / KEYS + 1, n_tiles);
  State st;
  start(st);
  // This wave's copies of tile t + 1 have landed; those of the tiles behind it stay in flight.
  auto next = [&](int t) {
    if constexpr (P8) {
    } else if (t + STAGES - 1 < n_tiles) wait_vmcnt<(STAGES - 2) * 2 * GROUPS>();
    else wait_vmcnt<0>();
    __syncthreads();
  };
  // While tile t is worked on: the copies of the tile STAGES - 1 behind it begin, or (8-bit) tile t + 1 is
  // placed, in the stage that no wave has read since a barrier, and tile t + 2 fetched.
  auto advance = [&](int t) {
    if constexpr (P8) {
      if (t + 1 < n_tiles) place_next();
      if (t + 2 < n_tiles) fetch_next();
    } else {
      if (t + STAGES - 1 < n_tiles) copy_next();
    }
  };
  int t = 0;
  for (; t < n_live; ++t) {
    const lds_u16* kb = smem + (t & (STAGES - 1)) * STAGE + 8 * BLOCKS * half * GRP;
    f32x16 s[BLOCKS];
    // (the products first where two waves of a SIMD want to issue: four chunks of 2048 tokens, 28/4
    // heads 635 -> 618 us; nothing where a wave has its SIMD mostly to itself)
    __builtin_amdgcn_s_setprio(1);
    scores<E, BLOCKS>(kb, off, qf, s);
    __builtin_amdgcn_s_setprio(0);
    advance(t);
    u32x4 va[4], pf[BLOCKS][2];
#pragma unroll
    for (int j = 0; j < 4; ++j) va[j] = read_v(kb + TILE, off, j);
    const int kv0 = key0 + KEYS * t;
    soften<E, BLOCKS>(s, kv0 + 32 * BLOCKS - 1 > sight.from, sight.of(kv0), hi, scale_log2,
                      kRescaleLog2, st, pf);
    __builtin_amdgcn_s_setprio(1);
    weigh<E, BLOCKS>(kb + TILE, off, pf, va, st);
    __builtin_amdgcn_s_setprio(0);
    next(t);
  }
  for (; t < n_tiles; ++t) {  // past this strip's keys the wave only copies
    advance(t);
    next(t);
  }

  // (The last barrier has passed and every copy has landed: the LDS is free.) Two waves of a strip meet:
  // the second hands its rows over, in the accumulators' order.
  if constexpr (S::HALVES == 2) {
    lds_f32x4* xo = (lds_f32x4*)smem;
    lds_f32x4* xs = xo + 4 * 16 * 64;
    static_assert((4 * 16 + 4) * 64 * 16 + 4 * 32 * (8 * 16 + 8) * 2 <= S::LDS * 2,
                  "the rows and the row tiles fit in LDS");
    if (half == 1) {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        xo[(16 * strip + k) * 64 + lane] =
            f32x4{st.o[k >> 2][4 * (k & 3)], st.o[k >> 2][4 * (k & 3) + 1],
                  st.o[k >> 2][4 * (k & 3) + 2], st.o[k >> 2][4 * (k & 3) + 3]};
      xs[64 * strip + lane] = f32x4{st.m, st.l, 0.f, 0.f};
    }
    __syncthreads();
    if (half == 1) return;
    const f32x4 ml = xs[64 * strip + lane];
    const float m = fmaxf(st.m, ml[0]), m_use = m == -INFINITY ? 0.f : m;
    const float ca = fast_exp2(st.m - m_use), cb = fast_exp2(ml[0] - m_use);
    st.m = m;
    st.l = st.l * ca + ml[1] * cb;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const f32x4 y = xo[(16 * strip + k) * 64 + lane];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float& x = reinterpret_cast<float(&)[16]>(st.o[k >> 2])[4 * (k & 3) + e];
        x = x * ca + y[e] * cb;
      }
    }
  }
  const float l_row = sum_with_other_half(st.l);
  if (it.part_row >= 0) {
    if (l32 >= left) return;
    const long row = it.part_row + 32 * strip + l32;
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        f32x4* p = reinterpret_cast<f32x4*>(a.workspace + row * D + 16 * db + 64 * c + 8 * hi);
        // (non-temporal: written back while the kernel runs instead of at its end, 26.2 -> 24.1 us at
        // 512 new tokens on 1536, 12/2 heads)
        __builtin_nontemporal_store(f32x4{st.o[db][8 * c], st.o[db][8 * c + 1], st.o[db][8 * c + 2],
                                          st.o[db][8 * c + 3]}, p);
        __builtin_nontemporal_store(f32x4{st.o[db][8 * c + 4], st.o[db][8 * c + 5],
                                          st.o[db][8 * c + 6], st.o[db][8 * c + 7]}, p + 1);
      }
    if (hi == 0)
      *reinterpret_cast<f32x2*>(a.workspace + a.layout.max_part_rows * D + 2 * row) = f32x2{st.m, l_row};
    return;
  }
  const float inv = l_row == 0.f ? 0.f : 1.f / l_row;
  u32x4 w[8];  // chunk db + 4 c: d = 16 db + 64 c + 8 hi + 0..7 of the lane's row
#pragma unroll
  for (int db = 0; db < 4; ++db)
#pragma unroll
    for (int c = 0; c < 2; ++c)
      w[db + 4 * c] = pack8<E>(st.o[db][8 * c] * inv, st.o[db][8 * c + 1] * inv,
                               st.o[db][8 * c + 2] * inv, st.o[db][8 * c + 3] * inv,
                               st.o[db][8 * c + 4] * inv, st.o[db][8 * c + 5] * inv,
                               st.o[db][8 * c + 6] * inv, st.o[db][8 * c + 7] * inv);
  constexpr int ROWS = 32 * (8 * 16 + 8);  // a strip's row tile, behind what the halves hand over
  static_assert(4 * ROWS <= S::LDS, "row tiles fit in LDS");
  store_rows32<16>(smem + (S::HALVES == 2 ? (4 * 16 + 4) * 64 * 8 : 0) + strip * ROWS, w, lane,
                   [&](int r) {
                     int tok, h;
                     map.at(32 * strip + r, tok, h);
                     return (uint16_t*)a.out + ((long)(it.token0 + tok) * a.hq + head * group + h) * D;
                   },
                   left);
}

// Whether an entry of the list lies inside the call's rows, sequences, keys and workspace: a list that was
// made for other sizes computes nothing useful, but reads and writes nothing out of bounds. (Where a row
// stands, pos0, only moves its mask.)
__device__ inline bool inside(const PagedAttnArgs& a, const Item& it, int kind) {
  const int rows = it.row_end - it.row;
  if (it.row < 0 || it.row_end < 0 || rows <= 0) return false;
  if (kind == kPad) return rows <= kPagedPadRows && it.row_end <= a.n_tokens;
  const int group = a.hq / a.hkv;
  return rows <= (kind == kMany ? kPagedTileRows : kPagedFewRows) && it.token0 >= 0 &&
         (long)it.token0 * group + it.row_end <= (long)a.n_tokens * group && it.seq >= 0 &&
         it.seq < a.n_seqs && (it.head & 0xffff) < a.hkv && it.key >= 0 && it.key % kPagedChunkKeys == 0 &&
         it.key_end >= 0 && it.key_end <= a.pool.table_width << a.pool.page_shift &&
         (it.part_row < 0 || (long)it.part_row + rows <= a.layout.max_part_rows);
}
// (A sequence's parts lie at least the record's rows apart, which with the workspace bounds their number.)
__device__ inline bool inside(const PagedAttnArgs& a, const Merge& m) {
  const int group = a.hq / a.hkv;
  return m.rows > 0 && m.rows <= 8 && m.row >= 0 && m.token0 >= 0 && m.head >= 0 && m.head < a.hkv &&
         (long)m.token0 * group + m.row + m.rows <= (long)a.n_tokens * group && m.parts > 1 &&
         m.stride >= m.rows && m.part_row >= 0 &&
         m.part_row + (m.parts - 1) * (long)m.stride + m.rows <= a.layout.max_part_rows;
}

template <class E, int W, bool P8 = false, bool TREE = false>
__global__ __launch_bounds__(Shape<W>::THREADS, 2) void paged_attn_kernel(PagedAttnArgs a) {
  __shared__ __attribute__((aligned(16))) uint16_t smem_raw[Shape<W>::LDS];
  lds_u16* smem = (lds_u16*)smem_raw;
  const int n_items = a.plan[a.layout.counts];
  const Item* const p = reinterpret_cast<const Item*>(a.plan + a.layout.items) + blockIdx.x;
  const Item it{scalar(p->token0), scalar(p->seq), scalar(p->pos0), scalar(p->head), scalar(p->row),
                scalar(p->row_end), scalar(p->key), scalar(p->key_end), scalar(p->part_row), {}};
  // (the list has room for max_items: the item's words are in flight beside the count)
  if ((int)blockIdx.x >= scalar(n_items)) return;
  const int kind = it.head >> 16;
  if (!inside(a, it, kind)) return;  // (the same in all threads)
  if (kind == kMany) {
    many_rows<E, W, P8, TREE>(a, it, smem);
  } else if (kind == kFew) {
    if constexpr (P8) few_rows8<E, W, TREE>(a, it, smem, (char*)smem_raw);
    else few_rows<E, W, TREE>(a, it, smem, (char*)smem_raw);
  } else if (kind == kPad) {
    u32x4* out = (u32x4*)a.out + (long)it.row * a.hq * (D / 8);
    const int chunks = (it.row_end - it.row) * a.hq * (D / 8);
    for (int i = threadIdx.x; i < chunks; i += Shape<W>::THREADS) out[i] = u32x4{0u, 0u, 0u, 0u};
  }
}

// Parts of split key ranges: a record of 8 rows has 32 lanes (4 elements each) per row, one of a single
// row and many parts shares the parts out to the 8 groups of 32 lanes.
struct Sum {
  float m, l;
  f32x4 o;
};
// Adds N parts of one row, `step` parts apart (the first `count` of them exist), all loads at once.
template <int N>
__device__ inline void add_parts(const float* o, const float* ml, long row, long step, int count, int d0,
                                 Sum& sum) {
  f32x2 x[N];
  f32x4 y[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const long r = row + min(e, count - 1) * step;
    x[e] = *reinterpret_cast<const f32x2*>(ml + 2 * r);
    y[e] = *reinterpret_cast<const f32x4*>(o + r * D + d0);
  }
  float m = sum.m;
#pragma unroll
  for (int e = 0; e < N; ++e) m = fmaxf(m, x[e][0]);
  const float m_use = m == -INFINITY ? 0.f : m, alpha = fast_exp2(sum.m - m_use);
  sum.m = m;
  sum.l *= alpha;
  sum.o *= alpha;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float c = e < count ? fast_exp2(x[e][0] - m_use) : 0.f;
    sum.l = fmaf(c, x[e][1], sum.l);
    if (c != 0.f) sum.o += c * y[e];
  }
}

constexpr int kMergeGroups = 2048;
template <class E>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedAttnArgs a) {
  __shared__ f32x4 s_o[8][32];
  __shared__ float s_m[8], s_l[8];
  const int n = min(a.plan[a.layout.counts + 1], (int)a.layout.max_merges);
  const Merge* merges = reinterpret_cast<const Merge*>(a.plan + a.layout.merges);
  const float* o = a.workspace;
  const float* ml = a.workspace + a.layout.max_part_rows * D;
  const int g = threadIdx.x >> 5, d0 = 4 * (threadIdx.x & 31), group = a.hq / a.hkv;
  Merge mg = merges[blockIdx.x];  // (there is room for every work-group's first record)
  for (int i = blockIdx.x; i < n; i += gridDim.x) {
    if (i != (int)blockIdx.x) mg = merges[i];
    if (!inside(a, mg)) continue;  // (the same in all threads)
    const bool spread = mg.spread != 0;
    const int r = spread ? 0 : g;
    const long row = mg.part_row + r;
    Sum sum{-INFINITY, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}};
    if (spread) {
      for (int p = g; p < mg.parts; p += 64)
        add_parts<8>(o, ml, row + (long)p * mg.stride, 8L * mg.stride,
                     min(8, (mg.parts - p + 7) / 8), d0, sum);
    } else if (g < mg.rows) {
      if (mg.parts <= 2) add_parts<2>(o, ml, row, mg.stride, mg.parts, d0, sum);
      else if (mg.parts <= 4) add_parts<4>(o, ml, row, mg.stride, mg.parts, d0, sum);
      else
        for (int p = 0; p < mg.parts; p += 8)
          add_parts<8>(o, ml, row + (long)p * mg.stride, mg.stride, min(8, mg.parts - p), d0, sum);
    }
    if (spread) {
      s_o[g][threadIdx.x & 31] = sum.o;
      if (d0 == 0) {
        s_m[g] = sum.m;
        s_l[g] = sum.l;
      }
      __syncthreads();
      if (g == 0) {
        float m_all = -INFINITY;
#pragma unroll
        for (int w = 0; w < 8; ++w) m_all = fmaxf(m_all, s_m[w]);
        const float m_use = m_all == -INFINITY ? 0.f : m_all;
        sum = Sum{m_all, 0.f, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          const float c = fast_exp2(s_m[w] - m_use);
          sum.l = fmaf(c, s_l[w], sum.l);
          sum.o += c * s_o[w][threadIdx.x & 31];
        }
      }
      __syncthreads();
    }
    if (spread ? g == 0 : g < mg.rows) {
      const int row_in = mg.row + r, tok = row_in / group, h = row_in % group;
      const float inv = sum.l == 0.f ? 0.f : 1.f / sum.l;
      uint16_t* out = (uint16_t*)a.out + ((long)(mg.token0 + tok) * a.hq + mg.head * group + h) * D + d0;
      __builtin_nontemporal_store(
          u32x2{pack2<E>(sum.o[0] * inv, sum.o[1] * inv), pack2<E>(sum.o[2] * inv, sum.o[3] * inv)},
          reinterpret_cast<u32x2*>(out));
    }
  }
}

// A pool without pages: every key and value is zero, and so is every row.
__global__ __launch_bounds__(256) void paged_zero_kernel(u32x4* out, long chunks) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i < chunks) out[i] = u32x4{0u, 0u, 0u, 0u};
}

template <class E, bool P8, bool TREE>
hipError_t launch_attention(const PagedAttnArgs& a) {
  if (P8 && a.pool.n_pages == 0) {
    const long chunks = (long)a.n_tokens * a.hq * (D / 8);
    hipLaunchKernelGGL(paged_zero_kernel, dim3((unsigned)((chunks + 255) / 256)), dim3(256), 0, a.stream,
                       (u32x4*)a.out, chunks);
    return hipGetLastError();
  }
  const auto kernel =
      a.layout.wide ? paged_attn_kernel<E, 8, P8, TREE> : paged_attn_kernel<E, 4, P8, TREE>;
  const int threads = a.layout.wide ? Shape<8>::THREADS : Shape<4>::THREADS;
  hipLaunchKernelGGL(kernel, dim3((unsigned)a.layout.max_items), dim3(threads), 0, a.stream, a);
  if (a.layout.max_merges > 0) {
    const unsigned groups = (unsigned)(a.layout.max_merges < kMergeGroups ? a.layout.max_merges : kMergeGroups);
    hipLaunchKernelGGL(paged_merge_kernel<E>, dim3(groups), dim3(256), 0, a.stream, a);
  }
  return hipGetLastError();
}
template <class E>
hipError_t launch_attention(const PagedAttnArgs& a) {
  if (a.pool.k_exp != nullptr || a.pool.k_exp_stride != 0)  // (a pool without pages may have no address)
    return a.tree == nullptr ? launch_attention<E, true, false>(a) : launch_attention<E, true, true>(a);
  return a.tree == nullptr ? launch_attention<E, false, false>(a) : launch_attention<E, false, true>(a);
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs& a) {
  const int placers = (a.n_tokens + kPlanRowsPerGroup - 1) / kPlanRowsPerGroup;
  const int64_t wanted = (a.layout.max_items + PT - 1) / PT;
  const int writers = (int)(wanted < kPlanWriters ? wanted : kPlanWriters);
  const bool tree = a.parents != nullptr, within = tree && a.n_seqs <= PT;
  const auto kernel = a.n_seqs <= PT       ? (tree ? paged_plan_kernel<1, true> : paged_plan_kernel<1, false>)
                      : a.n_seqs <= 4 * PT ? (tree ? paged_plan_kernel<4, true> : paged_plan_kernel<4, false>)
                      : tree               ? paged_plan_kernel<kPagedMaxSeqs / PT, true>
                                           : paged_plan_kernel<kPagedMaxSeqs / PT, false>;
  hipLaunchKernelGGL(kernel, dim3(2 * writers + placers + (within ? a.n_seqs : 0)), dim3(PT), 0, a.stream, a,
                     writers, placers);
  if (tree && !within) hipLaunchKernelGGL(paged_tree_kernel, dim3(a.n_seqs), dim3(PT), 0, a.stream, a);
  return hipGetLastError();
}

hipError_t launch_paged_attention(const PagedAttnArgs& a) {
  return a.dtype == 0 ? launch_attention<F16>(a) : launch_attention<BF16>(a);
}

}  // namespace va
