// Beam search's selection: of all continuations of a prompt's beams, score + log softmax of the logits, the
// best `count`, ties to the lowest beam and token.
//
// The logits are read once. A first kernel takes, of every cell (512 numbers of a row, or a power of two
// more), the largest number and, per wave, the sum of exponentials over the wave's own largest: no order is
// kept there. The `count` best continuations of a prompt lie in its `count` best cells: were one outside,
// each of those cells would hold a better one, or one as good of a lower number, since cells are runs of
// numbers in order. So a second kernel, a work-group per prompt, picks the best cells from their largest
// numbers, and the best numbers in them. Scores are formed and compared in 64 bits, score + (number - log
// of the sum): a rounding to 32 would make ties of continuations that are not as good. The sum itself is off by
// what a wave's additions in fp32 lose, (8 ceil(vocab / 2048) + 48) 2^-24 of it at most: the order is exact within a
// row and between rows of the same numbers; continuations of other rows whose scores are closer than twice that may
// change places.
//
// The first kernel is bounded by memory, and for 16-bit numbers nearly as much by its arithmetic (a
// power of two, 16 cycles of a wave, and six other instructions a number): 512 rows of 150,016 numbers
// (154 MB) 34 us, 4.6 TB/s; of 75,008 fp32 numbers, as many bytes, 30 us. 1, 2 and 4 pieces on their
// way and 1024 to 8192 work-groups measured 34 to 47. The second kernel is, for ordinary logits and counts of 16 or
// so (see select), bounded by the latency of its dozen steps between barriers, some 0.45 us each, and of its first loads (1.7 and 1.1): 8.2 us for a prompt of four
// beams, 10.2 us for 64 of eight (with scores compared as whole numbers and ranks added up in LDS 8.8 and
// 11.2; with 256 threads 13.8 and 33.7; with one copy of the code for all picks 8.9 and 12.8).
#include <climits>
#include <type_traits>

#include "va_beams.h"
#include "va_common.h"

namespace va {

namespace {

constexpr int T = 64 * kBeamsWaves;
constexpr int kNumbers = 8;  // per lane and load

enum { kF16 = 0, kBF16 = 1, kF32 = 2 };

// 8 numbers of a row, as loaded.
template <int DT>
struct Numbers {
  static constexpr int W = DT == kF32 ? 8 : 4;  // words
  uint32_t w[W];
  __device__ inline void load(const void* base, int64_t at) {  // at any address of an element
    __builtin_memcpy(w, (const char*)base + at * (DT == kF32 ? 4 : 2), 4 * W);
  }
  __device__ inline void load_some(const void* base, int64_t at, int count) {  // the others: -infinity
#pragma unroll
    for (int i = 0; i < kNumbers; ++i) {
      if constexpr (DT == kF32) {
        w[i] = i < count ? ((const uint32_t*)base)[at + i] : 0xff800000u;
      } else {
        const uint32_t x = i < count ? ((const uint16_t*)base)[at + i] : DT == kF16 ? 0xfc00u : 0xff80u;
        w[i >> 1] = i & 1 ? w[i >> 1] | x << 16 : x;
      }
    }
  }
  __device__ inline float get(int i) const {
    if constexpr (DT == kF32) return __builtin_bit_cast(float, w[i]);
    else if constexpr (DT == kF16) return F16::to_f32((uint16_t)(w[i >> 1] >> (16 * (i & 1))));
    else return __builtin_bit_cast(float, i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
  }
};

// The same on the way: 16-bit numbers that begin in the middle of a word (ODD) are loaded as the words that
// they lie in, from the number before them to the one behind them, and shifted when they are used (512 rows
// of 150,001: 36 us, 39 with loads that straddle words). Not by cells that begin elsewhere: rows that
// hold the same numbers have the same sum to the last bit, or equal scores would be no ties.
template <int DT, bool ODD>
struct Coming {
  Numbers<DT> x;
  uint32_t last;
  // numbers i to i + 7 of the row at `row`, of which the one before and the one behind exist if ODD
  __device__ inline void load(const void* logits, int64_t row, int i) {
    x.load(logits, row + i - ODD);
    if constexpr (ODD) __builtin_memcpy(&last, (const char*)logits + 2 * (row + i + kNumbers - 1), 4);
  }
  __device__ inline Numbers<DT> numbers() const {
    Numbers<DT> y = x;
    if constexpr (ODD) {
#pragma unroll
      for (int k = 0; k < Numbers<DT>::W; ++k)
        y.w[k] = __builtin_amdgcn_alignbit(k + 1 < Numbers<DT>::W ? x.w[k + 1] : last, x.w[k], 16);
    }
    return y;
  }
};

// The largest number of a wave, in all lanes (not-a-numbers are passed over).
__device__ inline float wave_max(float x) {
  x = fmaxf(x, dpp_mov<0xb1>(x));
  x = fmaxf(x, dpp_mov<0x4e>(x));
  x = fmaxf(x, dpp_mov<0x141>(x));
  x = fmaxf(x, dpp_mov<0x140>(x));
  x = fmaxf(x, __shfl_xor(x, 16));
  return max_with_other_half(x);
}

// The same in the last lane only, without LDS.
template <int CTRL, int ROWS>
__device__ inline float dpp_max(float x) {
  const int i = __builtin_bit_cast(int, x);
  return fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, ROWS, 0xf, false)));
}
__device__ inline float wave_max_last(float x) {
  x = dpp_max<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8: within rows of 16 lanes
  x = dpp_max<0x112, 0xf>(x);
  x = dpp_max<0x114, 0xf>(x);
  x = dpp_max<0x118, 0xf>(x);
  x = dpp_max<0x142, 0xa>(x);  // row_bcast 15: the last lane of a row to the next one (rows 1, 3)
  return dpp_max<0x143, 0xc>(x);  // row_bcast 31: lane 31 to rows 2, 3
}

// Exponentials are powers of two, number * kLog2e less the reference of the largest number so far. Up
// to 2^16 that is largest * kLog2e rounded, so that a power costs a fused multiply-add and one
// rounding, of a difference; from there on, where that rounding would count, the product itself:
// differences of numbers are taken first. kLog2e, rounded, stands for the base: the second kernel
// divides by it, so a shift of all numbers shifts the result.
__device__ inline bool far_out(float largest) { return fabsf(largest) >= 65536.f; }
// Power of two by which a sum over the reference of `was` has to be multiplied for that of `is`. (References are
// the rounded products: their difference may not become a multiply-add of an unrounded one.)
__device__ inline float rescale(float was, float is) {
#pragma clang fp contract(off)
  const float a = was * kLog2e, b = is * kLog2e;
  const float d = far_out(is) ? (far_out(was) ? (was - is) * kLog2e : __builtin_fmaf(-is, kLog2e, a))
                              : (far_out(was) ? __builtin_fmaf(was, kLog2e, -b) : a - b);
  return fast_exp2(d);
}

// A wave's part of a row: the largest numbers of its cells, every step-th one from c0 on, and per lane the
// largest number and the sum. Cells are gone through in pieces of 64 kNumbers numbers, PIECES at a time (of
// as many cells, or of one), as many on their way: a reduction over the wave, the exponentials' latency and
// the test for a new largest number are then paid once.
constexpr int PIECES = 2;
template <int DT, bool ODD>
__device__ inline void read_row(const BeamsArgs& a, int64_t base, float* tops, int c0, int step, float& top,
                                float& sum) {
  const BeamsLayout& l = a.layout;
  const int lane = threadIdx.x & 63, shift = __builtin_ctz(l.cell / (64 * kNumbers));
  const int pieces = c0 < l.cells ? ((l.cells - 1 - c0) / step + 1) << shift : 0;
  auto cell_of = [&](int p) { return c0 + (p >> shift) * step; };
  auto begin_of = [&](int p) { return cell_of(p) * l.cell + (p & ((1 << shift) - 1)) * (64 * kNumbers); };
  // Loads are the same for all pieces, from inside the row; what a row's first or last piece, or one that
  // there is not, got from elsewhere is replaced when it is used.
  const int least = ODD, most = a.vocab - kNumbers - ODD;
  auto plain = [&](int p) {
    return p < pieces && begin_of(p) >= least && begin_of(p) + 64 * kNumbers <= a.vocab - ODD;
  };
  Coming<DT, ODD> next[PIECES];
  auto fetch = [&](int p) {
    if (most < least) return;  // (a row of a few numbers: replaced)
#pragma unroll
    for (int j = 0; j < PIECES; ++j)
      next[j].load(a.logits, base, max(min(begin_of(p + j) + kNumbers * lane, most), least));
  };
  float ref = 0.f, cell = -INFINITY;
  bool some_far = false;  // some lane's largest number is far out
  fetch(0);
  for (int p = 0; p < pieces; p += PIECES) {
    Numbers<DT> x[PIECES];
#pragma unroll
    for (int j = 0; j < PIECES; ++j) x[j] = next[j].numbers();
    fetch(p + PIECES);
#pragma unroll
    for (int j = 0; j < PIECES; ++j)
      if (!plain(p + j)) {
        const int i = p + j < pieces ? begin_of(p + j) + kNumbers * lane : a.vocab;
        x[j].load_some(a.logits, base + min(i, a.vocab), a.vocab - i);
      }
    float mine[PIECES], part[PIECES];
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      part[j] = 0.f;
      mine[j] = x[j].get(0);
#pragma unroll
      for (int e = 1; e < kNumbers; ++e) mine[j] = fmaxf(mine[j], x[j].get(e));
    }
    float all = mine[0];
#pragma unroll
    for (int j = 1; j < PIECES; ++j) all = fmaxf(all, mine[j]);
    if (__builtin_amdgcn_ballot_w64(all > top) != 0) {
      const float more = fmaxf(top, all);
      sum *= top == -INFINITY ? 0.f : rescale(top, more);
      top = more;
      ref = more == -INFINITY ? 0.f : more * kLog2e;
      some_far = __builtin_amdgcn_ballot_w64(more != -INFINITY && far_out(more)) != 0;
    }
    if (!some_far) {
#pragma unroll
      for (int e = 0; e < kNumbers; ++e)
#pragma unroll
        for (int j = 0; j < PIECES; ++j) part[j] += fast_exp2(__builtin_fmaf(x[j].get(e), kLog2e, -ref));
    } else {
      const bool mine_far = top != -INFINITY && far_out(top);
#pragma unroll
      for (int e = 0; e < kNumbers; ++e)
#pragma unroll
        for (int j = 0; j < PIECES; ++j)
          part[j] += fast_exp2(mine_far ? (x[j].get(e) - top) * kLog2e
                                        : __builtin_fmaf(x[j].get(e), kLog2e, -ref));
    }
#pragma unroll
    for (int j = 0; j < PIECES; ++j) sum += part[j];
    if (shift == 0) {
#pragma unroll
      for (int j = 0; j < PIECES; ++j) mine[j] = wave_max_last(mine[j]);
#pragma unroll
      for (int j = 0; j < PIECES; ++j)
        if (lane == 63 && p + j < pieces) tops[cell_of(p + j)] = mine[j];
    } else {
#pragma unroll
      for (int j = 0; j < PIECES; ++j) {
        cell = fmaxf(cell, mine[j]);
        if (((p + j + 1) & ((1 << shift) - 1)) == 0) {
          cell = wave_max_last(cell);
          if (lane == 63 && p + j < pieces) tops[cell_of(p + j)] = cell;
          cell = -INFINITY;
        }
      }
    }
  }
}

template <int DT>
__global__ __launch_bounds__(T) void beams_read_kernel(BeamsArgs a) {
  const int row = blockIdx.x, split = blockIdx.y, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (a.ended != nullptr && a.ended[row] != 0) return;  // (its logits do not count)
  const int64_t base = row * a.row_stride;
  const BeamsLayout& l = a.layout;
  float* tops = a.workspace + (int64_t)row * l.cells;
  float top = -INFINITY, sum = 0.f;
  const int c0 = split * kBeamsWaves + wave, step = l.splits * kBeamsWaves;
  if (DT != kF32 && ((((uintptr_t)a.logits >> 1) + (uint64_t)base) & 1) != 0)
    read_row<DT, DT != kF32>(a, base, tops, c0, step, top, sum);
  else
    read_row<DT, false>(a, base, tops, c0, step, top, sum);
  const float all = wave_max(top);
  sum *= top == -INFINITY ? 1.f : rescale(top, all);  // (of -infinity: 0, or not a number)
#pragma unroll
  for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  if (lane == 0) {
    const int64_t at = ((int64_t)row * l.splits + split) * kBeamsWaves + wave;
    *reinterpret_cast<f32x2*>(a.workspace + l.sums + 2 * at) = f32x2{all, sum};
  }
}

// ------------------------------------------------------------------------------------------------
// selection
// ------------------------------------------------------------------------------------------------
// A candidate: its score (not a number: -infinity) and its number; none: -infinity and INT_MAX, behind all.
struct Pick {
  double score;
  int index, pad;
};
__device__ inline bool before(double score, int index, double than, int than_index) {
  return score > than || (score == than && index < than_index);
}

constexpr int PT = 1024, PW = PT / 64;  // threads and waves of a work-group that picks
constexpr int kPool = 4096;             // candidates that pass the threshold, at most
struct Picks {
  Pick pool[kPool], best[64], out[kBeamsCount], least;
  int n;
};

// Over the 16 lanes of a row: the total, and the first in order, in all of them.
template <int CTRL>
__device__ inline int turned(int x) {  // (row_ror)
  return __builtin_amdgcn_update_dpp(x, x, CTRL, 0xf, 0xf, false);
}
__device__ inline int row_sum(int x) {
  x += turned<0x128>(x);
  x += turned<0x124>(x);
  x += turned<0x122>(x);
  return x + turned<0x121>(x);
}
template <int CTRL>
__device__ inline void first_of(double& score, int& index) {
  const uint64_t b = __builtin_bit_cast(uint64_t, score);
  const uint32_t lo = (uint32_t)turned<CTRL>((int)(uint32_t)b), hi = (uint32_t)turned<CTRL>((int)(b >> 32));
  const double x = __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  const int i = turned<CTRL>(index);
  if (before(x, i, score, index)) score = x, index = i;
}
// How many of v[0..n) come before `mine`, which the 16 lanes of a row have in common and share the others of.
__device__ inline int count_before(const Pick* v, int n, const Pick& mine) {
  int r = 0;
#pragma unroll 4
  for (int j = threadIdx.x & 15; j < n; j += 16) {
    const Pick p = v[j];
    r += before(p.score, p.index, mine.score, mine.index);
  }
  return row_sum(r);
}

// The best `count` of all threads' E candidates (a thread's in the order of their numbers), in order, to s.out; returns how many there
// are. Each group of 16 threads brings its best one; the count-th best of those 64 is a bound that `count`
// candidates reach, and only those of the groups whose best reaches it: at most 16 E count (and not more
// than there are; the callers see to it that kPool is no less). They are then put in order by counting who
// comes before, n^2 reads of LDS for a pool of n. Ordinary logits leave little more than `count`. Where the count-th
// best group's best is -infinity, or equal to others, order goes by number alone and whole groups pass: 129, 516 and
// 1032 candidates where all beams of a prompt have ended, at 1 beam and count 2, 4 and 8, 8 and 16; counts near the
// 64 groups have a bound that many pass in any case. A work-group is then as slow as its pool (us a call of 32,000
// fp16 numbers a row, ordinary / a prompt all of whose beams have ended / equal logits / 10 allowed tokens): 64 prompts
// of 4 beams, count 8, 15.9 / 43 / 94 / 45, of 8, count 16, 20 / 119 / 353 / 130; 16 of 32, count 64, 135 / 241 / 244 /
// 249, and 1164 where every other beam has ended. Sums over 16 lanes stay in registers.
template <int E>
__device__ inline int select(Picks& s, int count, const double (&score)[E], const int (&index)[E]) {
  const int tid = threadIdx.x, group = tid >> 4;
  double top = score[0];
  int at = index[0];
#pragma unroll
  for (int e = 1; e < E; ++e)
    if (score[e] > top || at == INT_MAX) top = score[e], at = index[e];
  first_of<0x128>(top, at);
  first_of<0x124>(top, at);
  first_of<0x122>(top, at);
  first_of<0x121>(top, at);
  __syncthreads();  // (the pool and the counts may be in use from before)
  if ((tid & 15) == 0) s.best[group] = Pick{top, at, 0};
  if (tid == 0) {
    s.n = 0;
    s.least = Pick{-__builtin_inf(), INT_MAX - 1, 0};  // (where fewer groups than `count` have a candidate)
  }
  __syncthreads();
  // (groups without a candidate are alike and come behind the others)
  const int rank = count_before(s.best, 64, Pick{top, at, 0});
  if (rank == count - 1 && at != INT_MAX && (tid & 15) == 0) s.least = Pick{top, at, 0};
  __syncthreads();
  const Pick least = s.least;
  uint64_t hits[E];
  int total = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    hits[e] = __builtin_amdgcn_ballot_w64(!before(least.score, least.index, score[e], index[e]));
    total += __builtin_popcountll(hits[e]);
  }
  if (total > 0) {  // (the same in all lanes)
    int place = 0;
    if ((tid & 63) == 0) place = atomicAdd(&s.n, total);
    place = __builtin_amdgcn_readfirstlane(place);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (hits[e] == 0) continue;
      const int n = place + __builtin_amdgcn_mbcnt_hi((uint32_t)(hits[e] >> 32),
                                                      __builtin_amdgcn_mbcnt_lo((uint32_t)hits[e], 0));
      if (hits[e] >> (tid & 63) & 1 && n < kPool) s.pool[n] = Pick{score[e], index[e], 0};
      place += __builtin_popcountll(hits[e]);
    }
  }
  __syncthreads();
  const int n = min(s.n, kPool);
  for (int i = group; i - group < n; i += PT / 16) {  // (whole waves stay together)
    const Pick p = s.pool[max(0, min(i, n - 1))];
    const int r = count_before(s.pool, n, p);
    if ((tid & 15) == 0 && i < n && r < count) s.out[r] = p;
  }
  __syncthreads();
  return min(n, count);
}

// Where the chosen runs of numbers begin, in the order of their numbers.
template <class First>
__device__ inline void in_order(const Picks& s, int n, int* runs, First first) {
  const int tid = threadIdx.x;
  if (tid < n) {
    int r = 0;
    for (int j = 0; j < n; ++j) r += s.out[j].index < s.out[tid].index;
    runs[r] = first(s.out[tid].index);
  }
  __syncthreads();
}

template <int DT>
__global__ __launch_bounds__(PT) void beams_pick_kernel(BeamsArgs a) {
  __shared__ Picks s;
  __shared__ double s_score[kBeamsMost], s_sum[kBeamsMost];
  __shared__ bool s_ended[kBeamsMost];
  __shared__ int s_runs[kBeamsCount];
  constexpr int CELLS = kBeamsCells / PT;
  const BeamsLayout& l = a.layout;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, first = blockIdx.x * a.beams;

  // the cells' largest numbers, on their way while the sums are formed
  const int cells = a.beams * l.cells;
  const float* tops = a.workspace + (int64_t)first * l.cells;
  float top[CELLS];
#pragma unroll
  for (int e = 0; e < CELLS; ++e) top[e] = e * PT + tid < cells ? tops[e * PT + tid] : 0.f;
  // log of the sum of exponentials of every beam (an ended one: all of its weight on its end token)
  const int waves = l.splits * kBeamsWaves;
  for (int b = wave; b < a.beams; b += PW) {
    const f32x2* sums = reinterpret_cast<const f32x2*>(a.workspace + l.sums) + (int64_t)(first + b) * waves;
    const float score = a.scores[first + b];
    const bool done = a.ended != nullptr && a.ended[first + b] != 0;
    double sum = 0, ref = 0;
    if (!done) {
      const f32x2 none = {-INFINITY, 0.f}, mine = lane < waves ? sums[lane] : none;
      float m = mine[0];
      for (int i = lane + 64; i < waves; i += 64) m = fmaxf(m, sums[i][0]);
      m = wave_max(m);
      auto ref_of = [](float x) { return far_out(x) ? (double)x * (double)kLog2e : (double)(x * kLog2e); };
      ref = ref_of(m);
      // (-infinity with a sum of 0: nothing was read, or nothing but -infinity)
      auto add = [&](const f32x2& x) {
        if (x[0] != -INFINITY || x[1] != 0.f) sum += (double)x[1] * exp2(ref_of(x[0]) - ref);
      };
      add(mine);
      for (int i = lane + 64; i < waves; i += 64) add(sums[i]);
      for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    }
    if (lane == 0) {
      s_score[b] = score;
      s_sum[b] = done ? 0.0 : (ref + log2(sum)) / (double)kLog2e;
      s_ended[b] = done;
    }
  }
  __syncthreads();
  constexpr double none = -__builtin_inf();
  auto score_of = [&](int beam, float x) { return fmax(s_score[beam] + ((double)x - s_sum[beam]), none); };

  // the best cells
  int n;
  {
    // (quotients of small numbers: exact in fp32, half a unit to spare)
    const float inv = 1.f / (float)l.cells;
    const int end_cell = a.end_token / l.cell;
    double score[CELLS];
    int index[CELLS];
#pragma unroll
    for (int e = 0; e < CELLS; ++e) {
      const int i = e * PT + tid;
      index[e] = i < cells ? i : INT_MAX;
      score[e] = none;
      if (i < cells) {
        const int beam = (int)(((float)i + 0.5f) * inv);
        if (s_ended[beam]) top[e] = i - beam * l.cells == end_cell ? 0.f : -INFINITY;
        score[e] = score_of(beam, top[e]);
      }
    }
    n = select(s, min(a.count, cells), score, index);
  }
  in_order(s, n, s_runs, [&](int i) { return i / l.cells * kBeamsVocab + i % l.cells * l.cell; });

  // the best runs in them where their numbers are too many, then the numbers. Each thread takes
  // kNumbers at a time. Index of a number: beam * 2^18 + token (of a run: its first number's).
  auto see = [&](int at, float (&x)[kNumbers]) {  // numbers from `at` on; returns how many there are
    const int beam = at / kBeamsVocab, token = at % kBeamsVocab, some = min(a.vocab - token, kNumbers);
    if (some <= 0) return 0;
    const int64_t base = (int64_t)(first + beam) * a.row_stride + token;
    const bool done = s_ended[beam];
    Numbers<DT> w;
    if (some == kNumbers) w.load(a.logits, base);
    else w.load_some(a.logits, base, some);
#pragma unroll
    for (int e = 0; e < kNumbers; ++e)
      x[e] = !done ? w.get(e) : token + e == a.end_token ? 0.f : -INFINITY;
    return some;
  };
  int run = l.cell;  // (a power of two from here on)
  if (n * (run / kNumbers) > PT || (16 * kNumbers * a.count > kPool && n * run > kPool)) {
    constexpr int RUNS = 64 * kBeamsCount / PT;
    const int part = run / 64;
    double score[RUNS];
    int index[RUNS];
#pragma unroll
    for (int e = 0; e < RUNS; ++e) {
      const int i = e * PT + tid;
      score[e] = none;
      index[e] = INT_MAX;
      if (i < 64 * n) {
        const int at = s_runs[i >> 6] + (i & 63) * part;
        float best = -INFINITY;
        bool any = false;
        for (int k = 0; k < part; k += kNumbers) {
          float x[kNumbers];
          const int some = see(at + k, x);
#pragma unroll
          for (int j = 0; j < kNumbers; ++j)
            if (j < some) best = fmaxf(best, x[j]);
          any = any || some > 0;
        }
        if (any) {
          index[e] = at;
          score[e] = score_of(at / kBeamsVocab, best);
        }
      }
    }
    n = select(s, a.count, score, index);
    in_order(s, n, s_runs, [](int i) { return i; });
    run = part;
  }
  {
    const int shift = __builtin_ctz(run / kNumbers), loads = n << shift;
    double score[kNumbers];
    int index[kNumbers];
    float x[kNumbers];
    const int at = tid < loads ? s_runs[tid >> shift] + (tid & ((1 << shift) - 1)) * kNumbers : 0;
    const int some = tid < loads ? see(at, x) : 0;
#pragma unroll
    for (int e = 0; e < kNumbers; ++e) {
      index[e] = e < some ? at + e : INT_MAX;
      score[e] = e < some ? score_of(at / kBeamsVocab, x[e]) : none;
    }
    n = select(s, a.count, score, index);
  }
  if (tid < a.count) {  // (n is count: there are no fewer numbers)
    const Pick p = s.out[min(tid, n - 1)];
    const int64_t at = (int64_t)blockIdx.x * a.count + tid;
    a.scores_out[at] = (float)p.score;
    a.parents_out[at] = first + p.index / kBeamsVocab;
    a.tokens_out[at] = p.index % kBeamsVocab;
  }
}

template <int DT>
void select_beams(const BeamsArgs& a) {
  hipLaunchKernelGGL(beams_read_kernel<DT>, dim3(a.groups * a.beams, a.layout.splits), dim3(T), 0, a.stream, a);
  hipLaunchKernelGGL(beams_pick_kernel<DT>, dim3(a.groups), dim3(PT), 0, a.stream, a);
}

}  // namespace

hipError_t launch_select_beams(const BeamsArgs& a) {
  (a.dtype == kF16 ? select_beams<kF16> : a.dtype == kBF16 ? select_beams<kBF16> : select_beams<kF32>)(a);
  return hipGetLastError();
}

}  // namespace va
