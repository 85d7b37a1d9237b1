// Beam search's selection: of all continuations of a prompt's beams, score + log softmax of the logits, the
// best `count`, ties to the lowest beam and token.
//
// The logits are read once. A first kernel takes, of every cell (512 numbers of a row, or a power of two
// more), the largest number and, per wave, the sum of exponentials over the wave's own largest: no order is
// kept there. The `count` best continuations of a prompt lie in its `count` best cells: were one outside,
// each of those cells would hold a better one, or one as good of a lower number, since cells are runs of
// numbers in order. So a second kernel, a work-group per prompt, picks the best cells from their largest
// numbers, and the best numbers in them. Scores are formed and compared in 64 bits, score + (number - log
// of the sum): a rounding to 32 would make ties of continuations that are not as good.
//
// The first kernel is bounded by memory (its arithmetic, 11 instructions a number, takes 2/3 as long); the
// second by the latency of its steps.
#include <climits>
#include <type_traits>

#include "va_beams.h"
#include "va_common.h"

namespace va {

namespace {

constexpr int T = 64 * kBeamsWaves;
constexpr int kNumbers = 8;  // per lane and load

enum { kF16 = 0, kBF16 = 1, kF32 = 2 };

// 8 numbers from `p` on, at any alignment of the element.
template <int DT>
struct Numbers {
  static constexpr int W = DT == kF32 ? 8 : 4;  // words
  uint32_t w[W];
  __device__ inline void load(const void* base, int64_t at) {
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

// The largest number of a wave, in all lanes (not-a-numbers are passed over).
__device__ inline float wave_max(float x) {
  x = fmaxf(x, dpp_mov<0xb1>(x));
  x = fmaxf(x, dpp_mov<0x4e>(x));
  x = fmaxf(x, dpp_mov<0x141>(x));
  x = fmaxf(x, dpp_mov<0x140>(x));
  x = fmaxf(x, __shfl_xor(x, 16));
  return max_with_other_half(x);
}

template <int DT>
__global__ __launch_bounds__(T) void beams_read_kernel(BeamsArgs a) {
  const int row = blockIdx.x, split = blockIdx.y, lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (a.ended != nullptr && a.ended[row] != 0) return;  // (its logits do not count)
  const int64_t base = row * a.row_stride;
  const BeamsLayout& l = a.layout;
  float* tops = a.workspace + (int64_t)row * l.cells;
  float m = -INFINITY, sum = 0.f;  // this lane's
  for (int c = split * kBeamsWaves + wave; c < l.cells; c += l.splits * kBeamsWaves) {
    float top = -INFINITY;
    for (int i = c * l.cell + kNumbers * lane; i < (c + 1) * l.cell; i += kNumbers * 64) {
      Numbers<DT> x;
      if (i + kNumbers <= a.vocab) x.load(a.logits, base + i);
      else x.load_some(a.logits, base + min(i, a.vocab), a.vocab - i);
      float mine = -INFINITY;
#pragma unroll
      for (int e = 0; e < kNumbers; ++e) mine = fmaxf(mine, x.get(e));
      top = fmaxf(top, mine);
      // (differences, not products with the largest number taken apart: what counts is exact)
      const float now = fmaxf(m, mine), ref = now == -INFINITY ? 0.f : now;
      sum *= fast_exp2((m - ref) * kLog2e);
      m = now;
#pragma unroll
      for (int e = 0; e < kNumbers; ++e) sum += fast_exp2((x.get(e) - ref) * kLog2e);
    }
    top = wave_max(top);
    if (lane == 0) tops[c] = top;
  }
  const float all = wave_max(m), ref = all == -INFINITY ? 0.f : all;
  sum *= fast_exp2((m - ref) * kLog2e);
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
// A candidate: its score as a whole number of the same order (0: none) and its number.
struct Pick {
  uint64_t key;
  int index, pad;
};
__device__ inline bool before(uint64_t key, int index, uint64_t than, int than_index) {
  return key > than || (key == than && index < than_index);
}
// 64-bit floats in order; not a number counts as -infinity.
__device__ inline uint64_t key_of(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x != x ? -__builtin_inf() : x == 0 ? 0.0 : x);
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ inline double value_of(uint64_t key) {
  return __builtin_bit_cast(double, key >> 63 ? key & ~(1ull << 63) : ~key);
}

constexpr int kPool = 4096;  // candidates that pass the threshold, at most
struct Picks {
  Pick pool[kPool], best[64], out[kBeamsCount];
  int n;
};

// The best `count` of all candidates that each(visit) shows to visit(key, index), in order, to s.out; returns how
// many there are. Each group of 4 threads brings its best one; the count-th best of those 64 is a bound
// that `count` candidates reach, and only those of the groups whose best reaches it: at most 4 count times the
// candidates of a thread (kPool is no less). They are then put in order by counting who comes before.
template <class Each>
__device__ inline int select(Picks& s, int count, Each each) {
  const int tid = threadIdx.x;
  uint64_t key = 0;
  int index = INT_MAX;
  each([&](uint64_t k, int i) {
    if (k != 0 && before(k, i, key, index)) key = k, index = i;
  });
#pragma unroll
  for (int d = 1; d < 4; d *= 2) {
    const uint64_t k = __shfl_xor((unsigned long long)key, d);
    const int i = __shfl_xor(index, d);
    if (before(k, i, key, index)) key = k, index = i;
  }
  __syncthreads();  // (the pool and s.n may be in use from before)
  if ((tid & 3) == 0) s.best[tid >> 2] = Pick{key, index, 0};
  if (tid == 0) s.n = 0;
  __syncthreads();
  // every wave finds the bound for itself: lane l ranks group l
  const Pick mine = s.best[tid & 63];
  int rank = 0;
#pragma unroll 8
  for (int j = 0; j < 64; ++j) {
    const Pick p = s.best[j];
    rank += before(p.key, p.index, mine.key, mine.index);
  }
  // (groups without a candidate are equal: all of them rank behind the others)
  const uint64_t at = __builtin_amdgcn_ballot_w64(rank == count - 1 && mine.key != 0);
  uint64_t least = 0;
  int last = INT_MAX;
  if (at != 0) {
    const int l = __builtin_ctzll(at);
    least = __shfl((unsigned long long)mine.key, l);
    last = __shfl(mine.index, l);
  }
  each([&](uint64_t k, int i) {
    if (k != 0 && !before(least, last, k, i)) {
      const int n = atomicAdd(&s.n, 1);
      if (n < kPool) s.pool[n] = Pick{k, i, 0};
    }
  });
  __syncthreads();
  const int n = min(s.n, kPool);
  for (int i = tid; i < n; i += T) {
    const Pick p = s.pool[i];
    int r = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) {
      const Pick o = s.pool[j];
      r += before(o.key, o.index, p.key, p.index);
    }
    if (r < count) s.out[r] = p;
  }
  __syncthreads();
  return min(n, count);
}

// Cells, or runs of numbers, are gone through in the order of their numbers.
__device__ inline void in_order(const Picks& s, int n, int* order) {
  const int tid = threadIdx.x;
  if (tid < n) {
    int r = 0;
    for (int j = 0; j < n; ++j) r += s.out[j].index < s.out[tid].index;
    order[r] = s.out[tid].index;
  }
  __syncthreads();
}

template <int DT>
__global__ __launch_bounds__(T) void beams_pick_kernel(BeamsArgs a) {
  __shared__ Picks s;
  __shared__ double s_score[kBeamsMost], s_sum[kBeamsMost];
  __shared__ int s_runs[kBeamsCount];
  const BeamsLayout& l = a.layout;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, first = blockIdx.x * a.beams;
  auto ended = [&](int beam) { return a.ended != nullptr && a.ended[first + beam] != 0; };

  // log of the sum of exponentials of every beam (an ended one: all of its weight on its end token)
  const int waves = l.splits * kBeamsWaves;
  for (int b = wave; b < a.beams; b += kBeamsWaves) {
    const f32x2* sums = reinterpret_cast<const f32x2*>(a.workspace + l.sums) + (int64_t)(first + b) * waves;
    const bool done = ended(b);
    float m = -INFINITY;
    for (int i = lane; i < waves && !done; i += 64) m = fmaxf(m, sums[i][0]);
    m = wave_max(m);
    double sum = 0;
    for (int i = lane; i < waves && !done; i += 64) {
      const f32x2 x = sums[i];
      if (x[0] != -INFINITY || x[1] != 0.f) sum += (double)x[1] * exp((double)x[0] - (double)m);
    }
    for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
    if (lane == 0) {
      s_score[b] = a.scores[first + b];
      s_sum[b] = done ? 0.0 : (double)m + log(sum);
    }
  }
  __syncthreads();
  auto key = [&](int beam, float x) { return key_of(s_score[beam] + ((double)x - s_sum[beam])); };

  // the best cells
  const int cells = a.beams * l.cells;
  int n = select(s, min(a.count, cells), [&](auto visit) {
    for (int i = tid; i < cells; i += T) {
      const int beam = i / l.cells, c = i % l.cells;
      const float top = ended(beam) ? (a.end_token / l.cell == c ? 0.f : -INFINITY)
                                    : a.workspace[(int64_t)(first + beam) * l.cells + c];
      visit(key(beam, top), i);
    }
  });
  in_order(s, n, s_runs);

  // the largest numbers of runs of `run` numbers of them, then the numbers themselves; each thread takes
  // kNumbers numbers at a time. Index of a number: beam * 2^18 + token (of a run: its first number's).
  auto number = [&](int at) { return s_runs[at]; };
  auto see = [&](int beam, int token, auto visit) {  // up to kNumbers numbers from `token` on
    if (token >= a.vocab) return;
    Numbers<DT> x;
    const int64_t base = (int64_t)(first + beam) * a.row_stride + token;
    const int some = min(a.vocab - token, kNumbers);
    const bool done = ended(beam);
    if (some == kNumbers) x.load(a.logits, base);
    else x.load_some(a.logits, base, some);
#pragma unroll
    for (int e = 0; e < kNumbers; ++e)
      if (e < some) visit(done ? (token + e == a.end_token ? 0.f : -INFINITY) : x.get(e), e);
  };
  int run = l.cell;
  for (int i = tid; i < n; i += T) s_runs[i] = s_runs[i] / l.cells * kBeamsVocab + s_runs[i] % l.cells * l.cell;
  __syncthreads();
  // (what a group of 4 threads then goes through, count times, has to fit in the pool)
  if (a.count * ((n * (run / kNumbers) + T - 1) / T) * 4 * kNumbers > kPool) {
    const int part = run / 64;
    n = select(s, a.count, [&](auto visit) {
      for (int i = tid; i < 64 * n; i += T) {
        const int at = number(i >> 6) + (i & 63) * part, beam = at / kBeamsVocab, token = at % kBeamsVocab;
        float top = -INFINITY;
        for (int k = 0; k < part; k += kNumbers)
          see(beam, token + k, [&](float x, int) { top = fmaxf(top, x); });
        if (token < a.vocab) visit(key(beam, top), at);
      }
    });
    in_order(s, n, s_runs);
    run = part;
  }
  const int loads = run / kNumbers;
  n = select(s, a.count, [&](auto visit) {
    for (int i = tid; i < n * loads; i += T) {
      const int at = number(i / loads) + i % loads * kNumbers, beam = at / kBeamsVocab;
      see(beam, at % kBeamsVocab, [&](float x, int e) { visit(key(beam, x), at + e); });
    }
  });
  if (tid < a.count) {  // (n is count: there are no fewer numbers)
    const Pick p = s.out[min(tid, n - 1)];
    const int64_t at = (int64_t)blockIdx.x * a.count + tid;
    a.scores_out[at] = (float)value_of(p.key);
    a.parents_out[at] = first + p.index / kBeamsVocab;
    a.tokens_out[at] = p.index % kBeamsVocab;
  }
}

template <int DT>
void select_beams(const BeamsArgs& a) {
  hipLaunchKernelGGL(beams_read_kernel<DT>, dim3(a.groups * a.beams, a.layout.splits), dim3(T), 0, a.stream, a);
  hipLaunchKernelGGL(beams_pick_kernel<DT>, dim3(a.groups), dim3(T), 0, a.stream, a);
}

}  // namespace

hipError_t launch_select_beams(const BeamsArgs& a) {
  (a.dtype == kF16 ? select_beams<kF16> : a.dtype == kBF16 ? select_beams<kBF16> : select_beams<kF32>)(a);
  return hipGetLastError();
}

}  // namespace va
