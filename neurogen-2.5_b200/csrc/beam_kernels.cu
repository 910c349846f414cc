// Beam selection and state reordering.
//
// A candidate (beam w, token v) has the cumulative log probability
//   total = score[w] + (x[w][v] - lse[w]),  lse[w] = log sum_{v allowed} exp x[w][v],
// a finished beam the one candidate (w, pad) of total score[w].  Only finite
// totals are candidates: a beam that does not exist (score -inf), a row whose
// mask leaves nothing and a row holding a NaN or +inf have none.  The `beams`
// best, in order, are the next beams.
//
// The comparison between beams is one of sums of the same size, so lse and
// totals are formed in 64 bits, with exponentials good to 1e-12: which beam
// survives does not depend on how a row was split over threads unless two
// totals lie that close.  Within a beam the order of totals is the order
// of logits, which needs no arithmetic: equal logits go to the lower token,
// equal totals of two beams to the lower beam.
//
// Each row therefore gives a sorted list of its at most `beams` best logits,
// and the rows' lists are joined (finish_group).
//
// A warp streams over a row, or a part of one.  Its best 32 are kept sorted,
// one a lane; values above the last that matters gather in shared memory and
// are sorted and merged in 32 at a time, so that most values cost a comparison.
// (Taking the best out one by one with warp-wide maxima cost 120 instructions
// a beam and row: 64 x 32 x 264 38 us, 15.9 now.)
#include "beam_kernels.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <stdexcept>

namespace ngb {
namespace {

constexpr unsigned kAll = 0xFFFFFFFFu;

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// Logits as unsigned keys in their order: the bits, negative ones inverted,
// from -inf = 0 up.  0 is also a masked token: no candidate.  +inf and NaN (of
// either sign: the addition, which makes -0 +0, also makes every NaN the same
// positive one) leave the row's distribution undefined: kBadKey and above.
constexpr uint32_t kLowest = 0x007FFFFFu, kBadKey = 0xFF800000u - kLowest;
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(__fadd_rn(x, 0.f));
  return (u ^ (uint32_t(int(u) >> 31) | 0x80000000u)) - kLowest;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  const uint32_t k = key + kLowest;
  return __uint_as_float(k ^ (~uint32_t(int(k) >> 31) | 0x80000000u));
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = __dadd_rn(v, __shfl_xor_sync(kAll, v, o));
  return v;
}

// exp of N values in [-140, 0], each to about 1e-12 of it: 2^n times the Taylor
// polynomial of degree 10 on |r| <= ln 2 / 2 (its remainder is below 3e-13).
// The values go through each step together, which the volatile statements keep
// (9 values of a warp: 916 clocks; one after the other, as the compiler orders
// plain code, 1,492).
__constant__ double kTaylor[11] = {1.0 / 3628800, 1.0 / 362880, 1.0 / 40320, 1.0 / 5040, 1.0 / 720, 1.0 / 120,
                                   1.0 / 24,      1.0 / 6,      0.5,         1.0,        1.0};
__constant__ double kExp[3] = {6755399441055744.0, // 1.5 * 2^52: the sum's low word is the nearest integer
                               1.4426950408889634, 0.6931471805599453};
__device__ __forceinline__ double step_fma(double a, double b, double c) {
  double r;
  asm volatile("fma.rn.f64 %0, %1, %2, %3;" : "=d"(r) : "d"(a), "d"(b), "d"(c));
  return r;
}
template <int N> __device__ __forceinline__ void exp_below(double (&v)[N]) {
  double t[N], p[N];
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = step_fma(v[i], kExp[1], kExp[0]);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = step_fma(-__dsub_rn(t[i], kExp[0]), kExp[2], v[i]);
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = step_fma(v[i], kTaylor[0], kTaylor[1]);
#pragma unroll
  for (int k = 2; k < 11; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = step_fma(p[i], v[i], kTaylor[k]);
#pragma unroll
  for (int i = 0; i < N; ++i)
    v[i] = __hiloint2double(__double2hiint(p[i]) + (__double2loint(t[i]) << 20), __double2loint(p[i]));
}

// Sums of exponentials against the largest logit seen, as its key (0: none).
// Terms 80 or more below it are left out: against a sum of at least 1 they have
// no bit.  With a top of kBadKey or more the sum means nothing.
struct LogSum {
  uint32_t top = 0;
  double sum = 0;
  __device__ __forceinline__ void raise(uint32_t to) { // to >= top
    if (to == top) return;
    double d[1] = {__dsub_rn(double(logit_of(top)), double(logit_of(to)))};
    const bool counts = top && d[0] >= -80.0;
    exp_below(d);
    sum = counts ? __dmul_rn(sum, d[0]) : 0.0;
    top = to;
  }
  // Adds N logits' terms; none above top, -inf for none.  TOGETHER at a time.
  // The bound is one fp32 subtraction: rounded, it still lies within 140 of top.
  template <int TOGETHER, int N> __device__ __forceinline__ void add(const float (&x)[N]) {
    static_assert(N % TOGETHER == 0, "values");
    const float most = logit_of(top), least = top ? __fsub_rn(most, 80.f) : INFINITY;
    const double m = most;
#pragma unroll
    for (int i = 0; i < N; i += TOGETHER) {
      double d[TOGETHER];
#pragma unroll
      for (int j = 0; j < TOGETHER; ++j) d[j] = __dsub_rn(double(x[i + j]), m);
      exp_below(d);
#pragma unroll
      for (int j = 0; j < TOGETHER; ++j)
        if (x[i + j] >= least) sum = __dadd_rn(sum, d[j]);
    }
  }
  __device__ __forceinline__ void join_warp() {
    raise(__reduce_max_sync(kAll, top));
    sum = warp_sum(sum);
  }
};

// A value of a row: its key and token, ordered as one number (descending: the
// larger logit, then the lower token); 0 is none.
__device__ __forceinline__ uint64_t entry(uint32_t key, uint32_t token) {
  return key ? (uint64_t(key) << 32) | uint32_t(~token) : 0;
}
__device__ __forceinline__ uint32_t entry_key(uint64_t e) { return uint32_t(e >> 32); }
__device__ __forceinline__ int entry_token(uint64_t e) { return int(~uint32_t(e)); }

// Of two lanes' entries `apart` apart, the larger to the lower lane or the other way round.
__device__ __forceinline__ uint64_t exchange(uint64_t v, int apart, bool larger) {
  const uint64_t o = __shfl_xor_sync(kAll, v, apart);
  return (v > o) == larger ? v : o;
}
// 32 entries, one a lane, in descending order (bitonic sort).
__device__ __forceinline__ uint64_t sort32(uint64_t v) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int k = 2; k <= 32; k *= 2)
#pragma unroll
    for (int j = k / 2; j > 0; j /= 2) v = exchange(v, j, ((lane & j) == 0) == ((lane & k) == 0));
  return v;
}
// A key that at least n of the lanes' keys reach, the n-th if they differ: the
// largest removed n - 1 times, or for more from the sorted keys.  (4 beams of
// 264: 4.3 us, always sorting 4.5; one removal is two instructions.)
constexpr int kRemove = 16;
__device__ __forceinline__ uint32_t nth_key(uint32_t v, int n) {
  if (n <= kRemove) {
    uint32_t most = __reduce_max_sync(kAll, v);
    for (int i = 1; i < n; ++i) {
      v = v == most ? 0 : v;
      most = __reduce_max_sync(kAll, v);
    }
    return most;
  }
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int k = 2; k <= 32; k *= 2)
#pragma unroll
    for (int j = k / 2; j > 0; j /= 2) {
      const uint32_t o = __shfl_xor_sync(kAll, v, j);
      v = ((lane & j) == 0) == ((lane & k) == 0) ? max(v, o) : min(v, o);
    }
  return __shfl_sync(kAll, v, n - 1);
}
// The best 32 of two sorted lists, sorted.
__device__ __forceinline__ uint64_t merge32(uint64_t a, uint64_t b) {
  const int lane = threadIdx.x % 32;
  const uint64_t r = __shfl_sync(kAll, b, 31 - lane);
  a = a > r ? a : r;
#pragma unroll
  for (int j = 16; j > 0; j /= 2) a = exchange(a, j, (lane & j) == 0);
  return a;
}

// A warp's best entries of what it has seen.
struct Best {
  uint64_t mine = 0; // the lane-th best
  uint64_t bar = 0;  // only entries above it can still matter
  int held = 0;      // entries waiting in the warp's kWaiting places
  bool any = false;  // mine is not empty
  __device__ __forceinline__ void flush(uint64_t *wait, int beams) {
    const int lane = threadIdx.x % 32;
    __syncwarp();
    const uint64_t v = lane < held ? wait[lane] : 0, later = 32 + lane < held ? wait[32 + lane] : 0;
    __syncwarp();
    wait[lane] = later;
    __syncwarp();
    held = max(held - 32, 0);
    mine = any ? merge32(mine, sort32(v)) : sort32(v);
    any = true;
    const uint64_t last = __shfl_sync(kAll, mine, beams - 1);
    bar = bar > last ? bar : last;
  }
  __device__ __forceinline__ void push(uint64_t e, uint64_t *wait, int beams) {
    const unsigned who = __ballot_sync(kAll, e > bar);
    if (!who) return;
    if (e > bar) wait[held + __popc(who & ((1u << (threadIdx.x % 32)) - 1u))] = e;
    held += __popc(who);
    if (held >= 32) flush(wait, beams);
  }
};

// The larger of two, a NaN if either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Streams over tokens [v0, v1) of a row.  kStep values a lane are in flight;
// nine cover the byte vocabulary (264) in one step.  A value costs its
// exponential, a maximum and a comparison; keys are made of the few that pass,
// and only a row's last step checks its end.
constexpr int kStep = 9, kStepValues = 32 * kStep;
template <bool WHOLE, class T>
__device__ __forceinline__ void load_step(T (&to)[kStep], const T *x, int v, int v1) {
  const int at = v + threadIdx.x % 32;
#pragma unroll
  for (int i = 0; i < kStep; ++i) to[i] = x[WHOLE ? at + 32 * i : min(at + 32 * i, v1 - 1)];
}
template <class T> __device__ __forceinline__ void load_step(T (&to)[kStep], const T *x, int v, int v1) {
  if (v1 - v >= kStepValues)
    load_step<true>(to, x, v, v1);
  else // past the end: the last value, which is not used
    load_step<false>(to, x, v, v1);
}
template <class T, int TOGETHER, bool SHARED>
__device__ __forceinline__ void stream_row(const BeamArgs &a, const T *x, int v0, int v1, LogSum &ls, Best &best,
                                           uint64_t *wait, uint32_t *shared_bar) {
  const int lane = threadIdx.x % 32;
  T next[kStep];
  if (v0 < v1) load_step(next, x, v0, v1);
  for (int v = v0; v < v1; v += kStepValues) {
    float logit[kStep], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kStep; ++i) logit[i] = to_f32<T>(next[i]);
    if (a.allowed) {
      uint8_t ok[kStep];
      load_step(ok, a.allowed, v, v1);
#pragma unroll
      for (int i = 0; i < kStep; ++i) logit[i] = ok[i] ? logit[i] : -INFINITY;
    }
    if (v1 - v < kStepValues) {
#pragma unroll
      for (int i = 0; i < kStep; ++i) logit[i] = v + 32 * i + lane < v1 ? logit[i] : -INFINITY;
    }
    if (v + kStepValues < v1) load_step(next, x, v + kStepValues, v1);
#pragma unroll
    for (int i = 0; i < kStep; ++i) top = max_nan(top, logit[i]);
    const uint32_t top_key = key_of(top);
    if (top_key > ls.top) ls.raise(top_key);
    ls.add<TOGETHER>(logit);
    if (v == v0) // of the lanes' largest, the beams-th: at least `beams` values reach it
      best.bar = uint64_t(nth_key(top_key, a.beams)) << 32;
    if constexpr (SHARED) { // `beams` values that another warp of the row has seen reach its bar
      uint32_t key = entry_key(best.bar);
      if (lane == 0) key = max(key, atomicMax(shared_bar, key));
      const uint64_t most = uint64_t(__shfl_sync(kAll, key, 0)) << 32;
      best.bar = best.bar > most ? best.bar : most;
    }
    // A lane's values that may matter, one a round: few do.
    const float bar = fmaxf(logit_of(entry_key(best.bar)), -FLT_MAX);
    uint32_t some = 0;
#pragma unroll
    for (int i = 0; i < kStep; ++i) some |= uint32_t(logit[i] >= bar) << i;
    while (__any_sync(kAll, some != 0)) {
      const int which = __ffs(some) - 1;
      float l = -INFINITY;
#pragma unroll
      for (int i = 0; i < kStep; ++i) l = i == which ? logit[i] : l;
      best.push(entry(key_of(l), v + 32 * which + lane), wait, a.beams);
      some &= some - 1;
    }
  }
  while (best.held) best.flush(wait, a.beams);
}

// A candidate among all of a group's: its total as a number in the same order
// (0: none), and where it stands, beam * 32 + place in the beam's list.
struct Cand {
  uint64_t key = 0;
  uint32_t id = kAll;
};
__device__ __forceinline__ uint64_t key_of_total(double t) {
  const uint64_t u = uint64_t(__double_as_longlong(__dadd_rn(t, 0.0))); // -0 is +0
  return (u >> 63) ? ~u : u | (uint64_t(1) << 63);
}
__device__ __forceinline__ double total_of(uint64_t key) {
  return __longlong_as_double((key >> 63) ? key & ~(uint64_t(1) << 63) : ~key);
}
__device__ __forceinline__ bool before(const Cand &a, const Cand &b) {
  return a.key > b.key || (a.key == b.key && a.id < b.id);
}
// The best 32 of two sorted lists, one entry a lane, sorted.
__device__ __forceinline__ Cand merge_cands(Cand a, const Cand &b) {
  const int lane = threadIdx.x % 32;
  Cand o{__shfl_sync(kAll, b.key, 31 - lane), __shfl_sync(kAll, b.id, 31 - lane)};
  if (before(o, a)) a = o;
#pragma unroll
  for (int j = 16; j > 0; j /= 2) {
    o = {__shfl_xor_sync(kAll, a.key, j), __shfl_xor_sync(kAll, a.id, j)};
    if (before(o, a) == ((lane & j) == 0)) a = o;
  }
  return a;
}

// A warp's part of shared memory: first the entries it holds back (Best), then
// its beam's list.
constexpr int kWaiting = 64;
union WarpShare {
  uint64_t wait[kWaiting];
  struct {
    uint64_t key[32];
    uint32_t id[32];
    int token[32];
  } list;
};

// A beam and what becomes of it: alive (its row counts), finished (one
// candidate of its own) or neither.
struct Beam {
  float score;
  bool finished, exists;
  __device__ __forceinline__ Beam(const BeamArgs &a, long row)
      : score(a.scores[row]), finished(a.finished && a.finished[row]), exists(fabsf(score) < INFINITY) {}
};

// A group's results from its beams' best logits; warp w is beam w, lane its
// place in the list.  Up to kCountBeams beams: every candidate counts those
// before it (W^3 / 32 comparisons a lane).  More: the lists are merged in pairs
// and the first warp's is the answer.  (4 beams: counting 1,090 clocks,
// merging 1,860; 8 beams: 2,450, 2,750; 32 beams: merging 6,500.)
constexpr int kCountBeams = 16;
__device__ __forceinline__ void finish_group(const BeamArgs &a, int group, const Beam &beam, const LogSum &ls,
                                             uint64_t mine, WarpShare *shares) {
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32, W = a.beams;
  Cand c;
  int token = a.pad;
  if (beam.exists && beam.finished) {
    if (lane == 0) c.key = key_of_total(double(beam.score));
  } else if (beam.exists && ls.top != 0 && ls.top < kBadKey) {
    const double lse = __dadd_rn(double(logit_of(ls.top)), log(ls.sum));
    token = entry_token(mine);
    if (lane < W && mine) c.key = key_of_total(__dadd_rn(double(beam.score), __dsub_rn(double(logit_of(entry_key(mine))), lse)));
  }
  if (c.key) c.id = w * 32 + lane;
  auto &list = shares[w].list;
  __syncwarp(); // the share's other use is over
  list.token[lane] = token;
  int *done = reinterpret_cast<int *>(shares + W); // of each beam
  if (lane == 0) done[w] = beam.finished;
  const auto write = [&](int slot, const Cand &best) {
    const long at = long(group) * W + slot;
    if (best.key) {
      const int parent = best.id / 32, chosen = shares[parent].list.token[best.id % 32];
      a.next_scores[at] = float(total_of(best.key));
      a.tokens[at] = chosen;
      a.parents[at] = parent;
      a.next_finished[at] = done[parent] || chosen == a.end;
    } else { // no candidate fills this slot
      a.next_scores[at] = -INFINITY;
      a.tokens[at] = a.pad;
      a.parents[at] = slot;
      a.next_finished[at] = 1;
    }
  };
  if (W <= kCountBeams) {
    // A candidate's slot is the number of candidates before it.  Each of the
    // warp's W is counted by 32 / P lanes.
    list.key[lane] = c.key;
    __syncthreads();
    const int P = W <= 1 ? 1 : 1 << (32 - __clz(W - 1)), p = lane % P;
    const uint64_t key = list.key[p];
    int rank = 0, empty = 0;
    for (int i = lane / P; i < W * W; i += 32 / P) {
      const int o = i / W;
      const uint64_t other = shares[o].list.key[i - o * W];
      rank += other > key || (other == key && i < w * W + p);
      empty += other == 0;
    }
    for (int o = 16; o >= P; o /= 2) rank += __shfl_xor_sync(kAll, rank, o), empty += __shfl_xor_sync(kAll, empty, o);
    if (lane < W && key && rank < W) write(rank, {key, uint32_t(w * 32 + lane)});
    if (w == 0 && lane < W && lane >= W * W - empty) write(lane, Cand());
    return;
  }
  for (int step = 1; step < W; step *= 2) {
    if (w % (2 * step) == step) list.key[lane] = c.key, list.id[lane] = c.id;
    __syncthreads();
    if (w % (2 * step) == 0 && w + step < W) {
      const auto &other = shares[w + step].list;
      c = merge_cands(c, {other.key[lane], other.id[lane]});
    }
  }
  if (w == 0 && lane < W) write(lane, c);
}
size_t share_bytes(int beams) { return beams * (sizeof(WarpShare) + sizeof(int)); }

// One launch: one CTA a group, one warp a beam.
template <class T, int THREADS> __global__ void __launch_bounds__(THREADS) k_beam_rows(BeamArgs a) {
  extern __shared__ uint64_t shared[];
  WarpShare *shares = reinterpret_cast<WarpShare *>(shared);
  const int w = threadIdx.x / 32;
  const long row = long(blockIdx.x) * a.beams + w;
  const Beam beam(a, row);
  LogSum ls;
  Best best;
  if (beam.exists && !beam.finished) {
    stream_row<T, THREADS == 512 ? 9 : 3, false>(a, static_cast<const T *>(a.logits) + row * a.ld, 0, a.vocab, ls, best,
                                                 shares[w].wait, nullptr);
    ls.join_warp();
  }
  finish_group(a, blockIdx.x, beam, ls, best.mine, shares);
}

// Two launches, where there are too few rows for their length: each row in up
// to kSlices slices, one CTA a slice; a slice leaves its sum and its sorted
// best entries in the workspace, and one CTA a group joins them.
constexpr int kSliceWarps = 8, kSlices = 32;

struct Slice {
  double sum;
  uint32_t top;
  uint64_t best[kMaxBeams];
};

// One launch serves short rows, and rows enough to give every SM eight warps
// (one launch / two: 64 rows x 512 8.3 / 12.4 us, x 2000 14.4 / 11.3; 512 rows
// x 2000 16.4 / 18.5, x 5000 31 / 25; 1024 rows x 20000 89 / 66; 2048 rows x
// 5000 39 / 53, x 20000 115 / 121).
__host__ __device__ inline bool in_slices(long rows, int vocab) {
  return rows < 8 * 148 && vocab > (rows < 256 ? 1024 : 2048);
}
__host__ __device__ inline int row_steps(int vocab) { return (vocab + kStepValues - 1) / kStepValues; }
// Slices of a row: so many steps a warp that all CTAs run at once (three an
// SM), and no more slices than these steps fill.
__host__ __device__ inline int slice_count(long rows, int vocab) {
  const int most = rows < 3 * 148 ? int(3 * 148 / rows) : 1, steps = row_steps(vocab);
  const int slots = (most < kSlices ? most : kSlices) * kSliceWarps, each = (steps + slots - 1) / slots;
  return (steps + each * kSliceWarps - 1) / (each * kSliceWarps);
}

template <class T> __global__ void __launch_bounds__(32 * kSliceWarps, 3) k_beam_slice(BeamArgs a, int slices) {
  __shared__ uint64_t wait[kSliceWarps][kWaiting];
  __shared__ double sums[kSliceWarps];
  __shared__ uint32_t tops[kSliceWarps], bar;
  if (threadIdx.x == 0) bar = 0;
  __syncthreads();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long row = blockIdx.x / slices;
  const int slice = blockIdx.x % slices;
  const Beam beam(a, row);
  if (!beam.exists || beam.finished) return; // the row's logits do not count
  // Whole steps to every warp.
  const long part = slice * kSliceWarps + warp, parts = slices * kSliceWarps, steps = row_steps(a.vocab);
  LogSum ls;
  Best best;
  stream_row<T, 9, true>(a, static_cast<const T *>(a.logits) + row * a.ld, int(min(long(a.vocab), part * steps / parts * kStepValues)),
                   int(min(long(a.vocab), (part + 1) * steps / parts * kStepValues)), ls, best, wait[warp], &bar);
  ls.join_warp();
  if (lane == 0) sums[warp] = ls.sum, tops[warp] = ls.top;
  for (int step = 1; step < kSliceWarps; step *= 2) { // the warps' lists, in pairs
    if (warp % (2 * step) == step) wait[warp][lane] = best.mine;
    __syncthreads();
    if (warp % (2 * step) == 0) best.mine = merge32(best.mine, wait[warp + step][lane]);
  }
  if (warp) return;
  LogSum all;
  if (lane < kSliceWarps) all.sum = sums[lane], all.top = tops[lane];
  all.join_warp();
  Slice *out = static_cast<Slice *>(a.work) + blockIdx.x;
  if (lane < a.beams) out->best[lane] = best.mine;
  if (lane == 0) out->sum = all.sum, out->top = all.top;
}

__global__ void __launch_bounds__(1024) k_beam_join(BeamArgs a, int slices) {
  extern __shared__ uint64_t shared[];
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const long row = long(blockIdx.x) * a.beams + w;
  const Beam beam(a, row);
  LogSum ls;
  uint64_t mine = 0;
  if (beam.exists && !beam.finished) {
    const Slice *s = static_cast<const Slice *>(a.work) + row * slices;
    if (lane < slices) ls.top = s[lane].top, ls.sum = s[lane].sum;
    ls.join_warp();
    // The slices' entries one after the other, 32 at a time, four loads in flight.
    const int entries = slices * a.beams;
    for (int i = 0; i < entries; i += 128) {
      uint64_t e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = i + 32 * j + lane, slice = at / a.beams;
        e[j] = at < entries ? s[slice].best[at - slice * a.beams] : 0;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + 32 * j < entries) mine = i + j ? merge32(mine, sort32(e[j])) : sort32(e[j]);
    }
  }
  finish_group(a, blockIdx.x, beam, ls, mine, reinterpret_cast<WarpShare *>(shared));
}

template <class T> void select_typed(const BeamArgs &a, cudaStream_t s) {
  const long rows = long(a.groups) * a.beams;
  if (in_slices(rows, a.vocab)) {
    const int slices = slice_count(rows, a.vocab);
    k_beam_slice<T><<<unsigned(rows * slices), 32 * kSliceWarps, 0, s>>>(a, slices);
    k_beam_join<<<a.groups, 32 * a.beams, share_bytes(a.beams), s>>>(a, slices);
  } else {
    // Up to 16 beams leave a thread the registers to keep its values of a step.
    if (a.beams <= 16)
      k_beam_rows<T, 512><<<a.groups, 32 * a.beams, share_bytes(a.beams), s>>>(a);
    else
      k_beam_rows<T, 1024><<<a.groups, 32 * a.beams, share_bytes(a.beams), s>>>(a);
  }
}

// Reordering: a thread owns U units (of 16, 4, 2 or 1 bytes) of the columns of
// one group's rows.  It reads them of every row that moves before it writes
// any, and no other thread touches these columns: the rows can be permuted, and
// copied to several places, in place and in one pass.  U makes up for few
// beams: about 16 units in flight a thread (2048 x 2 x 11008: one unit 45 us,
// four 31; 256 x 8 x 44032: one 86 us, two 78, the copy rate).
template <class T, int W, int U> __global__ void __launch_bounds__(W == 32 ? 128 : 256) k_state_reorder(ReorderArgs a, long units) {
  __shared__ int from[kMaxBeams];
  constexpr int kMoveThreads = W == 32 ? 128 : 256; // 32 rows: three small CTAs an SM, so that loads and stores overlap
  constexpr int kSpan = kMoveThreads * U;
  const long chunks = (units + kSpan - 1) / kSpan;
  const long group = blockIdx.x / chunks, u0 = blockIdx.x % chunks * kSpan + threadIdx.x;
  if (threadIdx.x < a.beams) {
    const int p = a.parents[group * a.beams + threadIdx.x];
    from[threadIdx.x] = p >= 0 && p < a.beams ? p : int(threadIdx.x);
  }
  __syncthreads();
  char *base = static_cast<char *>(a.states) + group * a.beams * a.ld_bytes + u0 * long(sizeof(T));
  T v[W][U];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w >= a.beams || from[w] == w) continue;
    const char *row = base + from[w] * a.ld_bytes;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (u0 + i * kMoveThreads < units) v[w][i] = *reinterpret_cast<const T *>(row + i * kMoveThreads * sizeof(T));
  }
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w >= a.beams || from[w] == w) continue;
    char *row = base + w * a.ld_bytes;
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (u0 + i * kMoveThreads < units) *reinterpret_cast<T *>(row + i * kMoveThreads * sizeof(T)) = v[w][i];
  }
}

template <class T, int W, int U> void reorder_launch(const ReorderArgs &a, cudaStream_t s) {
  constexpr int kMoveThreads = W == 32 ? 128 : 256;
  const long units = a.row_bytes / long(sizeof(T)), blocks = (units + kMoveThreads * U - 1) / (kMoveThreads * U) * a.groups;
  if (blocks > 0x7FFFFFFFL) throw std::invalid_argument("Too many states to reorder in one call");
  k_state_reorder<T, W, U><<<unsigned(blocks), kMoveThreads, 0, s>>>(a, units);
}

template <class T> void reorder_unit(const ReorderArgs &a, cudaStream_t s) {
  if (a.beams <= 2)
    reorder_launch<T, 2, 8>(a, s);
  else if (a.beams <= 4)
    reorder_launch<T, 4, 4>(a, s);
  else if (a.beams <= 8)
    reorder_launch<T, 8, 2>(a, s);
  else if (a.beams <= 16)
    reorder_launch<T, 16, 1>(a, s);
  else
    reorder_launch<T, 32, 1>(a, s);
}

} // namespace

size_t beam_workspace(int groups, int beams, int vocab) {
  const long rows = long(groups) * beams;
  return in_slices(rows, vocab) ? size_t(rows) * slice_count(rows, vocab) * sizeof(Slice) : 0;
}

void launch_beam_select(const BeamArgs &a, cudaStream_t s) {
  if (a.type == Elem::f32)
    select_typed<float>(a, s);
  else if (a.type == Elem::bf16)
    select_typed<__nv_bfloat16>(a, s);
  else
    select_typed<__half>(a, s);
}

void launch_state_reorder(const ReorderArgs &a, cudaStream_t s) {
  const auto fits = [&](long unit) {
    return reinterpret_cast<uintptr_t>(a.states) % unit == 0 && a.row_bytes % unit == 0 && a.ld_bytes % unit == 0;
  };
  if (fits(16))
    reorder_unit<uint4>(a, s);
  else if (fits(4))
    reorder_unit<uint32_t>(a, s);
  else if (fits(2))
    reorder_unit<uint16_t>(a, s);
  else
    reorder_unit<uint8_t>(a, s);
}

} // namespace ngb
