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
// totals are formed in 64 bits: which beam survives does not depend on how a
// row was split over threads.  Within a beam the order of totals is the order
// of logits, which needs no arithmetic: equal logits go to the lower token,
// equal totals of two beams to the lower beam.
//
// Each row therefore gives a sorted list of its at most `beams` best logits,
// and a candidate's place among all lists is its place in its own list plus,
// for every other list, the number of totals before its own (a binary search).
#include "beam_kernels.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <stdexcept>

namespace ngb {
namespace {

constexpr unsigned kAll = 0xFFFFFFFFu;

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// Logits as unsigned keys in their order; 0 is no candidate (a masked token or
// -inf), kBadKey a value that leaves the row's distribution undefined.
constexpr uint32_t kBadKey = 0xFFFFFFFFu;
__device__ __forceinline__ uint32_t key_of(float x) {
  x = __fadd_rn(x, 0.f); // -0 and +0 are equal logits
  const uint32_t u = __float_as_uint(x);
  if (x == -INFINITY) return 0u;
  if (!(x < INFINITY)) return kBadKey; // +inf or NaN
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = __dadd_rn(v, __shfl_xor_sync(kAll, v, o));
  return v;
}

// One group's lists: entry p of beam w is (total[w][p], token[w][p]), p < count[w].
struct Lists {
  double total[kMaxBeams][kMaxBeams];
  int token[kMaxBeams][kMaxBeams];
  int count[kMaxBeams];
  float score[kMaxBeams];
  int finished[kMaxBeams];
};

// Writes the group's results from its lists; all threads of the CTA, after a
// barrier that makes the lists visible.
__device__ void place(const BeamArgs &a, int group, const Lists &l) {
  const int W = a.beams;
  const long base = long(group) * W;
  int filled = 0;
  for (int w = 0; w < W; ++w) filled += l.count[w];
  for (int i = threadIdx.x; i < W * W; i += blockDim.x) {
    const int w = i / W, p = i % W;
    if (p >= l.count[w]) continue;
    const double mine = l.total[w][p];
    int rank = p;
    for (int o = 0; o < W && rank < W; ++o) {
      if (o == w) continue;
      // Totals of list o before mine: larger ones, and equal ones of a lower beam.
      int lo = 0, hi = l.count[o];
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        const double t = l.total[o][mid];
        if (t > mine || (t == mine && o < w))
          lo = mid + 1;
        else
          hi = mid;
      }
      rank += lo;
    }
    if (rank >= W) continue;
    a.next_scores[base + rank] = float(mine);
    a.tokens[base + rank] = l.token[w][p];
    a.parents[base + rank] = w;
    a.next_finished[base + rank] = l.finished[w] || l.token[w][p] == a.end;
  }
  for (int j = threadIdx.x; j < W; j += blockDim.x) {
    if (j < filled) continue; // slots that no candidate fills
    a.next_scores[base + j] = -INFINITY;
    a.tokens[base + j] = a.pad;
    a.parents[base + j] = j;
    a.next_finished[base + j] = 1;
  }
}

// The list of a beam that needs no logits: none, or a finished beam's own.
// Returns true when the list is done.  One warp.
__device__ bool settled(const BeamArgs &a, Lists &l, int w, long row) {
  const int lane = threadIdx.x % 32;
  const float score = a.scores[row];
  const int finished = a.finished ? a.finished[row] != 0 : 0;
  const bool dead = !(fabsf(score) < INFINITY);
  if (lane == 0) {
    l.score[w] = score;
    l.finished[w] = finished;
    l.count[w] = 0;
    if (finished && !dead) {
      l.total[w][0] = double(score);
      l.token[w][0] = a.pad;
      l.count[w] = 1;
    }
  }
  return finished || dead;
}

// Small vocabularies: one CTA a group, one warp a beam, the row in registers
// (N values a lane; value i of a lane is token 32 i + lane).
constexpr int kSmallVocab = 1024;

template <class T, int N> __global__ void __launch_bounds__(1024) k_beam_small(BeamArgs a) {
  __shared__ Lists l;
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
  const long row = long(blockIdx.x) * a.beams + w;
  if (!settled(a, l, w, row)) {
    const T *x = static_cast<const T *>(a.logits) + row * a.ld;
    uint32_t key[N], best = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int v = 32 * i + lane;
      key[i] = v < a.vocab && (!a.allowed || a.allowed[v]) ? key_of(to_f32<T>(x[v])) : 0u;
      best = max(best, key[i]);
    }
    uint32_t top = __reduce_max_sync(kAll, best);
    if (top != 0 && top != kBadKey) {
      const double m = logit_of(top);
      double sum = 0;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (key[i]) sum = __dadd_rn(sum, exp(__dsub_rn(double(logit_of(key[i])), m)));
      const double lse = __dadd_rn(m, log(warp_sum(sum)));
      const double score = l.score[w];
      int p = 0;
      for (; p < a.beams && top != 0; ++p) {
        // The first token that holds the largest key, then the lane's next best.
        unsigned token = kAll;
#pragma unroll
        for (int i = N - 1; i >= 0; --i)
          if (key[i] == top) token = 32 * i + lane;
        const unsigned first = __reduce_min_sync(kAll, token);
        if (first == token) {
          best = 0;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            if (32 * i + lane == int(first)) key[i] = 0;
            best = max(best, key[i]);
          }
        }
        if (lane == 0) {
          l.total[w][p] = __dadd_rn(score, __dsub_rn(double(logit_of(top)), lse));
          l.token[w][p] = int(first);
        }
        top = __reduce_max_sync(kAll, best);
      }
      if (lane == 0) l.count[w] = p;
    }
  }
  __syncthreads();
  place(a, blockIdx.x, l);
}

// Larger vocabularies: each row in up to kSlices slices, one CTA a slice; a
// slice leaves its largest logit, sum of exponentials and sorted best logits
// in the workspace, and one CTA a group joins them.
constexpr int kSliceThreads = 256, kPerThread = 16, kChunk = kSliceThreads * kPerThread;
constexpr int kSlices = 32;

struct Slice {
  double sum; // of exp(x - largest logit of the slice)
  uint32_t top;
  int count;
  uint64_t best[kMaxBeams]; // key << 32 | ~token: descending, equal keys by token
};

__host__ __device__ inline int slice_count(int vocab) {
  const int chunks = (vocab + kChunk - 1) / kChunk;
  return chunks < kSlices ? chunks : kSlices;
}

template <class T> __global__ void __launch_bounds__(kSliceThreads) k_beam_slice(BeamArgs a) {
  __shared__ uint64_t lead[kSliceThreads];
  __shared__ uint64_t kept[kMaxBeams], pool[kMaxBeams * (kPerThread + 1)];
  __shared__ int pooled;
  __shared__ double sums[kSliceThreads / 32];
  const int slices = slice_count(a.vocab), W = a.beams, tid = threadIdx.x;
  const long row = blockIdx.x / slices;
  const int slice = blockIdx.x % slices;
  Slice *out = static_cast<Slice *>(a.work) + blockIdx.x;
  const float score = a.scores[row];
  if (!(fabsf(score) < INFINITY) || (a.finished && a.finished[row])) return; // the row's logits do not count
  const T *x = static_cast<const T *>(a.logits) + row * a.ld;
  // Whole chunks to every slice, so that slices differ by one chunk at most.
  const long chunks = (long(a.vocab) + kChunk - 1) / kChunk;
  const int c0 = int(slice * chunks / slices), c1 = int((slice + 1) * chunks / slices);
  uint32_t top = 0; // largest key so far, and the sum of exponentials against it
  double sum = 0;
  int held = 0; // entries of kept
  for (int c = c0; c < c1; ++c) {
    uint32_t key[kPerThread];
    uint64_t best = 0;
    const long v0 = long(c) * kChunk + tid;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const long v = v0 + long(i) * kSliceThreads;
      key[i] = v < a.vocab && (!a.allowed || a.allowed[v]) ? key_of(to_f32<T>(x[v])) : 0u;
      const uint64_t k = key[i] ? (uint64_t(key[i]) << 32) | uint32_t(~uint32_t(v)) : 0;
      best = best > k ? best : k;
    }
    __syncthreads(); // the previous chunk's pool has been read
    lead[tid] = best;
    if (tid == 0) pooled = held;
    if (tid < held) pool[tid] = kept[tid];
    __syncthreads();
    // The threshold: the W-th largest of the threads' leaders (distinct, but
    // for 0).  At least W values reach it, and only W threads hold such values.
    int before = 0;
    for (int i = 0; i < kSliceThreads; ++i) before += lead[i] > best;
    if (best != 0 && before < W) {
      // This thread's leader is among the first W: the W-th largest bounds its values.
      // Every value of the thread may be among the best.
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) {
        const long v = v0 + long(i) * kSliceThreads;
        if (key[i]) pool[atomicAdd(&pooled, 1)] = (uint64_t(key[i]) << 32) | uint32_t(~uint32_t(v));
      }
    }
    uint32_t chunk_top = uint32_t(best >> 32);
    chunk_top = __reduce_max_sync(kAll, chunk_top);
    __syncthreads();
    if (tid % 32 == 0) lead[tid / 32] = chunk_top; // every leader has been compared
    // The best W of the pool, sorted: each entry's place is the number before it.
    const int n = pooled;
    for (int i = tid; i < n; i += kSliceThreads) {
      const uint64_t k = pool[i];
      int at = 0;
      for (int j = 0; j < n; ++j) at += pool[j] > k;
      if (at < W) kept[at] = k;
    }
    __syncthreads();
    held = min(n, W);
    uint32_t next = top;
#pragma unroll
    for (int i = 0; i < kSliceThreads / 32; ++i) next = max(next, uint32_t(lead[i]));
    if (next != 0 && next != kBadKey) {
      const double m = logit_of(next);
      if (top != 0 && top != next) sum = __dmul_rn(sum, exp(__dsub_rn(double(logit_of(top)), m)));
#pragma unroll
      for (int i = 0; i < kPerThread; ++i)
        if (key[i]) sum = __dadd_rn(sum, exp(__dsub_rn(double(logit_of(key[i])), m)));
    }
    top = next;
  }
  sum = warp_sum(sum);
  if (tid % 32 == 0) sums[tid / 32] = sum;
  __syncthreads();
  if (tid == 0) {
    for (int i = 1; i < kSliceThreads / 32; ++i) sum = __dadd_rn(sum, sums[i]);
    out->sum = sum;
    out->top = top;
    out->count = held;
  }
  if (tid < held) out->best[tid] = kept[tid];
}

__global__ void __launch_bounds__(1024) k_beam_join(BeamArgs a) {
  __shared__ Lists l;
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32, slices = slice_count(a.vocab);
  const long row = long(blockIdx.x) * a.beams + w;
  if (!settled(a, l, w, row)) {
    // Lane = slice.
    const Slice *s = static_cast<const Slice *>(a.work) + row * slices + lane;
    const uint32_t mine = lane < slices ? s->top : 0u;
    const uint32_t top = __reduce_max_sync(kAll, mine);
    if (top != 0 && top != kBadKey) {
      const double m = logit_of(top);
      const double part = mine ? __dmul_rn(s->sum, exp(__dsub_rn(double(logit_of(mine)), m))) : 0.0;
      const double lse = __dadd_rn(m, log(warp_sum(part)));
      const double score = l.score[w];
      const int count = lane < slices ? s->count : 0;
      int used = 0, p = 0;
      for (; p < a.beams; ++p) {
        const uint64_t head = used < count ? s->best[used] : 0;
        const uint32_t key = __reduce_max_sync(kAll, uint32_t(head >> 32));
        if (key == 0) break;
        const unsigned token = uint32_t(head >> 32) == key ? ~uint32_t(head) : kAll;
        const unsigned first = __reduce_min_sync(kAll, token);
        used += token == first;
        if (lane == 0) {
          l.total[w][p] = __dadd_rn(score, __dsub_rn(double(logit_of(key)), lse));
          l.token[w][p] = int(first);
        }
      }
      if (lane == 0) l.count[w] = p;
    }
  }
  __syncthreads();
  place(a, blockIdx.x, l);
}

template <class T> void select_typed(const BeamArgs &a, cudaStream_t s) {
  if (a.vocab <= kSmallVocab) {
    const dim3 grid(a.groups), block(32 * a.beams);
    if (a.vocab <= 128)
      k_beam_small<T, 4><<<grid, block, 0, s>>>(a);
    else if (a.vocab <= 288)
      k_beam_small<T, 9><<<grid, block, 0, s>>>(a);
    else if (a.vocab <= 512)
      k_beam_small<T, 16><<<grid, block, 0, s>>>(a);
    else
      k_beam_small<T, 32><<<grid, block, 0, s>>>(a);
  } else {
    k_beam_slice<T><<<unsigned(a.groups) * a.beams * slice_count(a.vocab), kSliceThreads, 0, s>>>(a);
    k_beam_join<<<a.groups, 32 * a.beams, 0, s>>>(a);
  }
}

// Reordering: a thread owns one unit (16, 4, 2 or 1 bytes) of the columns of
// one group's rows.  It reads that unit of every row that moves before it
// writes any, and no other thread touches these columns: the rows can be
// permuted, and copied to several places, in place and in one pass.
constexpr int kMoveThreads = 256;

template <class U, int W> __global__ void __launch_bounds__(kMoveThreads) k_state_reorder(ReorderArgs a, long units) {
  __shared__ int from[kMaxBeams];
  const long chunks = (units + kMoveThreads - 1) / kMoveThreads;
  const long group = blockIdx.x / chunks, u = blockIdx.x % chunks * kMoveThreads + threadIdx.x;
  if (threadIdx.x < a.beams) {
    const int p = a.parents[group * a.beams + threadIdx.x];
    from[threadIdx.x] = p >= 0 && p < a.beams ? p : int(threadIdx.x);
  }
  __syncthreads();
  if (u >= units) return;
  char *base = static_cast<char *>(a.states) + group * a.beams * a.ld_bytes + u * long(sizeof(U));
  U v[W];
#pragma unroll
  for (int w = 0; w < W; ++w)
    if (w < a.beams && from[w] != w) v[w] = *reinterpret_cast<const U *>(base + from[w] * a.ld_bytes);
#pragma unroll
  for (int w = 0; w < W; ++w)
    if (w < a.beams && from[w] != w) *reinterpret_cast<U *>(base + w * a.ld_bytes) = v[w];
}

template <class U> void reorder_unit(const ReorderArgs &a, cudaStream_t s) {
  const long units = a.row_bytes / long(sizeof(U)), blocks = (units + kMoveThreads - 1) / kMoveThreads * a.groups;
  if (blocks > 0x7FFFFFFFL) throw std::invalid_argument("Too many states to reorder in one call");
  if (a.beams <= 4)
    k_state_reorder<U, 4><<<unsigned(blocks), kMoveThreads, 0, s>>>(a, units);
  else if (a.beams <= 8)
    k_state_reorder<U, 8><<<unsigned(blocks), kMoveThreads, 0, s>>>(a, units);
  else if (a.beams <= 16)
    k_state_reorder<U, 16><<<unsigned(blocks), kMoveThreads, 0, s>>>(a, units);
  else
    k_state_reorder<U, 32><<<unsigned(blocks), kMoveThreads, 0, s>>>(a, units);
}

} // namespace

size_t beam_workspace(int groups, int beams, int vocab) {
  return vocab <= kSmallVocab ? 0 : size_t(groups) * beams * slice_count(vocab) * sizeof(Slice);
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
