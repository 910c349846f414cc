// Product of two block-scaled 8-bit matrices (block_kernels.h):
//   y[m][n] = sum_b sa[m][b] sw[n / 128][b] d_b[m][n] + bias[n] + c add[m][n],
//   d_b[m][n] = sum_{k in block b} a[m][k] w[n][k].
// The scales change every 128 columns, so no accumulator runs over more than
// one block: each block's sum d_b is formed by the tensor cores in fp32 and
// then added, scaled, into an fp32 register sum.
#include "block_kernels.h"
#include "common.h"
#include "tc_common.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cstdlib>
#include <mutex>

namespace ngb {
namespace {
namespace cg = cooperative_groups;
using namespace tc;

__device__ __forceinline__ void store_elem(void *y, Elem type, long at, float v) {
  if (type == Elem::f32)
    static_cast<float *>(y)[at] = v;
  else if (type == Elem::bf16)
    static_cast<__nv_bfloat16 *>(y)[at] = __float2bfloat16_rn(v);
  else
    static_cast<__half *>(y)[at] = __float2half_rn(v);
}

__device__ __forceinline__ void finish(const BlockMatmulArgs &a, int m, int n, float v) {
  if (a.bias) v = __fadd_rn(v, a.bias[n]);
  if (a.add) v = __fmaf_rn(a.add_scale, a.add[long(m) * a.ldadd + n], v);
  store_elem(a.y, a.type, long(m) * a.ldy + n, v);
}

// Sixteen consecutive bytes of a row from column k, zero past the row's end.
// Rows start on 16-byte boundaries, so a chunk with one valid byte can be read.
__device__ __forceinline__ uint4 load16(const uint8_t *row, int k, int cols) {
  if (k >= cols) return make_uint4(0, 0, 0, 0);
  uint4 u = __ldg(reinterpret_cast<const uint4 *>(row + k));
  const int left = cols - k;
  if (left < 16) {
    uint32_t *w = reinterpret_cast<uint32_t *>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int bytes = left - 4 * i;
      w[i] &= bytes >= 4 ? 0xFFFFFFFFu : bytes <= 0 ? 0u : (1u << (8 * bytes)) - 1u;
    }
  }
  return u;
}

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
               "{%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Few rows of a (a single token's projection): bound by the weights' bytes.
// CTA: 16 weight rows x 8 rows of a, the blocks along k dealt to 8 warps, whose
// sums meet in shared memory in warp order.  Weights are the matrix
// instruction's 16-row side.  A sum over k does not mind its order, so each
// lane takes 16 consecutive bytes of its row (one load) and feeds them to two
// instructions as if they were that instruction's own columns; both operands
// are permuted alike.
constexpr int kVecWarps = 8;

__global__ void __launch_bounds__(32 * kVecWarps) k_block_vec(BlockMatmulArgs a) {
  __shared__ float part[kVecWarps][16 * 8];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 8;
  const int kb = (a.k + kScaleBlock - 1) / kScaleBlock;
  const int na = min(n0 + g, a.n - 1), nb = min(n0 + g + 8, a.n - 1), mg = m0 + g;
  const uint8_t *wa = a.w + long(na) * a.ldw, *wb = a.w + long(nb) * a.ldw;
  const uint8_t *ar = a.a + long(min(mg, a.m - 1)) * a.lda;
  const int mc0 = min(m0 + 2 * t, a.m - 1), mc1 = min(m0 + 2 * t + 1, a.m - 1); // the result's columns of this lane
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  for (int b = warp; b < kb; b += kVecWarps) {
    float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = b * kScaleBlock + h * 64 + t * 16;
      const uint4 x = load16(wa, k, a.k), y = load16(wb, k, a.k), z = load16(ar, k, a.k);
      mma_e4m3(d, x.x, y.x, x.y, y.y, z.x, z.y);
      mma_e4m3(d, x.z, y.z, x.w, y.w, z.z, z.w);
    }
    const float sw = a.w_scale[long(n0 / kScaleBlock) * kb + b];
    const float s0 = __fmul_rn(sw, a.a_scale[long(mc0) * kb + b]), s1 = __fmul_rn(sw, a.a_scale[long(mc1) * kb + b]);
    sum[0] = __fmaf_rn(s0, d[0], sum[0]);
    sum[1] = __fmaf_rn(s1, d[1], sum[1]);
    sum[2] = __fmaf_rn(s0, d[2], sum[2]);
    sum[3] = __fmaf_rn(s1, d[3], sum[3]);
  }
  float *mine = part[warp];
  mine[(2 * t) * 16 + g] = sum[0];
  mine[(2 * t + 1) * 16 + g] = sum[1];
  mine[(2 * t) * 16 + g + 8] = sum[2];
  mine[(2 * t + 1) * 16 + g + 8] = sum[3];
  __syncthreads();
  if (threadIdx.x < 128) {
    const int n = n0 + threadIdx.x % 16, m = m0 + threadIdx.x / 16;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kVecWarps; ++i) v = __fadd_rn(v, part[i][threadIdx.x]);
    if (n < a.n && m < a.m) finish(a, m, n, v);
  }
}

// More rows: the tensor cores proper.  A tile is 128 weight rows (TMEM lanes)
// x TN rows of a (TMEM columns).  One thread streams the blocks of 128 bytes
// along k by TMA (SWIZZLE_128B, one swizzle atom a row), one issues each
// block's four MMAs (M=128, N=TN, K=32) into a TMEM accumulator of its own (a
// ring of them), and 4 or 8 warps add the finished accumulators, scaled, to
// the sums in their registers: a thread holds one weight row, whose scale is
// the tile's, and up to 128 columns, whose scales (times the weights') it
// reads from shared memory four at a time.  Adding is a packed fma a pair.
//
// The CTAs either walk over the tiles (splits = 1), or, where the tiles are
// too few to fill the GPU, `splits` CTAs of a cluster share a tile's k range:
// each leaves its sums in shared memory and adds up a slice of the columns
// over all of them, in rank order.
//
// Every wait is bounded.  One that runs out sets *err; its role stops, waits
// (bounded) for its own copies or MMAs in flight, and the CTA frees its TMEM.
constexpr int kTileN = 128;       // weight rows of a tile
constexpr int kScaleChunk = 32;   // blocks along k whose scales are staged at a time
constexpr long long kWaitClocks = 2000000000LL; // about a second
constexpr uint32_t kTileWBytes = kTileN * kScaleBlock;

template <int TN> struct TcShape {
  static constexpr int kGroups = TN > 128 ? TN / 128 : 1; // of four epilogue warps
  static constexpr int kCols = TN / kGroups;              // columns a group adds up
  // Two groups need more registers than 384 threads' even share: the groups
  // raise their limit to kMoreRegs a thread, the four other warps (two of them
  // idle) drop theirs; 256 * 208 + 128 * 80 <= 384 * 168 at launch.
  static constexpr bool kShift = kGroups == 2;
  static constexpr int kMoreRegs = 208, kFewerRegs = 80;
  static constexpr int kEpilogue = 128 * kGroups, kThreads = kEpilogue + (kShift ? 128 : 64);
  static constexpr uint32_t kStageBytes = kTileWBytes + TN * kScaleBlock;
  // More than half an SM's shared memory: one CTA an SM, so that a CTA never
  // waits for another's TMEM while its cluster waits for it.
  static constexpr int kStages = TN == 256 ? 4 : TN == 128 ? 6 : 8;
  static constexpr int kAccs = TN == 256 ? 2 : 4, kTmemCols = kAccs * TN;
  static constexpr int kScaleLd = TN + 4; // rows of 16 bytes, spread over the banks
  static constexpr size_t kBars = 2 * kStages + 2 * kAccs + 1;
  static constexpr size_t kSmem =
      1024 + kStages * size_t(kStageBytes) + kScaleChunk * kScaleLd * 4 + kBars * 8 + 16;
  static_assert(kSmem <= 232448, "shared memory");
  static_assert(size_t(kTileN) * TN * 4 <= kStages * size_t(kStageBytes), "partial sums lie over the stages");
};

// Instruction descriptor, kind::f8f6f4: D f32 (bits 4-5 = 1), A and B e4m3
// (bits 7-9, 10-12 = 0), both K-major (bits 15, 16 = 0), N >> 3 at bits
// 17-22, M >> 4 at bits 24-28.
template <int TN> constexpr uint32_t kIdesc = (1u << 4) | (uint32_t(TN >> 3) << 17) | (uint32_t(kTileN >> 4) << 24);

template <int TN>
__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\t"
               "setp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d_tmem), "l"(a), "l"(b), "r"(kIdesc<TN>), "r"(accumulate)
               : "memory");
}

// sum += d * scale, two columns at a time.
__device__ __forceinline__ void fma2(uint64_t &sum, float d0, float d1, float s0, float s1) {
  uint64_t d, s;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(d0), "f"(d1));
  asm("mov.b64 %0, {%1, %2};" : "=l"(s) : "f"(s0), "f"(s1));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sum) : "l"(d), "l"(s));
}
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}

__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile int *abort_s) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try(bar, parity)) {
    if (*abort_s) return false;
    if (clock64() - t0 > kWaitClocks) {
      *abort_s = 1;
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void group_sync(int group) {
  asm volatile("bar.sync %0, 128;" ::"r"(group + 1) : "memory");
}

template <class Y> __device__ __forceinline__ Y from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// One weight row's sums of kCols consecutive columns (rows m0.. of the result).
template <class Y, int kCols>
__device__ __forceinline__ void store_sums(const BlockMatmulArgs &a, int m0, int n, const uint64_t (&sum)[kCols / 2]) {
  if (n >= a.n) return;
  const float bias = a.bias ? a.bias[n] : 0.f;
  Y *y = static_cast<Y *>(a.y) + long(m0) * a.ldy + n;
  const float *add = a.add ? a.add + long(m0) * a.ldadd + n : nullptr;
#pragma unroll
  for (int j = 0; j < kCols; j += 8) {
    float v[8], e[8];
#pragma unroll
    for (int i = 0; i < 8; i += 2) unpack2(sum[(j + i) / 2], v[i], v[i + 1]);
    if (add) {
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = m0 + j + i < a.m ? add[long(j + i) * a.ldadd] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = __fadd_rn(v[i], bias);
      if (add) v[i] = __fmaf_rn(a.add_scale, e[i], v[i]);
      if (m0 + j + i < a.m) y[long(j + i) * a.ldy] = from_f32<Y>(v[i]);
    }
  }
}

template <int TN>
__global__ void __launch_bounds__(TcShape<TN>::kThreads, 1)
    k_block_tc(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, BlockMatmulArgs a,
               int splits, int tiles_n, int tiles, int *err, int stall_test) {
  using S = TcShape<TN>;
  extern __shared__ uint8_t smem_raw[];
  // 128-byte swizzled tiles start on 1024-byte boundaries of the shared window.
  uint8_t *stages = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u); // [kStages][weights, a]
  float *scales = reinterpret_cast<float *>(stages + S::kStages * size_t(S::kStageBytes)); // [kScaleChunk][kScaleLd]
  uint64_t *bars = reinterpret_cast<uint64_t *>(scales + kScaleChunk * S::kScaleLd);
  volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(bars + S::kBars);
  volatile int *abort_s = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int kb = (a.k + kScaleBlock - 1) / kScaleBlock;
  const int z = blockIdx.x % splits, first = blockIdx.x / splits, stride = gridDim.x / splits;
  const int kb0 = int(long(z) * kb / splits), kb1 = int(long(z + 1) * kb / splits);
  // full[stage], empty[stage]: a stage holds its block / has been read by its
  // MMAs; ready[acc], taken[acc]: an accumulator holds its block's sum / has
  // been added up.
  const uint32_t full = smem_u32(bars), empty = full + 8 * S::kStages, ready = empty + 8 * S::kStages,
                 taken = ready + 8 * S::kAccs, done = taken + 8 * S::kAccs;

  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
    for (int i = 0; i < S::kAccs; ++i) mbar_init(ready + 8 * i, 1), mbar_init(taken + 8 * i, 4 * S::kGroups);
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *abort_s = stall_test; // test switch: the path of a wait that ran out, with nothing in flight
  }
  if (warp == S::kEpilogue / 32 + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(const_cast<uint32_t *>(tmem_slot))),
                 "r"(S::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  const bool stalled = *abort_s != 0;

  uint64_t sum[S::kCols / 2];
  const int group = warp / 4, row = tid % 128;
  if (warp < S::kEpilogue / 32) {
    if constexpr (S::kShift) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kMoreRegs));
    bool alive = !stalled;
    int it = 0; // accumulators taken so far
    float *mine = scales + group * S::kCols;
    for (int tile = first; tile < tiles; tile += stride) {
      const int n0 = tile % tiles_n * kTileN, m0 = tile / tiles_n * TN + group * S::kCols;
#pragma unroll
      for (int j = 0; j < S::kCols / 2; ++j) sum[j] = 0;
      for (int c = kb0; c < kb1; c += kScaleChunk) {
        // The scales of this chunk: lane = block along k, each warp a quarter of the columns.
        group_sync(group); // the previous ones have been read
        const int b = c + lane;
        const float sw = b < kb1 ? a.w_scale[long(n0 / kScaleBlock) * kb + b] : 0.f;
#pragma unroll 8
        for (int j = warp % 4 * (S::kCols / 4); j < (warp % 4 + 1) * (S::kCols / 4); ++j)
          mine[lane * S::kScaleLd + j] =
              b < kb1 && m0 + j < a.m ? __fmul_rn(sw, a.a_scale[long(m0 + j) * kb + b]) : 0.f;
        group_sync(group);
        for (int b1 = c; b1 < min(c + kScaleChunk, kb1); ++b1, ++it) {
          const int acc = it % S::kAccs;
          if (alive) alive = __all_sync(0xFFFFFFFFu, wait_bar(ready + 8 * acc, (it / S::kAccs) & 1, abort_s));
          if (!alive) continue; // the barriers above are still met
          fence_after();
          const uint32_t from = tmem + (uint32_t(warp % 4 * 32) << 16) + acc * TN + group * S::kCols;
          const float4 *s4 = reinterpret_cast<const float4 *>(mine + (b1 - c) * S::kScaleLd);
#pragma unroll
          for (int j = 0; j < S::kCols; j += 32) {
            float d[32];
            tmem_ld32(from + j, d);
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const float4 s = s4[(j + i) / 4];
              fma2(sum[(j + i) / 2], d[i], d[i + 1], s.x, s.y);
              fma2(sum[(j + i) / 2 + 1], d[i + 2], d[i + 3], s.z, s.w);
            }
          }
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(taken + 8 * acc);
        }
      }
      if (splits == 1 && alive) {
        if (a.type == Elem::f32)
          store_sums<float, S::kCols>(a, m0, n0 + row, sum);
        else if (a.type == Elem::bf16)
          store_sums<__nv_bfloat16, S::kCols>(a, m0, n0 + row, sum);
        else
          store_sums<__half, S::kCols>(a, m0, n0 + row, sum);
      }
    }
    if (splits > 1 && alive) {
      // Every accumulator was ready, so every copy and MMA is done with the stages.
      float *part = reinterpret_cast<float *>(stages) + group * S::kCols * kTileN;
#pragma unroll
      for (int j = 0; j < S::kCols; j += 2) {
        float x, y;
        unpack2(sum[j / 2], x, y);
        part[j * kTileN + row] = x;
        part[(j + 1) * kTileN + row] = y;
      }
    }
  } else {
    if constexpr (S::kShift) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kFewerRegs));
    if (warp == S::kEpilogue / 32 && lane == 0 && !stalled) { // copies
      bool ok = true;
      int it = 0;
      for (int tile = first; tile < tiles && ok; tile += stride) {
        const int n0 = tile % tiles_n * kTileN, m0 = tile / tiles_n * TN;
        for (int b = kb0; b < kb1; ++b, ++it) {
          const int st = it % S::kStages;
          if (it >= S::kStages) ok = wait_bar(empty + 8 * st, (it / S::kStages - 1) & 1, abort_s);
          if (!ok) break;
          const uint32_t dst = smem_u32(stages + st * size_t(S::kStageBytes));
          mbar_expect(full + 8 * st, S::kStageBytes);
          tma_load_2d(dst, &tm_w, b * kScaleBlock, n0, full + 8 * st);
          tma_load_2d(dst + kTileWBytes, &tm_a, b * kScaleBlock, m0, full + 8 * st);
        }
      }
      // Copies in flight when a wait ran out, here or in another role.
      int none = 0;
      for (int i = max(0, it - S::kStages); i < it; ++i)
        wait_bar(full + 8 * (i % S::kStages), (i / S::kStages) & 1, &none);
    }
    if (warp == S::kEpilogue / 32 + 1 && lane == 0 && !stalled) { // MMAs
      bool ok = true;
      int it = 0;
      for (int tile = first; tile < tiles && ok; tile += stride) {
        for (int b = kb0; b < kb1; ++b, ++it) {
          const int st = it % S::kStages, acc = it % S::kAccs;
          if (it >= S::kAccs) ok = wait_bar(taken + 8 * acc, (it / S::kAccs - 1) & 1, abort_s);
          ok = ok && wait_bar(full + 8 * st, (it / S::kStages) & 1, abort_s);
          if (!ok) break;
          fence_after();
          const uint32_t w = smem_u32(stages + st * size_t(S::kStageBytes)), x = w + kTileWBytes;
#pragma unroll
          for (int j = 0; j < kScaleBlock / 32; ++j)
            mma_f8<TN>(tmem + acc * TN, sw128_desc(w + 32 * j), sw128_desc(x + 32 * j), j > 0);
          mma_commit(empty + 8 * st);
          mma_commit(ready + 8 * acc);
        }
      }
      mma_commit(done); // arrives once every MMA above has completed
      int none = 0;
      wait_bar(done, 0, &none);
    }
  }
  fence_before();
  __syncthreads();
  const bool failed = *abort_s != 0;
  if (failed && tid == 0) *reinterpret_cast<volatile int *>(err) = 1;
  if (splits > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync(); // every CTA's sums are visible
    if (!failed && tid < kTileN) {
      const int tile = first, n = tile % tiles_n * kTileN + tid, m0 = tile / tiles_n * TN;
      const float *part = reinterpret_cast<const float *>(stages);
      const int j0 = z * TN / splits, j1 = (z + 1) * TN / splits;
      for (int j = j0; j < j1; ++j) {
        float v = 0.f;
        for (int s = 0; s < splits; ++s) v = __fadd_rn(v, cluster.map_shared_rank(part, s)[j * kTileN + tid]);
        if (n < a.n && m0 + j < a.m) finish(a, m0 + j, n, v);
      }
    }
    cluster.sync(); // every CTA has read the others' sums
  }
  if (warp == S::kEpilogue / 32 + 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kTmemCols) : "memory");
  }
}

// An 8-bit matrix as TMA boxes of 128 columns x box_rows rows, 128-byte
// swizzle, zeros out of range.
bool make_map(CUtensorMap *m, const uint8_t *p, long rows, long cols, long ld, int box_rows) {
  const EncodeTiled enc = encode_tiled();
  if (!enc) return false;
  const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(ld)};
  const cuuint32_t box[2] = {cuuint32_t(kScaleBlock), cuuint32_t(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(p), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Per device: kernel attributes, SM count and the error word (pinned, mapped),
// set up at the first call.
constexpr int kMaxDevices = 64;
struct DeviceSetup {
  std::once_flag once;
  std::atomic<int *> err{nullptr};
  int *err_dev = nullptr;
  int sms = 0;
} g_setup[kMaxDevices];

template <int TN> void configure() {
  NGB_CUDA(cudaFuncSetAttribute(k_block_tc<TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(TcShape<TN>::kSmem)));
}

DeviceSetup &setup() {
  int device = 0;
  NGB_CUDA(cudaGetDevice(&device));
  if (device >= kMaxDevices) throw std::runtime_error("CUDA device index out of range");
  DeviceSetup &d = g_setup[device];
  std::call_once(d.once, [&] {
    configure<32>();
    configure<64>();
    configure<128>();
    configure<256>();
    cudaFuncAttributes fa;
    NGB_CUDA(cudaFuncGetAttributes(&fa, k_block_vec)); // loads the kernel
    NGB_CUDA(cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, device));
    int *host = nullptr;
    NGB_CUDA(cudaHostAlloc(reinterpret_cast<void **>(&host), sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable));
    *host = 0;
    NGB_CUDA(cudaHostGetDevicePointer(reinterpret_cast<void **>(&d.err_dev), host, 0));
    d.err = host;
  });
  return d;
}

// Test switch NEUROGEN_TEST_MATMUL_STALL=k: the first k tensor-core products of
// the process take the path of a wait that ran out before anything is issued.
int take_stall() {
  static std::atomic<int> left{[] {
    const char *e = std::getenv("NEUROGEN_TEST_MATMUL_STALL");
    return e ? std::atoi(e) : 0;
  }()};
  int k = left.load();
  while (k > 0 && !left.compare_exchange_weak(k, k - 1)) {
  }
  return k > 0 ? 1 : 0;
}

template <int TN> void launch_tc(const BlockMatmulArgs &a, int splits, DeviceSetup &d, cudaStream_t s) {
  CUtensorMap tm_w, tm_a;
  if (!make_map(&tm_w, a.w, a.n, a.k, a.ldw, kTileN) || !make_map(&tm_a, a.a, a.m, a.k, a.lda, TN))
    throw std::runtime_error("Cannot describe an 8-bit matrix to the copy engine");
  const int tiles_n = (a.n + kTileN - 1) / kTileN, tiles = tiles_n * ((a.m + TN - 1) / TN);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits == 1 ? std::min(tiles, d.sms) : tiles * splits);
  cfg.blockDim = dim3(TcShape<TN>::kThreads);
  cfg.dynamicSmemBytes = TcShape<TN>::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 1 : 0;
  NGB_CUDA(cudaLaunchKernelEx(&cfg, k_block_tc<TN>, tm_w, tm_a, a, splits, tiles_n, tiles, d.err_dev, take_stall()));
}

// Tile width and k split: the shape with the least estimated time.  A CTA's
// time is its blocks, each bound by the larger of its MMAs and its bytes from
// L2, plus a start; a split adds its exchange.
struct Plan {
  int tn, splits;
};
Plan plan(const BlockMatmulArgs &a, int sms) {
  const long kb = (a.k + kScaleBlock - 1) / kScaleBlock, tiles_n = (a.n + kTileN - 1) / kTileN;
  Plan best{128, 1};
  double least = 1e30;
  for (int tn : {32, 64, 128, 256}) {
    const long tiles = tiles_n * ((a.m + tn - 1) / tn);
    const double block = std::max(2.0 * tn, (kTileWBytes + tn * 128) / 80.0);
    for (int splits : {1, 2, 4, 8}) {
      if (splits > 1 && (splits > kb || tn > 128 || tiles * splits > sms)) continue;
      const long waves = (tiles * splits + sms - 1) / sms;
      const double t = 2500 + double(waves) * ((kb + splits - 1) / splits * block + 3.0 * tn) + (splits > 1 ? 1500 + 4.0 * tn : 0);
      if (t < least) least = t, best = {tn, splits};
    }
  }
  return best;
}

} // namespace

void check_block_matmul_errors(int device) {
  if (device < 0 || device >= kMaxDevices) return;
  int *err = g_setup[device].err;
  if (err && *reinterpret_cast<volatile int *>(err)) {
    *reinterpret_cast<volatile int *>(err) = 0;
    throw std::runtime_error("An 8-bit product timed out waiting for its tensor-core pipeline");
  }
}

void launch_block_matmul(const BlockMatmulArgs &a, cudaStream_t s) {
  DeviceSetup &d = setup();
  // Few rows are bound by the weights' bytes, and by latency.
  if (a.m <= 16) {
    const dim3 grid((a.n + 15) / 16, (a.m + 7) / 8);
    k_block_vec<<<grid, 32 * kVecWarps, 0, s>>>(a);
    return;
  }
  const Plan p = plan(a, d.sms);
  if (p.tn == 32)
    launch_tc<32>(a, p.splits, d, s);
  else if (p.tn == 64)
    launch_tc<64>(a, p.splits, d, s);
  else if (p.tn == 128)
    launch_tc<128>(a, p.splits, d, s);
  else
    launch_tc<256>(a, p.splits, d, s);
}

} // namespace ngb
