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
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <memory>
#include <mutex>
#include <type_traits>

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

// A block's sum d counts sa sw d.  d is 0 or lies between 2^-18 and 2^25, so
// that can be an ordinary number where s = sa sw overflows or is subnormal
// (bytes that use little of their range, values near fp32's ends).  There d
// first takes a power of two p = 2^100 or 2^-100, exactly, and s = sa sw / p
// rounds as a normal number: where even that leaves the range, the result is
// an infinity (or 0, for d = 0) or rounds to nothing.
struct ScalePair {
  float s, p;
};
__device__ __forceinline__ bool is_normal(float v) { // neither 0 nor subnormal nor infinite nor NaN
  return 2 * __float_as_uint(v) - (1u << 24) < (254u << 24);
}
__device__ __forceinline__ ScalePair scale_pair(float sa, float sw) {
  const float s = __fmul_rn(sa, sw);
  const auto counts = [](float v) { return v != 0.f && fabsf(v) <= FLT_MAX; };
  if (is_normal(s) || !counts(sa) || !counts(sw)) return {s, 1.f};
  const bool large = fabsf(s) > 1.f;
  const float half = large ? 0x1p-50f : 0x1p50f; // exact on both: neither is far on the other side
  const float rest = __fmul_rn(__fmul_rn(sa, half), __fmul_rn(sw, half));
  return {fminf(fmaxf(rest, -FLT_MAX), FLT_MAX), large ? 0x1p100f : 0x1p-100f};
}

// Outside 2^-63 .. 2^63: two scales within have a normal product.
__device__ __forceinline__ bool is_far(float v) {
  return (__float_as_uint(v) & 0x7FFFFFFFu) - (64u << 23) > (126u << 23);
}

// Sixteen consecutive bytes of a row from column k, zero past the row's end.
// Rows start on 16-byte boundaries, so a chunk with one valid byte can be read
// whole: it lies in one aligned word, which no allocation ends within.
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

// Few rows of a (a single token's projection): bound by the weights' bytes, and
// by latency where those are few.  CTA: 16 weight rows x 8 NT rows of a, the
// blocks along k dealt to 8 warps, whose sums meet in shared memory in warp
// order.  Weights are the matrix instruction's 16-row side.  A sum over k does
// not mind its order, so each lane takes 16 consecutive bytes of its row (one
// load) and feeds them to two instructions as if they were that instruction's
// own columns; both operands are permuted alike.  A warp's loads of AHEAD
// blocks are in flight together, and CTAS CTAs share an SM.
constexpr int kVecWarps = 8;

template <int NT> struct VecBlock {
  uint4 w[2][2], a[NT][2]; // [row or row + 8][half of the block], [8 rows of a][half]
  float sw, sa[NT][2];
};

template <int NT, int AHEAD, int CTAS>
__global__ void __launch_bounds__(32 * kVecWarps, CTAS) k_block_vec(BlockMatmulArgs a, int tiles_n) {
  __shared__ float part[kVecWarps][NT][8][16];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, t = lane % 4;
  const int n0 = blockIdx.x % tiles_n * 16, m0 = blockIdx.x / tiles_n * 8 * NT;
  const int kb = (a.k + kScaleBlock - 1) / kScaleBlock;
  const uint8_t *wa = a.w + long(min(n0 + g, a.n - 1)) * a.ldw, *wb = a.w + long(min(n0 + g + 8, a.n - 1)) * a.ldw;
  const float *sw = a.w_scale + long(n0 / kScaleBlock) * kb;
  const uint8_t *ar[NT];
  const float *sa[NT][2]; // of the result's columns of this lane
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    ar[i] = a.a + long(min(m0 + 8 * i + g, a.m - 1)) * a.lda;
    sa[i][0] = a.a_scale + long(min(m0 + 8 * i + 2 * t, a.m - 1)) * kb;
    sa[i][1] = a.a_scale + long(min(m0 + 8 * i + 2 * t + 1, a.m - 1)) * kb;
  }
  float sum[NT][4] = {};
  for (int b0 = warp; b0 < kb; b0 += kVecWarps * AHEAD) {
    VecBlock<NT> v[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int b = b0 + u * kVecWarps;
      if (b >= kb) continue;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = b * kScaleBlock + h * 64 + t * 16;
        v[u].w[0][h] = load16(wa, k, a.k);
        v[u].w[1][h] = load16(wb, k, a.k);
#pragma unroll
        for (int i = 0; i < NT; ++i) v[u].a[i][h] = load16(ar[i], k, a.k);
      }
      v[u].sw = sw[b];
#pragma unroll
      for (int i = 0; i < NT; ++i) v[u].sa[i][0] = sa[i][0][b], v[u].sa[i][1] = sa[i][1][b];
    }
    bool odd = false; // some scale product here needs two factors (ScalePair)
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (b0 + u * kVecWarps >= kb) continue;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) odd |= !is_normal(__fmul_rn(v[u].sa[i][j], v[u].sw));
    }
    const auto blocks = [&](auto split) {
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (b0 + u * kVecWarps >= kb) continue;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 x = v[u].w[0][h], y = v[u].w[1][h], z = v[u].a[i][h];
            mma_e4m3(d, x.x, y.x, x.y, y.y, z.x, z.y);
            mma_e4m3(d, x.z, y.z, x.w, y.w, z.z, z.w);
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float s = __fmul_rn(v[u].sa[i][j], v[u].sw);
            if constexpr (split.value) {
              const ScalePair f = scale_pair(v[u].sa[i][j], v[u].sw);
              s = f.s, d[j] = __fmul_rn(f.p, d[j]), d[j + 2] = __fmul_rn(f.p, d[j + 2]);
            }
            sum[i][j] = __fmaf_rn(s, d[j], sum[i][j]);
            sum[i][j + 2] = __fmaf_rn(s, d[j + 2], sum[i][j + 2]);
          }
        }
      }
    };
    if (__any_sync(0xFFFFFFFFu, odd))
      blocks(std::true_type());
    else
      blocks(std::false_type());
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    part[warp][i][2 * t][g] = sum[i][0];
    part[warp][i][2 * t + 1][g] = sum[i][1];
    part[warp][i][2 * t][g + 8] = sum[i][2];
    part[warp][i][2 * t + 1][g + 8] = sum[i][3];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 128 * NT; e += 32 * kVecWarps) {
    const int n = n0 + e % 16, m = m0 + e / 16;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < kVecWarps; ++i) v = __fadd_rn(v, (&part[i][0][0][0])[e]);
    if (n < a.n && m < a.m) finish(a, m, n, v);
  }
}

// More rows: the tensor cores proper.  A tile is 128 rows of a (TMEM lanes) x
// TN weight rows (TMEM columns).  One thread streams the blocks of 128 bytes
// along k by TMA (SWIZZLE_128B, one swizzle atom a row), one issues each
// block's four MMAs (M=128, N=TN, K=32) into a TMEM accumulator of its own,
// two warps stage the rows' scales, and 4 or 8 warps add the finished
// accumulators, scaled, to the sums in their registers.  TN divides 128 or is
// 256 in two halves, so a warp's columns share one weight scale and a thread's
// row one scale of a: a block's addition is one packed fma a pair of columns
// and nothing else.  A warp reads 64 columns at a time and gives a set back
// before it adds the last of them.
//
// What holds large products is the accumulators' way out: while MMAs run, one
// of 128 x 256 is in registers some 700 clocks after it is ready, and its own
// MMAs take 541 (8192 x 8192 x 4096: 251 us, tensor pipe 55%).  The 700 are
// two loads of 64 columns a warp, the second issued as the first is added: the
// marks do not tell TMEM's bandwidth from two of its latencies.  Pairs of CTAs on one tile (cta_group::2)
// halve the weights' copies and not that, and hand back over the cluster, 500
// clocks later: 512 us.
//
// The roles meet (mbarriers) once for kPair blocks: a meeting costs the MMAs'
// thread some 400 clocks, more than a block's MMAs take when TN is small
// (512 x 768 x 3200, TN = 32: one block a meeting 10.8 us, two 9.2 us).
//
// The CTAs either walk over the tiles (splits = 1), or, where the tiles are
// too few to fill the GPU, `splits` CTAs of a cluster share a tile's k range:
// each owns a slice of the rows, all send it their sums of these rows
// (distributed shared memory), and it adds them up in rank order.
//
// Every wait on an mbarrier is bounded.  One that runs out sets *err; its role
// stops, waits (bounded) for its own copies or MMAs in flight, and the CTA
// frees its TMEM and fills its part of the result with NaN.  The cluster's
// barriers and the TMEM allocation have no limit of their own and need none:
// every role of every CTA reaches each barrier, whether its waits ran out or
// not, and TMEM is held only by CTAs that run to their end without this one
// (of a cluster of this kernel an SM holds one CTA, so none waits for another's).
constexpr int kTileM = 128;       // rows of a in a tile
constexpr int kMaxSplits = 8;
constexpr int kScaleChunk = 16;   // blocks along k whose scales are staged at a time (two such buffers)
constexpr long long kWaitClocks = 2000000000LL; // about a second
constexpr uint32_t kTileABytes = kTileM * kScaleBlock;

template <int TN> struct TcShape {
  static constexpr int kGroups = TN > 128 ? TN / 128 : 1; // of four epilogue warps
  static constexpr int kCols = TN / kGroups;              // columns a group adds up
  // Epilogue warps, then one warp of copies, one of MMAs and two of scales.
  static constexpr int kEpilogue = 128 * kGroups, kThreads = kEpilogue + 128;
  static constexpr int kPair = TN == 256 ? 1 : 2; // blocks a stage and a set of accumulators hold
  static constexpr uint32_t kBlockBytes = kTileABytes + TN * kScaleBlock, kStageBytes = kPair * kBlockBytes;
  // More than half an SM's shared memory: one CTA an SM, so that a CTA never
  // waits for another's TMEM while its cluster waits for it.
  static constexpr int kStages = TN == 256 ? 4 : 3;
  static constexpr int kAccs = TN == 32 ? 4 : 2, kTmemCols = kAccs * kPair * TN; // sets of accumulators
  static constexpr size_t kBars = 2 * kStages + 2 * kAccs + 4 + 1;
  static constexpr size_t kScaleFloats = 2 * kScaleChunk * (kTileM + kGroups);
  static constexpr size_t kSwap = 4 * kGroups * 32 * 64; // 64 bytes of each row of a warp, on their way out
  // A split's sums of the rows a CTA owns: [splits][TN / 4][rows + 1] of 16
  // bytes (narrow tiles only: with 128 columns or more there are no splits).
  static constexpr size_t kPart = TN >= 128 ? 0 : TN * 4 * size_t(kTileM + kMaxSplits);
  static constexpr size_t kSmem =
      1024 + kStages * size_t(kStageBytes) + kPart + kSwap + kScaleFloats * 4 + kBars * 8 + 16;
  static_assert(kSmem <= 232448 && kSmem > 116736, "shared memory");
};

// Two groups need more registers than 384 threads' even share: they raise
// their limit to kMoreRegs a thread and the four other warps drop theirs;
// 256 * 216 + 128 * 72 <= 384 * 168 at launch.
constexpr int kMoreRegs = 216, kFewerRegs = 72;

// Instruction descriptor, kind::f8f6f4: D f32 (bits 4-5 = 1), A and B e4m3
// (bits 7-9, 10-12 = 0), both K-major (bits 15, 16 = 0), N >> 3 at bits
// 17-22, M >> 4 at bits 24-28.
template <int N> constexpr uint32_t kIdesc = (1u << 4) | (uint32_t(N >> 3) << 17) | (uint32_t(kTileM >> 4) << 24);

template <int N>
__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\t"
               "setp.ne.b32 p, %4, 0;\n\t"
               "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
               ::"r"(d_tmem), "l"(a), "l"(b), "r"(kIdesc<N>), "r"(accumulate)
               : "memory");
}

// sum += d * scale, two columns at a time.  Volatile: kept behind the TMEM load
// that was issued before it.
__device__ __forceinline__ void fma2(uint64_t &sum, uint32_t d0, uint32_t d1, uint64_t scale) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(d0), "r"(d1));
  asm volatile("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sum) : "l"(d), "l"(scale));
}
// The same where the scale is held in two factors (ScalePair).
__device__ __forceinline__ void fma2_split(uint64_t &sum, uint32_t d0, uint32_t d1, uint64_t scale, uint64_t power) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(d0), "r"(d1));
  asm volatile("{\n\t.reg .b64 t;\n\t"
               "mul.rn.f32x2 t, %1, %3;\n\t"
               "fma.rn.f32x2 %0, t, %2, %0;\n\t}"
               : "+l"(sum)
               : "l"(d), "l"(scale), "l"(power));
}
// 32 consecutive TMEM columns of this thread's lane: the load, and the wait
// for every load issued, which the registers pass through so that no use of
// them is moved before it.
__device__ __forceinline__ void tmem_issue32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
               "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
                 "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
                 "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
                 "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
                 "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(addr));
}
__device__ __forceinline__ void hold(uint32_t *r) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[2][32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  hold(r[0]), hold(r[0] + 16), hold(r[1]), hold(r[1] + 16);
}
__device__ __forceinline__ uint64_t pair(float v) {
  uint64_t p;
  asm("mov.b64 %0, {%1, %1};" : "=l"(p) : "f"(v));
  return p;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}

__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile int *abort_s) {
  if (mbar_try(bar, parity)) return true;
  long long t0 = 0;
#pragma unroll 1
  for (int i = 1;; ++i) {
    if (mbar_try(bar, parity)) return true;
    if (i % 64) continue;
    if (*abort_s) return false;
    const long long t = clock64();
    if (t0 == 0) t0 = t;
    if (t - t0 > kWaitClocks) {
      *abort_s = 1;
      return false;
    }
  }
}
// The same for a whole warp that goes on together or not at all.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int *abort_s) {
  return __all_sync(0xFFFFFFFFu, wait_bar(bar, parity, abort_s));
}
// True in one lane of the warp.
__device__ __forceinline__ bool elect() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\t"
               "elect.sync _|p, 0xFFFFFFFF;\n\t"
               "selp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(one));
  return one != 0;
}

// Every CTA of the cluster has come here; what it wrote before is visible.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

// Whether rows of the result, bias and memory term can be moved 16 bytes at a time.
__host__ inline bool vector_rows(const BlockMatmulArgs &a) {
  const auto ok = [](const void *p, long row_bytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row_bytes % 16 == 0;
  };
  return ok(a.y, a.ldy * long(elem_size(a.type))) && ok(a.bias, 0) && (!a.add || ok(a.add, a.ldadd * 4));
}

// Two values as 16-bit elements.
template <class Y> __device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t u;
  if constexpr (std::is_same_v<Y, __nv_bfloat16>)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u) : "f"(hi), "f"(lo));
  return u;
}

// A warp's 32 rows m0.. of kCols columns n0.., a row a lane in sum: bias and
// memory term, rounding, store.  Each 64 bytes of the rows change places in
// shared memory (16-byte pieces, spread over the banks), so that a store
// instruction writes 8 rows x 64 bytes and not 32 rows x 16; where the rows
// are not aligned for that, 32 elements of them.  The code is kept short: it
// runs once a tile, from instructions that the tile's main loop has pushed out
// of the cache.
template <class Y, int kCols>
__device__ __forceinline__ void store_rows(const BlockMatmulArgs &a, int m0, int n0, uint64_t (&sum)[kCols / 2],
                                           bool vec, uint4 *swap) {
  const int lane = threadIdx.x % 32, m = m0 + lane;
  if (a.bias || a.add) {
    const float *add = a.add + long(m) * a.ldadd + n0;
#pragma unroll
    for (int j = 0; j < kCols; j += 2) {
      float v[2];
      unpack2(sum[j / 2], v[0], v[1]);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (n0 + j + i >= a.n) continue;
        if (a.bias) v[i] = __fadd_rn(v[i], a.bias[n0 + j + i]);
        if (a.add && m < a.m) v[i] = __fmaf_rn(a.add_scale, add[j + i], v[i]);
      }
      asm("mov.b64 %0, {%1, %2};" : "=l"(sum[j / 2]) : "f"(v[0]), "f"(v[1]));
    }
  }
  constexpr int kStep = 64 / sizeof(Y), kPiece = 16 / sizeof(Y); // columns in 64 bytes, in 16
  const int piece = lane % 4, spread = lane / 2 % 4;
  Y *y = static_cast<Y *>(a.y) + long(m0) * a.ldy + n0;
  const bool whole = vec && a.n % kPiece == 0;
#pragma unroll
  for (int j = 0; j < kCols; j += kStep) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t u[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x, z;
        if constexpr (sizeof(Y) == 2) {
          unpack2(sum[j / 2 + 4 * i + e], x, z);
          u[e] = pack16<Y>(x, z);
        } else {
          unpack2(sum[j / 2 + 2 * i + e / 2], x, z);
          u[e] = __float_as_uint(e % 2 ? z : x);
        }
      }
      swap[4 * lane + (i ^ spread)] = make_uint4(u[0], u[1], u[2], u[3]);
    }
    __syncwarp();
    if (whole) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + lane / 4;
        const uint4 u = swap[4 * r + (piece ^ (r / 2 % 4))];
        if (m0 + r < a.m && n0 + j + piece * kPiece < a.n)
          *reinterpret_cast<uint4 *>(y + r * a.ldy + j + piece * kPiece) = u;
      }
    } else {
      const Y *held = reinterpret_cast<const Y *>(swap);
#pragma unroll 4
      for (int i = 0; i < kStep; ++i) { // 32 elements an iteration, along the rows
        const int r = (32 * i + lane) / kStep, col = (32 * i + lane) % kStep;
        const Y v = held[(4 * r + ((col / kPiece) ^ (r / 2 % 4))) * kPiece + col % kPiece];
        if (m0 + r < a.m && n0 + j + col < a.n) y[r * a.ldy + j + col] = v;
      }
    }
    __syncwarp();
  }
}

// Four consecutive columns n.. of row m of a split's joined sums.
template <class Y>
__device__ __forceinline__ void store4(const BlockMatmulArgs &a, int m, int n, float4 s, bool vec) {
  float v[4] = {s.x, s.y, s.z, s.w};
  const bool whole = vec && n + 4 <= a.n;
  if (whole) {
    if (a.bias) {
      const float4 b = *reinterpret_cast<const float4 *>(a.bias + n);
      v[0] = __fadd_rn(v[0], b.x), v[1] = __fadd_rn(v[1], b.y), v[2] = __fadd_rn(v[2], b.z), v[3] = __fadd_rn(v[3], b.w);
    }
    if (a.add) {
      const float4 e = *reinterpret_cast<const float4 *>(a.add + long(m) * a.ldadd + n);
      const float c = a.add_scale;
      v[0] = __fmaf_rn(c, e.x, v[0]), v[1] = __fmaf_rn(c, e.y, v[1]), v[2] = __fmaf_rn(c, e.z, v[2]), v[3] = __fmaf_rn(c, e.w, v[3]);
    }
    Y *y = static_cast<Y *>(a.y) + long(m) * a.ldy + n;
    if constexpr (sizeof(Y) == 4)
      *reinterpret_cast<float4 *>(y) = make_float4(v[0], v[1], v[2], v[3]);
    else
      *reinterpret_cast<uint2 *>(y) = make_uint2(pack16<Y>(v[0], v[1]), pack16<Y>(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.n) finish(a, m, n + i, v[i]);
  }
}

template <int TN, class Y>
__global__ void __launch_bounds__(TcShape<TN>::kThreads, 1)
    k_block_tc(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_w, BlockMatmulArgs a,
               int splits, int tiles_n, int tiles, bool vec, int *err, int stall_test) {
  using S = TcShape<TN>;
  extern __shared__ uint8_t smem_raw[];
  // 128-byte swizzled tiles start on 1024-byte boundaries of the shared window.
  uint8_t *stages = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u); // [kStages][a, weights]
  float4 *part = reinterpret_cast<float4 *>(stages + S::kStages * size_t(S::kStageBytes));
  uint4 *swap = reinterpret_cast<uint4 *>(part + S::kPart / 16);     // [epilogue warps][32][4]
  float *scales_a = reinterpret_cast<float *>(swap + S::kSwap / 16); // [2][kScaleChunk][kTileM]
  float *scales_w = scales_a + 2 * kScaleChunk * kTileM;             // [2][kScaleChunk][kGroups]
  uint64_t *bars = reinterpret_cast<uint64_t *>(scales_w + 2 * kScaleChunk * S::kGroups);
  volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(bars + S::kBars);
  volatile int *abort_s = reinterpret_cast<volatile int *>(tmem_slot + 1);
  // [2][2], of a buffer and of the warp that filled it: a scale product may need two factors.
  volatile uint8_t *far_scales = reinterpret_cast<volatile uint8_t *>(abort_s + 1);
  // One value for the whole warp, known as such: the roles' branches are uniform.
  const int tid = threadIdx.x, warp = __shfl_sync(0xFFFFFFFFu, tid / 32, 0), lane = tid % 32;
  const int kb = (a.k + kScaleBlock - 1) / kScaleBlock;
  const int z = blockIdx.x % splits, first = blockIdx.x / splits, stride = gridDim.x / splits;
  const int kb0 = int(long(z) * kb / splits), kb1 = int(long(z + 1) * kb / splits);
  // full / empty[stage]: a stage holds its blocks / has been read by its MMAs;
  // ready / taken[acc]: a set of accumulators holds its blocks' sums / has been
  // added up; sfull / sempty[buffer]: scales are staged / have been used.
  const uint32_t full = smem_u32(bars), empty = full + 8 * S::kStages, ready = empty + 8 * S::kStages,
                 taken = ready + 8 * S::kAccs, sfull = taken + 8 * S::kAccs, sempty = sfull + 16, done = sempty + 16;
  constexpr int kCopyWarp = S::kEpilogue / 32, kMmaWarp = kCopyWarp + 1, kScaleWarp = kCopyWarp + 2;

  const bool stalled = stall_test != 0; // test switch: the path of a wait that ran out, with nothing in flight
  // Scales of 16 blocks along k from b on: lane = block and one of four rows
  // (two warps); 1 for rows and blocks out of range, whose bytes are zeros.
  const int quarter = (warp - kScaleWarp) * 2 + lane / kScaleChunk, at = lane % kScaleChunk;
  constexpr int kBatch = S::kGroups == 1 ? 32 : 16; // loads in flight together
  float v[kBatch], vw;
  const auto load_scales = [&](int tile, int c, int r) {
    const int b = c + at, m = tile / tiles_n * kTileM + quarter + r, n = tile % tiles_n * TN + quarter * S::kCols;
    const float *from = a.a_scale + long(m) * kb + b;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) v[i] = b < kb1 && m + 4 * i < a.m ? from[4 * i * long(kb)] : 1.f;
    vw = quarter < S::kGroups && b < kb1 && n < a.n ? a.w_scale[long(n / kScaleBlock) * kb + b] : 1.f;
  };
  // Before the CTA meets, only what does not make it wait.
  if (warp == kCopyWarp) {
    if (lane == 0) {
      for (int i = 0; i < S::kStages; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
      for (int i = 0; i < S::kAccs; ++i) mbar_init(ready + 8 * i, 1), mbar_init(taken + 8 * i, 4 * S::kGroups);
      for (int i = 0; i < 2; ++i) mbar_init(sfull + 8 * i, 2), mbar_init(sempty + 8 * i, 4 * S::kGroups);
      mbar_init(done, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      *abort_s = stall_test;
    }
    if (lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_a)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_w)) : "memory");
    }
    __syncwarp();
  } else if (warp >= kScaleWarp) {
    if (first < tiles) load_scales(first, kb0, 0);
  } else if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(const_cast<uint32_t *>(tmem_slot))),
                 "r"(S::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (splits > 1) cluster_arrive(); // this CTA runs: the others may write to its shared memory
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < kCopyWarp) {
    if constexpr (S::kGroups == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMoreRegs));
    const int group = warp / 4, row = tid % 128;
    const uint32_t from = tmem + (uint32_t(warp % 4 * 32) << 16) + group * S::kCols;
    uint64_t sum[S::kCols / 2];
    uint32_t d[2][32];
    bool alive = !stalled, met = false; // met: the cluster's CTAs are known to run
    const int sets = (kb1 - kb0 + S::kPair - 1) / S::kPair;                       // of accumulators a tile
    int left = first < tiles ? ((tiles - 1 - first) / stride + 1) * sets : 0; // still to add
    int acc = 0, chunk = 0; // set in turn, scale buffers taken so far
    uint32_t parity = 0;    // of the ring's round
    // 32 columns i of a set: of its block i / kPer.
    constexpr int kPer = S::kCols / 32;
    const auto load = [&](int i) {
      tmem_issue32(from + acc * (S::kPair * TN) + i / kPer * TN + i % kPer * 32, d[i % 2]);
    };
    // The first columns of the set in turn, once it is ready, on their way to registers.
    const auto begin = [&] {
      alive = wait_warp(ready + 8 * acc, parity, abort_s);
      fence_after();
      if (alive) load(0), load(1);
    };
    if (alive && left) begin();
    for (int tile = first; tile < tiles && alive; tile += stride) {
#pragma unroll
      for (int j = 0; j < S::kCols / 2; ++j) sum[j] = 0;
      for (int c = kb0; c < kb1 && alive; c += kScaleChunk, ++chunk) {
        const int buf = chunk % 2;
        alive = wait_warp(sfull + 8 * buf, (chunk / 2) & 1, abort_s);
        const float *sa = scales_a + buf * kScaleChunk * kTileM + row, *sw = scales_w + buf * kScaleChunk * S::kGroups + group;
        // far: some scale of the chunk lies outside 2^-63 .. 2^63, so a product of two may leave the
        // normal range.  Two loops, told apart once a chunk (8192 x 8192 x 4096: 252 us, as without
        // the second; the split form in the one loop 282).
        const auto add_chunk = [&](auto far) {
          for (int b = min(kScaleChunk, kb1 - c); b > 0 && alive; b -= S::kPair) {
            const int blocks = min(b, S::kPair);
            uint64_t scale[S::kPair];
            uint64_t power[S::kPair];
#pragma unroll
            for (int u = 0; u < S::kPair; ++u, sa += kTileM, sw += S::kGroups) {
              if constexpr (far.value) {
                const ScalePair s = u < blocks ? scale_pair(*sa, *sw) : ScalePair{0.f, 1.f};
                scale[u] = pair(s.s), power[u] = pair(s.p);
              } else {
                scale[u] = u < blocks ? pair(__fmul_rn(*sa, *sw)) : 0;
              }
            }
#pragma unroll
            for (int i = 0; i < S::kPair * kPer; i += 2) {
              if (i / kPer >= blocks) continue;
              const bool last = i + 2 >= blocks * kPer; // of the set
              tmem_wait(d);
              if (last) {
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(taken + 8 * acc);
              }
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int u = (i + h) / kPer, j = (i + h) % kPer * 32;
                if (u < blocks) {
#pragma unroll
                  for (int e = 0; e < 32; e += 2) {
                    if constexpr (far.value)
                      fma2_split(sum[(j + e) / 2], d[h][e], d[h][e + 1], scale[u], power[u]);
                    else
                      fma2(sum[(j + e) / 2], d[h][e], d[h][e + 1], scale[u]);
                  }
                }
                if (!last) load(i + 2 + h);
              }
              if (last) {
                acc = acc + 1 == S::kAccs ? 0 : acc + 1;
                parity ^= acc == 0;
                if (--left) begin();
              }
            }
          }
        };
        if (__any_sync(0xFFFFFFFFu, far_scales[2 * buf] | far_scales[2 * buf + 1]))
          add_chunk(std::true_type());
        else
          add_chunk(std::false_type());
        __syncwarp();
        if (lane == 0) mbar_arrive(sempty + 8 * buf);
      }
      if (!alive && left) break;
      const int n0 = tile % tiles_n * TN + group * S::kCols, m0 = tile / tiles_n * kTileM + row / 32 * 32;
      if (splits == 1) {
        store_rows<Y, S::kCols>(a, m0, n0, sum, vec, swap + warp * 128);
      } else {
        cluster_wait();
        met = true;
        const int rows = kTileM / splits, owner = row / rows;
        float4 *to = cg::this_cluster().map_shared_rank(part, owner) + long(z) * (S::kCols / 4) * (rows + 1) + row % rows;
#pragma unroll
        for (int j = 0; j < S::kCols; j += 4) {
          float4 v;
          unpack2(sum[j / 2], v.x, v.y);
          unpack2(sum[j / 2 + 1], v.z, v.w);
          to[j / 4 * (rows + 1)] = v;
        }
      }
    }
    if (splits > 1 && !met) cluster_wait();
  } else {
    if constexpr (S::kGroups == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFewerRegs));
    // The copies' and MMAs' warps run as one and elect the lane that issues:
    // the instructions' operands stay in uniform registers.
    if (warp == kCopyWarp && !stalled) {
      bool ok = true;
      int it = 0;
      for (int tile = first; tile < tiles && ok; tile += stride) {
        for (int b = kb0; b < kb1; b += S::kPair, ++it) {
          const int st = it % S::kStages;
          if (it >= S::kStages) ok = wait_warp(empty + 8 * st, (it / S::kStages - 1) & 1, abort_s);
          if (!ok) break;
          if (elect()) {
            const int blocks = min(S::kPair, kb1 - b);
            mbar_expect(full + 8 * st, blocks * S::kBlockBytes);
            for (int u = 0; u < blocks; ++u) {
              const uint32_t dst = smem_u32(stages + st * size_t(S::kStageBytes) + u * S::kBlockBytes);
              tma_load_2d(dst, &tm_a, (b + u) * kScaleBlock, tile / tiles_n * kTileM, full + 8 * st);
              tma_load_2d(dst + kTileABytes, &tm_w, (b + u) * kScaleBlock, tile % tiles_n * TN, full + 8 * st);
            }
          }
          __syncwarp();
        }
      }
      // Copies in flight when a wait ran out, here or in another role.
      int none = 0;
      for (int i = max(0, it - S::kStages); i < it; ++i)
        wait_bar(full + 8 * (i % S::kStages), (i / S::kStages) & 1, &none);
    } else if (warp == kMmaWarp && !stalled) {
      bool ok = true;
      int it = 0;
      const uint64_t desc_a = sw128_desc(smem_u32(stages)), desc_w = sw128_desc(smem_u32(stages) + kTileABytes);
      for (int tile = first; tile < tiles && ok; tile += stride) {
        for (int b = kb0; b < kb1; b += S::kPair, ++it) {
          const int st = it % S::kStages, acc = it % S::kAccs;
          ok = wait_warp(full + 8 * st, (it / S::kStages) & 1, abort_s);
          if (ok && it >= S::kAccs) ok = wait_warp(taken + 8 * acc, (it / S::kAccs - 1) & 1, abort_s);
          if (!ok) break;
          fence_after();
          if (elect()) {
            const uint64_t at = uint64_t(st) * (S::kStageBytes >> 4); // descriptors count 16 bytes
#pragma unroll
            for (int u = 0; u < S::kPair; ++u) {
              if (b + u >= kb1) continue;
#pragma unroll
              for (int j = 0; j < kScaleBlock / 32; ++j) {
                const uint64_t off = at + u * (S::kBlockBytes >> 4) + 2 * j;
                mma_f8<TN>(tmem + (acc * S::kPair + u) * TN, desc_a + off, desc_w + off, j > 0);
              }
            }
            mma_commit(empty + 8 * st);
            mma_commit(ready + 8 * acc);
          }
          __syncwarp();
        }
      }
      if (elect()) mma_commit(done); // arrives once every MMA above has completed
      __syncwarp();
      int none = 0;
      wait_bar(done, 0, &none);
    } else if (warp >= kScaleWarp && !stalled) {
      bool ok = true;
      int chunk = 0;
      for (int tile = first; tile < tiles && ok; tile += stride) {
        for (int c = kb0; c < kb1; c += kScaleChunk, ++chunk) {
          const int buf = chunk % 2;
          if (chunk >= 2) ok = wait_warp(sempty + 8 * buf, (chunk / 2 - 1) & 1, abort_s);
          if (!ok) break;
          float *sa = scales_a + (buf * kScaleChunk + at) * kTileM;
          bool far = is_far(vw);
#pragma unroll 1
          for (int r = 0; r < kTileM; r += 4 * kBatch) {
            if (r > 0) load_scales(tile, c, r);
#pragma unroll
            for (int i = 0; i < kBatch; ++i) sa[quarter + r + 4 * i] = v[i], far |= is_far(v[i]);
          }
          far = __any_sync(0xFFFFFFFFu, far);
          if (lane == 0) far_scales[2 * buf + warp - kScaleWarp] = far;
          if (quarter < S::kGroups) scales_w[(buf * kScaleChunk + at) * S::kGroups + quarter] = vw;
          __syncwarp();
          if (lane == 0) mbar_arrive(sfull + 8 * buf);
          // The next ones, while these are used.
          if (c + kScaleChunk < kb1)
            load_scales(tile, c + kScaleChunk, 0);
          else if (tile + stride < tiles)
            load_scales(tile + stride, kb0, 0);
        }
      }
    }
    if (splits > 1) cluster_wait();
  }
  fence_before();
  __syncthreads();
  bool failed = *abort_s != 0;
  if (failed && tid == 0) *reinterpret_cast<volatile int *>(err) = 1;
  if (splits > 1) {
    // Rows of the cluster's other CTAs lack a failed one's sums: they fail with it.
    if (failed && tid < splits) *cg::this_cluster().map_shared_rank(const_cast<int *>(abort_s), tid) = 1;
    cluster_arrive();
    cluster_wait(); // every CTA has sent its sums
    failed = *abort_s != 0;
    if (!failed) {
      const int n0 = first % tiles_n * TN, rows = kTileM / splits, m0 = first / tiles_n * kTileM + z * rows;
      const int valid = min(rows, a.m - m0);
      for (int i = tid; i < valid * (TN / 4); i += S::kThreads) {
        const int r = i / (TN / 4), j = i % (TN / 4);
        float4 x[kMaxSplits];
#pragma unroll
        for (int s = 0; s < kMaxSplits; ++s)
          if (s < splits) x[s] = part[(long(s) * (TN / 4) + j) * (rows + 1) + r];
        float4 v = x[0];
#pragma unroll
        for (int s = 1; s < kMaxSplits; ++s)
          if (s < splits)
            v.x = __fadd_rn(v.x, x[s].x), v.y = __fadd_rn(v.y, x[s].y), v.z = __fadd_rn(v.z, x[s].z), v.w = __fadd_rn(v.w, x[s].w);
        store4<Y>(a, m0 + r, n0 + 4 * j, v, vec);
      }
    }
  }
  // A lost result reads NaN, not what its memory held before.
  if (failed) {
    const int rows = kTileM / splits;
    for (int tile = first; tile < tiles; tile += stride) {
      const int m0 = tile / tiles_n * kTileM + (splits > 1 ? z * rows : 0), n0 = tile % tiles_n * TN;
      for (int i = tid; i < rows * TN; i += S::kThreads)
        if (m0 + i / TN < a.m && n0 + i % TN < a.n)
          store_elem(a.y, a.type, long(m0 + i / TN) * a.ldy + n0 + i % TN, __int_as_float(0x7FFFFFFF));
    }
  }
  if (warp == kMmaWarp) {
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

// Per device: kernel attributes, SM count and the error word of products whose
// caller brings none, set up at the first call and kept until the process ends.
constexpr int kMaxDevices = 64;
struct DeviceSetup {
  std::once_flag once;
  std::atomic<ErrorWord *> err{nullptr};
  int sms = 0;
  int clusters[4] = {}; // clusters of 1, 2, 4 and 8 CTAs that run at once
} g_setup[kMaxDevices];

void cluster_config(cudaLaunchConfig_t &cfg, cudaLaunchAttribute *attr, int grid, int splits, int threads, size_t smem) {
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 1 : 0;
}

template <int TN> void configure() {
  const int smem = int(TcShape<TN>::kSmem);
  NGB_CUDA(cudaFuncSetAttribute(k_block_tc<TN, float>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  NGB_CUDA(cudaFuncSetAttribute(k_block_tc<TN, __nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  NGB_CUDA(cudaFuncSetAttribute(k_block_tc<TN, __half>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
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
    for (const void *f : {reinterpret_cast<const void *>(k_block_vec<1, 4, 1>), reinterpret_cast<const void *>(k_block_vec<1, 1, 5>),
                          reinterpret_cast<const void *>(k_block_vec<2, 4, 1>), reinterpret_cast<const void *>(k_block_vec<4, 2, 1>),
                          reinterpret_cast<const void *>(k_block_vec<4, 1, 2>)})
      NGB_CUDA(cudaFuncGetAttributes(&fa, f)); // loads the kernel
    NGB_CUDA(cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, device));
    d.clusters[0] = d.sms;
    for (int i = 1; i < 4; ++i) {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[1];
      cluster_config(cfg, attr, 1 << i, 1 << i, TcShape<64>::kThreads, TcShape<64>::kSmem);
      NGB_CUDA(cudaOccupancyMaxActiveClusters(&d.clusters[i], k_block_tc<64, float>, &cfg));
    }
    auto err = std::make_unique<ErrorWord>();
    err->ensure();
    d.err = err.release();
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

template <int NT, int AHEAD, int CTAS> void launch_vec(const BlockMatmulArgs &a, cudaStream_t s) {
  const int tiles_n = (a.n + 15) / 16;
  k_block_vec<NT, AHEAD, CTAS><<<tiles_n * ((a.m + 8 * NT - 1) / (8 * NT)), 32 * kVecWarps, 0, s>>>(a, tiles_n);
}

template <int TN> void launch_tc(const BlockMatmulArgs &a, int splits, DeviceSetup &d, cudaStream_t s) {
  CUtensorMap tm_a, tm_w;
  if (!make_map(&tm_a, a.a, a.m, a.k, a.lda, kTileM) || !make_map(&tm_w, a.w, a.n, a.k, a.ldw, TN))
    throw std::runtime_error("Cannot describe an 8-bit matrix to the copy engine");
  const long tiles_n = (a.n + TN - 1) / TN, tiles = tiles_n * ((a.m + kTileM - 1) / kTileM);
  if (tiles > INT_MAX / kMaxSplits) throw std::invalid_argument("Matrix size out of range");
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cluster_config(cfg, attr, int(splits == 1 ? std::min(tiles, long(d.sms)) : tiles * splits), splits, TcShape<TN>::kThreads,
                 TcShape<TN>::kSmem);
  cfg.stream = s;
  const auto kernel = a.type == Elem::f32    ? k_block_tc<TN, float>
                      : a.type == Elem::bf16 ? k_block_tc<TN, __nv_bfloat16>
                                             : k_block_tc<TN, __half>;
  NGB_CUDA(cudaLaunchKernelEx(&cfg, kernel, tm_a, tm_w, a, splits, int(tiles_n), int(tiles), vector_rows(a),
                              a.err ? a.err : d.err.load()->device(), take_stall()));
}

// The launch with the least estimated time, in microseconds.  The estimates
// are lines fitted to measured times (sizes 1..8192 x 200..8192 x 100..6400,
// fp32 result, operands from memory); a sample, estimate / measured:
//   32 x 928 x 768     vec<2> 2.4 / 2.4, tc<32> 5.7 / 5.6    few tiles: latency
//   256 x 768 x 3200   tc<64>, 4 splits 8.1 / 8.2, tc<32> 9.2 / 9.2
//   1 x 8192 x 4096    vec<1> one block ahead 10.4 / 10.3, four ahead 13.9
//   8192 x 8192 x 4096 tc<256> 253 / 251, tc<128> 316 / 320
struct Plan {
  int vec; // rows of a a CTA of k_block_vec takes / 8; 0: k_block_tc with the two below
  int tn, splits;
};
Plan plan(const BlockMatmulArgs &a, const DeviceSetup &d) {
  const double kb = (a.k + kScaleBlock - 1) / kScaleBlock;
  Plan best{0, 256, 1};
  double least = 1e30;
  const auto offer = [&](double t, Plan p) {
    if (t < least) least = t, best = p;
  };
  // k_block_vec: a start, and the rounds of a warp's loads; beyond a CTA an SM
  // the SM's share of the bytes.
  const double rounds = std::ceil(kb / kVecWarps);
  for (int nt : {1, 2, 4}) {
    const double load = std::ceil(a.n / 16.0) * std::ceil(a.m / (8.0 * nt)) / d.sms;
    const bool one = load <= 1;
    if (nt == 1) offer(one ? 1.7 + 0.45 * rounds : 1.5 + 0.8 * rounds * std::max(1.0, 0.8 * load), {1, 0, 0});
    if (nt == 2) offer(1.7 + 0.67 * rounds * (one ? 1 : 1.6 * load), {2, 0, 0});
    if (nt == 4) offer(1.85 + 1.08 * rounds * (one ? 1 : 1.3 * load), {4, 0, 0});
  }
  // k_block_tc: a start, a tile's blocks, and for each further tile of a CTA
  // its blocks (their bytes now compete) and its stores.
  static constexpr struct {
    int tn;
    double start, block;
  } kShapes[] = {{32, 4.6, 0.185}, {64, 5.4, 0.215}, {128, 6.2, 0.25}, {256, 7.7, 0.39}};
  for (const auto &shape : kShapes) {
    const double tiles = std::ceil(a.m / double(kTileM)) * std::ceil(a.n / double(shape.tn));
    for (int i = 0; i < 4; ++i) {
      const int splits = 1 << i;
      if (splits > 1 && (splits > kb || shape.tn >= 128 || tiles > d.clusters[i])) continue;
      const double blocks = std::ceil(kb / splits) * shape.block, more = std::ceil(tiles / d.clusters[i]) - 1;
      offer(shape.start + blocks + more * (1.15 * blocks + 0.5 + 0.012 * shape.tn) + (splits > 1 ? 1.2 : 0),
            {0, shape.tn, splits});
    }
  }
  return best;
}

} // namespace

void preload_quantize_kernels(); // block_quant.cu

void preload_block_kernels() {
  setup();
  preload_quantize_kernels();
}

void check_block_matmul_errors(int device) {
  if (device < 0 || device >= kMaxDevices) return;
  const ErrorWord *err = g_setup[device].err;
  if (err && err->take()) throw std::runtime_error(kBlockMatmulTimeout);
}

int block_matmul_kind(int m, int n, int k) {
  BlockMatmulArgs a{};
  a.m = m, a.n = n, a.k = k;
  const Plan p = plan(a, setup());
  return p.vec ? 8 * p.vec : 1000 * p.tn + p.splits;
}

void launch_block_matmul(const BlockMatmulArgs &a, cudaStream_t s) {
  DeviceSetup &d = setup();
  const Plan p = plan(a, d);
  if (p.vec) {
    const bool one = long((a.n + 15) / 16) * ((a.m + 8 * p.vec - 1) / (8 * p.vec)) <= d.sms; // a CTA an SM at most
    if (p.vec == 1)
      one ? launch_vec<1, 4, 1>(a, s) : launch_vec<1, 1, 5>(a, s);
    else if (p.vec == 2)
      launch_vec<2, 4, 1>(a, s);
    else
      one ? launch_vec<4, 2, 1>(a, s) : launch_vec<4, 1, 2>(a, s);
    return;
  }
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
