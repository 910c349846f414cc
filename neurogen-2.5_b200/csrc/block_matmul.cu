// Product of two block-scaled 8-bit matrices (block_kernels.h):
//   y[m][n] = sum_b sa[m][b] sw[n / 128][b] d_b[m][n] + bias[n] + c add[m][n],
//   d_b[m][n] = sum_{k in block b} a[m][k] w[n][k].
// The scales change every 128 columns, so no accumulator runs over more than
// one block: each block's sum d_b is formed by the tensor cores in fp32 and
// then added, scaled, into an fp32 register sum.
#include "block_kernels.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ngb {
namespace {

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

} // namespace

void launch_block_matmul(const BlockMatmulArgs &a, cudaStream_t s) {
  const dim3 grid((a.n + 15) / 16, (a.m + 7) / 8);
  k_block_vec<<<grid, 32 * kVecWarps, 0, s>>>(a);
}

} // namespace ngb
