// Quantisation to e4m3 with a scale for each block of 128 columns:
//   scale = max(fl(amax |x| / 448), 2^-126),   q = e4m3(fl(x / scale))
// Both divisions are IEEE fp32 divisions and the conversion rounds to nearest
// even, so the result is a function of the block's values alone (any order,
// any launch shape gives the same bytes).  448 is e4m3's largest value; the
// floor on the scale keeps a block of zeros (or of numbers so small that the
// quotient would underflow) at finite quotients.  amax is taken on the bits of
// |x|, where a NaN orders above infinity: a block that holds one has a NaN
// scale, a block with an infinity an infinite scale and NaN in its place, so
// that every product with it is NaN.
#include "block_kernels.h"
#include "common.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ngb {
namespace {

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
  const float s = __fdiv_rn(__uint_as_float(amax_bits), 448.f);
  return s < 1.17549435e-38f ? 1.17549435e-38f : s; // a NaN stays
}

// Four values as four e4m3 bytes, round to nearest even.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  uint16_t lo, hi; // the second operand goes to the low byte
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return uint32_t(lo) | (uint32_t(hi) << 16);
}

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// Four consecutive values of a row from column k (values past the row's end
// are zero).  VEC: the row's start and stride allow one vector load.
template <class T, bool VEC> __device__ __forceinline__ void load4(const T *row, long k, long cols, float (&v)[4]) {
  if (VEC && k + 4 <= cols) {
    if constexpr (sizeof(T) == 4) {
      const float4 f = *reinterpret_cast<const float4 *>(row + k);
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2 *>(row + k);
      const T *e = reinterpret_cast<const T *>(&u);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = to_f32<T>(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + i < cols ? to_f32<T>(row[k + i]) : 0.f;
  }
}

__device__ __forceinline__ void store4(uint8_t *row, long k, long cols, const float (&v)[4], float scale) {
  const uint32_t u = pack_e4m3(__fdiv_rn(v[0], scale), __fdiv_rn(v[1], scale), __fdiv_rn(v[2], scale),
                               __fdiv_rn(v[3], scale));
  if (k + 4 <= cols) {
    *reinterpret_cast<uint32_t *>(row + k) = u; // the rows start on 16-byte boundaries
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (k + i < cols) row[k + i] = uint8_t(u >> (8 * i));
  }
}

// 1 x 128 blocks: one warp a block, four values a lane.
template <class T, bool VEC> __global__ void __launch_bounds__(256) k_quant_rows(QuantArgs a, long kb, long blocks) {
  const int lane = threadIdx.x % 32;
  const long b = (long(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
  if (b >= blocks) return;
  const long r = b / kb, c = b % kb, k = c * kScaleBlock + 4 * lane;
  const T *row = static_cast<const T *>(a.x) + (a.xidx ? long(a.xidx[r]) : r) * a.ldx;
  float v[4];
  load4<T, VEC>(row, k, a.cols, v);
  const uint32_t mine = max(max(abs_bits(v[0]), abs_bits(v[1])), max(abs_bits(v[2]), abs_bits(v[3])));
  const float scale = block_scale(__reduce_max_sync(0xFFFFFFFFu, mine));
  if (lane == 0) a.scale[b] = scale;
  store4(a.q + r * a.ldq, k, a.cols, v, scale);
}

// 128 x 128 blocks: one CTA a block, its values in registers between the
// maximum and the conversion (8 warps x 16 rows, four values a lane and row).
template <class T, bool VEC> __global__ void __launch_bounds__(256) k_quant_tiles(QuantArgs a, long kb) {
  constexpr int kWarps = 8, kRows = kScaleBlock / kWarps;
  __shared__ uint32_t part[kWarps];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const long rb = blockIdx.x / kb, c = blockIdx.x % kb, k = c * kScaleBlock + 4 * lane;
  float v[kRows][4];
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long r = rb * kScaleBlock + i * kWarps + warp;
    if (r < a.rows) {
      load4<T, VEC>(static_cast<const T *>(a.x) + (a.xidx ? long(a.xidx[r]) : r) * a.ldx, k, a.cols, v[i]);
    } else {
      v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i)
    mine = max(mine, max(max(abs_bits(v[i][0]), abs_bits(v[i][1])), max(abs_bits(v[i][2]), abs_bits(v[i][3]))));
  mine = __reduce_max_sync(0xFFFFFFFFu, mine);
  if (lane == 0) part[warp] = mine;
  __syncthreads();
  mine = part[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) mine = max(mine, part[i]);
  const float scale = block_scale(mine);
  if (threadIdx.x == 0) a.scale[rb * kb + c] = scale;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long r = rb * kScaleBlock + i * kWarps + warp;
    if (r < a.rows) store4(a.q + r * a.ldq, k, a.cols, v[i], scale);
  }
}

template <class T> void launch_typed(const QuantArgs &a, cudaStream_t s) {
  const long kb = (a.cols + kScaleBlock - 1) / kScaleBlock;
  const bool vec = reinterpret_cast<uintptr_t>(a.x) % (4 * sizeof(T)) == 0 && a.ldx % 4 == 0;
  if (a.block == 1) {
    const long blocks = a.rows * kb;
    const unsigned grid = unsigned((blocks + 7) / 8);
    if (vec)
      k_quant_rows<T, true><<<grid, 256, 0, s>>>(a, kb, blocks);
    else
      k_quant_rows<T, false><<<grid, 256, 0, s>>>(a, kb, blocks);
  } else {
    const unsigned grid = unsigned(kb * ((a.rows + kScaleBlock - 1) / kScaleBlock));
    if (vec)
      k_quant_tiles<T, true><<<grid, 256, 0, s>>>(a, kb);
    else
      k_quant_tiles<T, false><<<grid, 256, 0, s>>>(a, kb);
  }
}

template <class T> void preload_typed() {
  cudaFuncAttributes fa;
  for (const void *f : {reinterpret_cast<const void *>(k_quant_rows<T, true>), reinterpret_cast<const void *>(k_quant_rows<T, false>),
                        reinterpret_cast<const void *>(k_quant_tiles<T, true>), reinterpret_cast<const void *>(k_quant_tiles<T, false>)})
    NGB_CUDA(cudaFuncGetAttributes(&fa, f));
}

} // namespace

void preload_quantize_kernels() {
  preload_typed<float>();
  preload_typed<__nv_bfloat16>();
  preload_typed<__half>();
}

void launch_block_quantize(const QuantArgs &a, cudaStream_t s) {
  if (a.type == Elem::f32)
    launch_typed<float>(a, s);
  else if (a.type == Elem::bf16)
    launch_typed<__nv_bfloat16>(a, s);
  else
    launch_typed<__half>(a, s);
}

} // namespace ngb
