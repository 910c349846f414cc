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

// fl(amax / 448), at least 2^-126.  The quotient by a constant is one product
// and its exact remainder's correction (Markstein; equal to the IEEE division
// for every fp32 amax whose quotient is at least 2^-126).
__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
  constexpr float kInverse = 1.f / 448.f;
  const float amax = __uint_as_float(amax_bits), q = __fmul_rn(amax, kInverse);
  const float s = __fmaf_rn(__fmaf_rn(-448.f, q, amax), kInverse, q);
  if (amax_bits >= 0x7F800000u) return amax; // infinite or NaN
  return fmaxf(s, 1.17549435e-38f);
}

// Four values as four e4m3 bytes, round to nearest even.
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d) {
  uint16_t lo, hi; // the second operand goes to the low byte
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return uint32_t(lo) | (uint32_t(hi) << 16);
}

// Packed pairs of fp32: each half is one IEEE operation.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// fl(x / scale) for a whole block by one reciprocal and exact remainders
// (Markstein): with down + lo = 1 / scale to 2^-46, q = fl(x down + fl(x lo)) is
// a neighbour of the quotient, its remainder is exact, and one step from a
// neighbour by the rounded reciprocal hi gives the correctly rounded quotient.
// Four operations a value, two a packed instruction (8192 x 8192 bf16 40 us,
// 45 one by one), where the divisions cost more than the block's bytes (a
// product that divides only near the ties of e4m3 was no faster: bf16 ratios
// are often short, and most warps had one).  The remainders are exact
// while scale is at least 2^-90 (a quotient below 2^-11, where they might not
// be, is the byte 0 in any case) and lo is while it is at most 2^90; other
// blocks divide.  down is 1 / scale rounded down and lo not negative, so that
// both parts of a zero's quotient have its sign; the last step's signs keep it.
struct BlockScale {
  float scale, hi, down, lo;
  bool divide;
  __device__ __forceinline__ explicit BlockScale(uint32_t amax_bits) {
    scale = block_scale(amax_bits);
    hi = __fdiv_rn(1.f, scale);
    down = __fmaf_rn(-scale, hi, 1.f) < 0.f ? __uint_as_float(__float_as_uint(hi) - 1u) : hi;
    lo = __fmul_rn(__fmaf_rn(-scale, down, 1.f), hi);
    divide = !(scale >= 0x1p-90f && scale <= 0x1p90f);
  }
  // Four values, the quotients negated until the last step so that no value
  // changes sign before; pairs go through one packed instruction a step.
  __device__ __forceinline__ uint32_t quantize4(const float (&v)[4]) const {
    float q[4];
    if (divide) {
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = __fdiv_rn(v[i], scale);
      return pack_e4m3(q[0], q[1], q[2], q[3]);
    }
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const f32x2 x = pack2(v[i], v[i + 1]), n = fma2(x, pack2(-down, -down), mul2(x, pack2(-lo, -lo)));
      unpack2(fma2(fma2(n, pack2(scale, scale), x), pack2(-hi, -hi), n), q[i], q[i + 1]);
    }
    return pack_e4m3(q[0], q[1], q[2], q[3]) ^ 0x80808080u;
  }
};

// Sixteen bytes of a row from column k: kN values, zero past the row's end.
// VEC: the row's start and stride allow one load.  Otherwise four loads of 32
// bits, or for 16-bit types the one or two aligned 16-byte words that hold
// them, shifted into place; a word with one byte of the row lies within the
// row's memory.  (8000 x 8100 bf16, 128 x 128 blocks: 48 us, 57 with a load a
// value; fp32 58 us, 80 with shifted words; with one load 36 and 50.)
// WHOLE: the row does not end in the block.  Checks and addresses were a third
// of these kernels' instructions (8000 x 8100 from 61 and 65 us), so blocks are
// told apart once and not every chunk.
template <class T, bool VEC> struct Chunk {
  static constexpr int kN = 16 / sizeof(T);
  union {
    uint4 words;
    uint32_t word[4];
    T raw[kN];
  };
  __device__ __forceinline__ Chunk() : words(make_uint4(0, 0, 0, 0)) {}
  // First the word that holds the first value, of all of a thread's chunks ...
  template <bool WHOLE> __device__ __forceinline__ void fetch(const T *row, int k, int cols) {
    if ((!WHOLE && k + kN > cols) || (!VEC && sizeof(T) == 4)) { // the row's end
#pragma unroll
      for (int i = 0; i < kN; ++i)
        if (WHOLE || k + i < cols) raw[i] = row[k + i];
    } else {
      words = __ldg(reinterpret_cast<const uint4 *>(reinterpret_cast<uintptr_t>(row + k) & ~uintptr_t(15)));
    }
  }
  // ... then the next one, which is mostly another lane's first.
  template <bool WHOLE> __device__ __forceinline__ void align(const T *row, int k, int cols) {
    if constexpr (!VEC && sizeof(T) == 2) {
      const uintptr_t p = reinterpret_cast<uintptr_t>(row + k);
      const uint32_t skip = p % 16;
      if ((!WHOLE && k + kN > cols) || skip == 0) return;
      const uint4 hi = __ldg(reinterpret_cast<const uint4 *>(p - skip + 16));
      uint32_t w[8] = {word[0], word[1], word[2], word[3], hi.x, hi.y, hi.z, hi.w};
      if (skip & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
      }
      if (skip & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) word[i] = __funnelshift_r(w[i], w[i + 1], 8 * (skip & 3));
    }
  }
  // The largest |value|, as bits of its type (their order is the values', a
  // NaN's above infinity's).  16-bit types: two at a time, one in each half.
  __device__ __forceinline__ uint32_t amax(uint32_t m) const {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = sizeof(T) == 4 ? max(m, word[i] & 0x7FFFFFFFu) : __vmaxu2(m, word[i] & 0x7FFF7FFFu);
    return m;
  }
  template <bool WHOLE> __device__ __forceinline__ void store(uint8_t *row, int k, int cols, const BlockScale &s) const {
    uint32_t u[kN / 4];
#pragma unroll
    for (int j = 0; j < kN / 4; ++j) {
      const float v[4] = {to_f32<T>(raw[4 * j]), to_f32<T>(raw[4 * j + 1]), to_f32<T>(raw[4 * j + 2]), to_f32<T>(raw[4 * j + 3])};
      u[j] = s.quantize4(v);
    }
    if (WHOLE || k + kN <= cols) { // the rows start on 16-byte boundaries
      if constexpr (kN == 8)
        *reinterpret_cast<uint2 *>(row + k) = make_uint2(u[0], u[1]);
      else
        *reinterpret_cast<uint32_t *>(row + k) = u[0];
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i)
        if (k + i < cols) row[k + i] = uint8_t(u[i / 4] >> (8 * (i % 4)));
    }
  }
};

// fp32 bits of an amax over chunks, from the bits of T.
template <class T> __device__ __forceinline__ uint32_t amax_f32_bits(uint32_t m) {
  if constexpr (sizeof(T) == 4) {
    return m;
  } else {
    const uint16_t top = uint16_t(max(m & 0xFFFFu, m >> 16));
    return __float_as_uint(to_f32<T>(*reinterpret_cast<const T *>(&top)));
  }
}
template <class T> __device__ __forceinline__ uint32_t amax_join(uint32_t a, uint32_t b) {
  return sizeof(T) == 4 ? max(a, b) : __vmaxu2(a, b);
}

// 1 x 128 blocks: few lanes a block, so that a block's scale and addresses cost
// a fraction of a warp's instructions.  (8192 x 8192 bf16: a warp a block 103
// us, eight lanes 38, four 33, 6.2 TB/s; 2048 x 6400 fp32 10.0 us, 6.6 TB/s.)
template <class T> constexpr int kRowLanes = sizeof(T) == 4 ? 8 : 4;

template <class T, bool VEC> __global__ void __launch_bounds__(256) k_quant_rows(QuantArgs a, int kb, int blocks) {
  using C = Chunk<T, VEC>;
  constexpr int kLanes = kRowLanes<T>, kChunks = kScaleBlock / (kLanes * C::kN);
  const long b = (long(blockIdx.x) * blockDim.x + threadIdx.x) / kLanes;
  const auto [r, c, cols, whole] = row_block(b, blocks, kb, a.cols);
  const int lane = threadIdx.x % kLanes, k = c * kScaleBlock + lane * C::kN;
  const T *row = static_cast<const T *>(a.x) + (a.xidx ? a.xidx[r] : r) * a.ldx;
  C v[kChunks];
  uint32_t m = 0;
  if (whole) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) v[i].template fetch<true>(row, k + i * kLanes * C::kN, cols);
#pragma unroll
    for (int i = 0; i < kChunks; ++i) v[i].template align<true>(row, k + i * kLanes * C::kN, cols);
  } else {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      v[i].template fetch<false>(row, k + i * kLanes * C::kN, cols);
      v[i].template align<false>(row, k + i * kLanes * C::kN, cols);
    }
  }
#pragma unroll
  for (int i = 0; i < kChunks; ++i) m = v[i].amax(m);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o /= 2) m = amax_join<T>(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  if (b >= blocks) return;
  const BlockScale s(amax_f32_bits<T>(m));
  if (lane == 0) a.scale[b] = s.scale;
  uint8_t *q = a.q + r * a.ldq;
  if (whole) {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) v[i].template store<true>(q, k + i * kLanes * C::kN, cols, s);
  } else {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) v[i].template store<false>(q, k + i * kLanes * C::kN, cols, s);
  }
}

// 128 x 128 blocks: one CTA a block, its values in registers between the
// maximum and the conversion.  Three or four CTAs an SM cover one another's
// loads and meeting (fp32, 8000 x 8100 and one load a chunk: 50 us, 6.5 TB/s).
// One CTA going from block to block with the next one's loads in flight had
// half the warps and was slower (51 and 71 us where this took 45 and 66).
template <class T, bool VEC, bool WHOLE> __device__ __forceinline__ void quant_tile(const QuantArgs &a, int rb, int c, int kb) {
  using C = Chunk<T, VEC>;
  constexpr int kWarps = 16, kAcross = kScaleBlock / C::kN, kRowsAtOnce = 512 / kAcross;
  constexpr int kChunks = kScaleBlock / kRowsAtOnce;
  __shared__ uint32_t part[kWarps];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, cols = int(a.cols);
  const int k = c * kScaleBlock + threadIdx.x % kAcross * C::kN;
  const long r0 = long(rb) * kScaleBlock + threadIdx.x / kAcross;
  const T *row = static_cast<const T *>(a.x) + r0 * a.ldx;
  const long step = a.ldx * kRowsAtOnce;
  const int rows = WHOLE ? kScaleBlock : int(a.rows - r0); // left from here
  C v[kChunks];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kChunks; ++i)
    if (WHOLE || i * kRowsAtOnce < rows) v[i].template fetch<WHOLE>(row + i * step, k, cols);
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    if (WHOLE || i * kRowsAtOnce < rows) v[i].template align<WHOLE>(row + i * step, k, cols);
    m = v[i].amax(m);
  }
  m = __reduce_max_sync(0xFFFFFFFFu, amax_f32_bits<T>(m));
  if (lane == 0) part[warp] = m;
  __syncthreads();
  const BlockScale s(__reduce_max_sync(0xFFFFFFFFu, part[lane % kWarps]));
  if (threadIdx.x == 0) a.scale[long(rb) * kb + c] = s.scale;
  uint8_t *q = a.q + r0 * a.ldq;
  const long q_step = a.ldq * kRowsAtOnce;
#pragma unroll
  for (int i = 0; i < kChunks; ++i)
    if (WHOLE || i * kRowsAtOnce < rows) v[i].template store<WHOLE>(q + i * q_step, k, cols, s);
}
template <class T, bool VEC> __global__ void __launch_bounds__(512, sizeof(T) == 4 ? 2 : VEC ? 4 : 3) k_quant_tiles(QuantArgs a, int kb) {
  const int rb = blockIdx.x / kb, c = blockIdx.x - rb * kb;
  if (long(rb + 1) * kScaleBlock <= a.rows && (c + 1) * kScaleBlock <= a.cols)
    quant_tile<T, VEC, true>(a, rb, c, kb);
  else
    quant_tile<T, VEC, false>(a, rb, c, kb);
}

template <class T> void launch_typed(const QuantArgs &a, cudaStream_t s) {
  const int kb = int((a.cols + kScaleBlock - 1) / kScaleBlock);
  const bool vec = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.ldx * sizeof(T) % 16 == 0;
  if (a.block == 1) {
    const int blocks = int(a.rows * kb); // the callers keep it in 31 bits
    const unsigned grid = (unsigned(blocks) + 256 / kRowLanes<T> - 1) / (256 / kRowLanes<T>);
    if (vec)
      k_quant_rows<T, true><<<grid, 256, 0, s>>>(a, kb, blocks);
    else
      k_quant_rows<T, false><<<grid, 256, 0, s>>>(a, kb, blocks);
  } else {
    const unsigned grid = unsigned(kb * ((a.rows + kScaleBlock - 1) / kScaleBlock));
    if (vec)
      k_quant_tiles<T, true><<<grid, 512, 0, s>>>(a, kb);
    else
      k_quant_tiles<T, false><<<grid, 512, 0, s>>>(a, kb);
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
