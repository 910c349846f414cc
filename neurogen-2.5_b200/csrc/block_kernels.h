// 8-bit block-scaled operands: quantisation and product (block_quant.cu,
// block_matmul.cu).  A matrix [rows][cols] is held as e4m3 bytes, row stride a
// multiple of 16 bytes, with one fp32 scale for each block of 128 columns and
// `block` rows (1 for activations, 128 for weights), scales row-major
// [ceil(rows / block)][ceil(cols / 128)].
#pragma once
#include <cuda_runtime.h>
#include <cstdint>

namespace ngb {

constexpr int kScaleBlock = 128;

// Element types of the operators' 16- and 32-bit arrays (NG_F32, NG_BF16, NG_F16).
enum class Elem : int { f32 = 0, bf16 = 1, f16 = 2 };
inline long block_row_bytes(long cols) { return (cols + 15) / 16 * 16; }
inline long scale_blocks(long n) { return (n + kScaleBlock - 1) / kScaleBlock; }
inline size_t elem_size(Elem t) { return t == Elem::f32 ? 4 : 2; }

// Block b of a matrix of `blocks` <= 2^31 - 1 blocks of 1 x 128, kb of them a row
// of cols <= 2^30 columns.  A block past the last one has row 0 and no columns:
// all its values lie past its end, and no index is formed from its number, which
// may pass 31 bits.
struct RowBlock {
  int row, block, cols;
  bool whole; // the row does not end in the block
};
__host__ __device__ inline RowBlock row_block(long b, long blocks, int kb, long cols) {
  if (b >= blocks) return {0, 0, 0, false};
  const int row = int(b) / kb, block = int(b) - row * kb;
  return {row, block, int(cols), (block + 1) * kScaleBlock <= int(cols)};
}

struct QuantArgs {
  const void *x; // [rows] rows of cols, row stride ldx elements
  Elem type;
  const int *xidx; // optional row gather: row r of the result comes from row xidx[r] of x
  long rows, cols, ldx;
  int block; // rows a scale covers: 1 or 128
  uint8_t *q;
  long ldq; // bytes
  float *scale;
};
void launch_block_quantize(const QuantArgs &a, cudaStream_t s);
// Loads these kernels and sets up the product on the current device, so that
// no later launch does (it allocates, and may load code): once per device,
// outside any stream capture.
void preload_block_kernels();

// y[m][n] = sum_b a_scale[m][b] w_scale[n / 128][b] sum_{k in block b} a[m][k] w[n][k]
//           + bias[n] + add_scale * add[m][n]
struct BlockMatmulArgs {
  const uint8_t *a;
  long lda;
  const float *a_scale;
  const uint8_t *w;
  long ldw;
  const float *w_scale;
  const float *bias; // [n] or null
  const float *add;  // [m] rows of n or null
  long ldadd;
  float add_scale;
  void *y;
  Elem type;
  long ldy;
  int m, n, k;
  int *err; // word to set when a wait runs out (ErrorWord::device), or null: the device's own
};
void launch_block_matmul(const BlockMatmulArgs &a, cudaStream_t s);
// Which launch a product of this size takes on the current device: 8, 16 or 32
// for the few-row kernel with so many rows of a a CTA, 1000 * columns + CTAs
// for the tensor-core kernel with tiles of so many columns, each tile's k range
// shared by so many CTAs.
int block_matmul_kind(int m, int n, int k);
// Throws when a product without a word of its own reported a wait that ran out
// on this device since the last check (its result is lost; later products run
// normally).
void check_block_matmul_errors(int device);
constexpr char kBlockMatmulTimeout[] = "An 8-bit product timed out waiting for its tensor-core pipeline";

} // namespace ngb
