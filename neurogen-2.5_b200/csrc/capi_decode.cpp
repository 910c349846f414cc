// C ABI of the decoding operators (include/neurogen_b200.h, part 5): argument
// checks, the device and stream a call runs on, and the launch.  Everything
// that can be checked without reading device memory is checked before the
// first CUDA call.
#include "beam_kernels.h"
#include "block_kernels.h"
#include "capi_common.h"
#include "common.h"
#include "neurogen_b200.h"

#include <atomic>
#include <climits>

namespace ngb {
namespace {

constexpr int kMaxDevices = 64;
std::atomic<bool> g_device_ok[kMaxDevices];

// Makes `device` current for a call and puts the caller's device back.
class OnDevice {
public:
  explicit OnDevice(int device) {
    if (device < 0 || device >= kMaxDevices) throw std::invalid_argument("CUDA device index out of range");
    int count = 0;
    if (!g_device_ok[device] && (cudaGetDeviceCount(&count) != cudaSuccess || device >= count)) {
      (void)cudaGetLastError();
      throw std::runtime_error("No such CUDA device for the B200 engine; there is no CPU fallback");
    }
    NGB_CUDA(cudaGetDevice(&before_));
    if (before_ != device) NGB_CUDA(cudaSetDevice(device));
    moved_ = before_ != device;
    if (!g_device_ok[device]) {
      try {
        require_sm100_device();
      } catch (...) {
        restore();
        throw;
      }
      g_device_ok[device] = true;
    }
  }
  ~OnDevice() { restore(); }

private:
  void restore() {
    if (moved_) cudaSetDevice(before_);
    moved_ = false;
  }
  int before_ = 0;
  bool moved_ = false;
};

Elem elem(int dtype) {
  if (dtype < NG_F32 || dtype > NG_F16) throw std::invalid_argument("Element type must be NG_F32, NG_BF16 or NG_F16");
  return Elem(dtype);
}

void require(bool ok, const char *message) {
  if (!ok) throw std::invalid_argument(message);
}

bool aligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
void typed(const void *p, Elem t) { require(aligned(p, elem_size(t)), "Array is not aligned to its element type"); }

int64_t blocks_of(int64_t n, int64_t block) { return (n + block - 1) / block; }

} // namespace
} // namespace ngb

using namespace ngb;

extern "C" {

int ng_block_quantize(int device, const void *x, int dtype, int64_t rows, int64_t cols, int64_t ldx, int block_rows,
                      void *q, int64_t ldq, float *scale, void *stream) {
  return guarded([&] {
    QuantArgs a{};
    a.type = elem(dtype);
    require(block_rows == 1 || block_rows == kScaleBlock, "A scale covers 1 or 128 rows");
    require(rows >= 0 && rows <= INT_MAX && cols >= 1 && cols <= INT_MAX / 2, "Matrix size out of range");
    require(ldx >= cols && ldq >= cols, "Row stride smaller than the row");
    const int64_t blocks = blocks_of(rows, block_rows) * blocks_of(cols, kScaleBlock);
    require(blocks <= INT_MAX, "Matrix size out of range");
    if (rows == 0) return;
    require(x && q && scale, "Null matrix");
    typed(x, a.type);
    require(aligned(scale, 4), "Array is not aligned to its element type");
    require(aligned(q, 16) && ldq % 16 == 0, "8-bit rows must start on 16-byte boundaries");
    a.x = x;
    a.rows = rows;
    a.cols = cols;
    a.ldx = ldx;
    a.block = block_rows;
    a.q = static_cast<uint8_t *>(q);
    a.ldq = ldq;
    a.scale = scale;
    OnDevice on(device);
    launch_block_quantize(a, static_cast<cudaStream_t>(stream));
    NGB_CUDA(cudaGetLastError());
  });
}

int ng_block_matmul(int device, const void *a, int64_t lda, const float *a_scale, const void *w, int64_t ldw,
                    const float *w_scale, int64_t m, int64_t n, int64_t k, const float *bias, const float *add,
                    int64_t ldadd, float add_scale, void *y, int dtype, int64_t ldy, void *stream) {
  return guarded([&] {
    BlockMatmulArgs g{};
    g.type = elem(dtype);
    require(m >= 0 && m <= INT_MAX / 2 && n >= 1 && n <= INT_MAX / 2 && k >= 1 && k <= INT_MAX / 2,
            "Matrix size out of range");
    require(lda >= k && ldw >= k && ldy >= n && (!add || ldadd >= n), "Row stride smaller than the row");
    require(lda % 16 == 0 && ldw % 16 == 0, "8-bit rows must start on 16-byte boundaries");
    if (m == 0) return;
    require(a && a_scale && w && w_scale && y, "Null matrix");
    require(aligned(a, 16) && aligned(w, 16), "8-bit rows must start on 16-byte boundaries");
    typed(y, g.type);
    require(aligned(a_scale, 4) && aligned(w_scale, 4) && aligned(bias, 4) && aligned(add, 4),
            "Array is not aligned to its element type");
    g.a = static_cast<const uint8_t *>(a);
    g.lda = lda;
    g.a_scale = a_scale;
    g.w = static_cast<const uint8_t *>(w);
    g.ldw = ldw;
    g.w_scale = w_scale;
    g.bias = bias;
    g.add = add;
    g.ldadd = ldadd;
    g.add_scale = add_scale;
    g.y = y;
    g.ldy = ldy;
    g.m = int(m);
    g.n = int(n);
    g.k = int(k);
    OnDevice on(device);
    check_block_matmul_errors(device);
    launch_block_matmul(g, static_cast<cudaStream_t>(stream));
    NGB_CUDA(cudaGetLastError());
  });
}

int ng_block_matmul_kind(int device, int64_t m, int64_t n, int64_t k) {
  int kind = 0;
  const int code = guarded([&] {
    require(m >= 1 && m <= INT_MAX / 2 && n >= 1 && n <= INT_MAX / 2 && k >= 1 && k <= INT_MAX / 2,
            "Matrix size out of range");
    OnDevice on(device);
    kind = block_matmul_kind(int(m), int(n), int(k));
  });
  return code ? code : kind;
}

int ng_block_check(int device) {
  return guarded([&] {
    require(device >= 0 && device < kMaxDevices, "CUDA device index out of range");
    check_block_matmul_errors(device);
  });
}

size_t ng_beam_workspace(int groups, int beams, int vocab) {
  if (groups < 1 || beams < 1 || beams > kMaxBeams || vocab < 1) return 0;
  return beam_workspace(groups, beams, vocab);
}

int ng_beam_select(int device, const void *logits, int dtype, int64_t ld, int groups, int beams, int vocab,
                   const float *scores, const uint8_t *finished, const uint8_t *allowed, int end, int pad,
                   float *next_scores, int32_t *tokens, int32_t *parents, uint8_t *next_finished, void *workspace,
                   size_t workspace_bytes, void *stream) {
  return guarded([&] {
    BeamArgs a{};
    a.type = elem(dtype);
    require(beams >= 1 && beams <= kMaxBeams, "Beams must be 1..32");
    require(vocab >= 1, "Vocabulary must not be empty");
    require(vocab <= 1 << 30, "Vocabulary too large");
    require(groups >= 0 && int64_t(groups) * beams <= INT_MAX / 32, "Too many beams in one call");
    require(ld >= vocab, "Row stride smaller than the row");
    require(pad >= 0 && pad < vocab, "Padding token outside the vocabulary");
    require(end < vocab, "End token outside the vocabulary");
    if (groups == 0) return;
    require(logits && scores && next_scores && tokens && parents && next_finished, "Null beam array");
    typed(logits, a.type);
    require(aligned(scores, 4) && aligned(next_scores, 4) && aligned(tokens, 4) && aligned(parents, 4),
            "Array is not aligned to its element type");
    const size_t need = beam_workspace(groups, beams, vocab);
    require(need == 0 || (workspace && workspace_bytes >= need && aligned(workspace, 16)),
            "Workspace smaller than ng_beam_workspace, or not on a 16-byte boundary");
    a.logits = logits;
    a.ld = ld;
    a.groups = groups;
    a.beams = beams;
    a.vocab = vocab;
    a.scores = scores;
    a.finished = finished;
    a.allowed = allowed;
    a.end = end;
    a.pad = pad;
    a.next_scores = next_scores;
    a.tokens = tokens;
    a.parents = parents;
    a.next_finished = next_finished;
    a.work = workspace;
    OnDevice on(device);
    launch_beam_select(a, static_cast<cudaStream_t>(stream));
    NGB_CUDA(cudaGetLastError());
  });
}

int ng_state_reorder(int device, void *states, int64_t row_bytes, int64_t ld_bytes, int groups, int beams,
                     const int32_t *parents, void *stream) {
  return guarded([&] {
    require(beams >= 1 && beams <= kMaxBeams, "Beams must be 1..32");
    require(groups >= 0 && row_bytes >= 0, "State size out of range");
    require(ld_bytes >= row_bytes, "Row stride smaller than the row");
    if (groups == 0 || row_bytes == 0) return;
    require(states && parents, "Null states or parents");
    require(aligned(parents, 4), "Array is not aligned to its element type");
    OnDevice on(device);
    launch_state_reorder({states, long(row_bytes), long(ld_bytes), groups, beams, parents},
                         static_cast<cudaStream_t>(stream));
    NGB_CUDA(cudaGetLastError());
  });
}

} // extern "C"
