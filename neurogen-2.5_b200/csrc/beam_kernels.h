// Beam search on the device: selection over beams and vocabulary, and the
// reordering of session states that follows it (beam_kernels.cu).
#pragma once
#include "block_kernels.h"

namespace ngb {

constexpr int kMaxBeams = 32;

// One step of `groups` independent searches of `beams` beams each.  Row
// r = group * beams + beam of logits holds that beam's next-token logits.
struct BeamArgs {
  const void *logits; // [groups * beams] rows of vocab, row stride ld elements
  Elem type;
  long ld;
  int groups, beams, vocab;
  const float *scores;     // [groups][beams] cumulative log probabilities, -inf: no such beam
  const uint8_t *finished; // [groups][beams] or null
  const uint8_t *allowed;  // [vocab] or null: tokens that may follow
  int end, pad;            // token that finishes a beam (< 0: none), token a finished beam repeats
  float *next_scores;      // [groups][beams], best first; the four results may alias scores / finished
  int *tokens, *parents;   // [groups][beams]; parents within the group
  uint8_t *next_finished;
  void *work; // beam_workspace(...) bytes, 16-byte aligned, or null when that is 0
};
size_t beam_workspace(int groups, int beams, int vocab);
void launch_beam_select(const BeamArgs &a, cudaStream_t s);

// states[g][w] = old states[g][parents[g][w]], in place; rows of row_bytes at a
// stride of ld_bytes.  A parent outside 0..beams-1 leaves its row as it was.
struct ReorderArgs {
  void *states;
  long row_bytes, ld_bytes;
  int groups, beams;
  const int *parents;
};
void launch_state_reorder(const ReorderArgs &a, cudaStream_t s);

} // namespace ngb
