"""Beam search on the GPU (include/neurogen_b200.h part 5): selection over beams and vocabulary, and
the reordering of session states that follows it.

``SessionPool.beam_search`` (language.py) runs them over a pool's device-resident sessions.  Both
take CUDA tensors, run on the current stream of the tensors' device and do not synchronise;
nothing is kept between calls.
"""
import torch

from ._lib import library, check, stream_of
from .blockscale import ELEMENTS, _matrix, _row_stride, _vector

PAD = 256        # the byte vocabulary's padding token (neurogen/language/model.py:16-17)
MAX_BEAMS = 32


def beam_select(logits, scores, finished=None, allowed=None, end=None, pad=PAD):
    """One step of beam search for every group: (scores, tokens, parents, finished), each
    [groups, beams], best first.

    ``logits`` [groups * beams, vocab] (float32, bfloat16 or float16), ``scores`` float32
    [groups, beams]: the beams' cumulative log probabilities, -inf where there is no beam (a
    search starts as [0, -inf, ...]).  ``finished`` bool [groups, beams], ``allowed`` bool [vocab]:
    the tokens that may follow; the log softmax is over them.

    Candidates are every beam's allowed tokens at score + log probability, and for a finished
    beam token ``pad`` at its own score.  A new beam is finished when its parent is or its token is
    ``end``.  Scores are formed in 64 bits, from exponentials good to 1e-12, and rounded once; a beam's
    equal logits go to the lower token, equal 64-bit scores of two beams to the lower beam (two within
    some 1e-12 may come in either order, the same one for the same input).  A candidate without a finite
    score is none; slots that no candidate fills have score -inf, token ``pad``, their own index as
    parent, and count as finished.  tokens and parents are int32; parents count within the group.
    """
    rows, vocab = _matrix(logits, 'logits')
    code = ELEMENTS.get(logits.dtype)
    if code is None:
        raise ValueError('logits must be float32, bfloat16 or float16')
    if not isinstance(scores, torch.Tensor) or scores.dim() != 2:
        raise ValueError('scores must be a tensor [groups, beams]')
    groups, beams = shape = scores.shape
    if not 1 <= beams <= MAX_BEAMS:
        raise ValueError('Beams must be 1..32')
    if rows != groups * beams:
        raise ValueError(f'Need one row of logits for each of the {groups} x {beams} beams')
    if vocab < 1:
        raise ValueError('Vocabulary must not be empty')
    device = logits.device
    _vector(scores, shape, torch.float32, device, 'scores')
    if finished is not None:
        _vector(finished, shape, torch.bool, device, 'finished')
    if allowed is not None:
        _vector(allowed, (vocab,), torch.bool, device, 'allowed')
    if not 0 <= pad < vocab:
        raise ValueError('Padding token outside the vocabulary')
    if end is None:
        end = -1
    elif not 0 <= end < vocab:
        raise ValueError('End token outside the vocabulary')
    lib = library()
    need = lib.ng_beam_workspace(groups, beams, vocab)
    work = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=device) if need else None
    stride = (beams, 1)
    next_scores = torch.empty_strided(shape, stride, dtype=torch.float32, device=device)
    tokens = torch.empty_strided(shape, stride, dtype=torch.int32, device=device)
    parents = torch.empty_strided(shape, stride, dtype=torch.int32, device=device)
    done = torch.empty_strided(shape, stride, dtype=torch.bool, device=device)
    check(lib.ng_beam_select(device.index, logits.data_ptr(), code, _row_stride(logits, rows, vocab), groups,
                             beams, vocab, scores.data_ptr(), None if finished is None else finished.data_ptr(),
                             None if allowed is None else allowed.data_ptr(), end, pad, next_scores.data_ptr(),
                             tokens.data_ptr(), parents.data_ptr(), done.data_ptr(),
                             None if work is None else work.data_ptr(), need, stream_of(device)))
    return next_scores, tokens, parents, done


def reorder(states, parents):
    """Row [g, w] of ``states`` [groups * beams, ...] becomes the old row [g, parents[g, w]], in
    place; returns ``states``.

    ``parents`` int32 [groups, beams] counts within the group (``beam_select``'s).  Rows are of any
    type and may lie at any stride; each row is contiguous.  A parent outside 0..beams-1 leaves
    its row as it was.
    """
    if not isinstance(states, torch.Tensor) or states.dim() < 1:
        raise ValueError('states must be a tensor [groups * beams, ...]')
    if not states.is_cuda:
        raise ValueError('states must be on a CUDA device; there is no CPU fallback')
    if not isinstance(parents, torch.Tensor) or parents.dim() != 2:
        raise ValueError('parents must be a tensor [groups, beams]')
    groups, beams = parents.shape
    device = states.device
    _vector(parents, (groups, beams), torch.int32, device, 'parents')
    if not 1 <= beams <= MAX_BEAMS:
        raise ValueError('Beams must be 1..32')
    rows = states.shape[0]
    if rows != groups * beams:
        raise ValueError(f'Need one row of states for each of the {groups} x {beams} beams')
    if not states.is_contiguous() and rows and not states[0].is_contiguous():
        raise ValueError('Each row of states must be contiguous')
    size = states.element_size()
    row = states.numel() // rows * size if rows else 0
    stride = states.stride(0) * size if rows > 1 else row
    check(library().ng_state_reorder(device.index, states.data_ptr(), row, stride, groups, beams,
                                     parents.data_ptr(), stream_of(device)))
    return states
