"""Decoding operators without a GPU: every refusal comes before the first CUDA call, at the C
boundary and in Python, and the host-side backtrace of a beam search."""
import ctypes as ct

import numpy as np
import pytest
import torch

from conftest import gpu_available
from neurogen_b200 import blockscale, decoding, library
from neurogen_b200.language import trace_beams

P = 1 << 20   # an aligned address that no refused call follows


def refused(code, text):
    assert code == -1
    message = library().ng_error().decode()
    assert text in message, message


def quantize(x=P, dtype=0, rows=4, cols=300, ldx=300, block=1, q=P, ldq=304, scale=P):
    return library().ng_block_quantize(0, x, dtype, rows, cols, ldx, block, q, ldq, scale, None)


@pytest.mark.parametrize('change,text', [
    (dict(dtype=3), 'Element type'), (dict(dtype=-1), 'Element type'), (dict(block=2), '1 or 128 rows'),
    (dict(rows=-1), 'out of range'), (dict(cols=0), 'out of range'), (dict(rows=1 << 31), 'out of range'),
    (dict(rows=(1 << 31) - 1, cols=1 << 20, ldx=1 << 20, ldq=1 << 20), 'out of range'),
    (dict(rows=1, cols=(1 << 30) + 1, ldx=1 << 31, ldq=1 << 31), 'out of range'),
    (dict(ldx=299), 'Row stride'), (dict(ldq=288), 'Row stride'), (dict(ldq=308), '16-byte'),
    (dict(q=P + 8), '16-byte'), (dict(x=None), 'Null'), (dict(q=None), 'Null'), (dict(scale=None), 'Null'),
    (dict(x=P + 2), 'aligned'), (dict(x=P + 1, dtype=1), 'aligned'), (dict(scale=P + 2), 'aligned'),
])
def test_quantize_refusals(change, text):
    refused(quantize(**change), text)


def matmul(a=P, lda=304, sa=P, w=P, ldw=304, sw=P, m=4, n=5, k=300, bias=None, add=None, ldadd=5, y=P, dtype=0, ldy=5):
    return library().ng_block_matmul(0, a, lda, sa, w, ldw, sw, m, n, k, bias, add, ldadd, 1.0, y, dtype, ldy, None)


@pytest.mark.parametrize('change,text', [
    (dict(dtype=7), 'Element type'), (dict(m=-1), 'out of range'), (dict(n=0), 'out of range'),
    (dict(k=0), 'out of range'), (dict(m=1 << 31), 'out of range'), (dict(lda=288), 'Row stride'),
    (dict(ldw=299), 'Row stride'), (dict(ldy=4), 'Row stride'), (dict(add=P, ldadd=4), 'Row stride'),
    (dict(lda=301), '16-byte'), (dict(ldw=300), '16-byte'), (dict(a=P + 4), '16-byte'), (dict(w=P + 1), '16-byte'),
    (dict(a=None), 'Null'), (dict(w=None), 'Null'), (dict(sa=None), 'Null'), (dict(sw=None), 'Null'),
    (dict(y=None), 'Null'), (dict(y=P + 2), 'aligned'), (dict(y=P + 1, dtype=1), 'aligned'),
    (dict(bias=P + 2), 'aligned'), (dict(add=P + 1), 'aligned'), (dict(sa=P + 1), 'aligned'),
])
def test_matmul_refusals(change, text):
    refused(matmul(**change), text)


def select(logits=P, dtype=0, ld=264, groups=2, beams=4, vocab=264, scores=P, end=258, pad=256, out=P, work=P,
           work_bytes=1 << 20):
    return library().ng_beam_select(0, logits, dtype, ld, groups, beams, vocab, scores, None, None, end, pad, out, out,
                                    out, out, work, work_bytes, None)


@pytest.mark.parametrize('change,text', [
    (dict(dtype=3), 'Element type'), (dict(beams=0), '1..32'), (dict(beams=33), '1..32'),
    (dict(vocab=0), 'Vocabulary'), (dict(vocab=(1 << 30) + 1, ld=1 << 31), 'Vocabulary'), (dict(groups=-1), 'Too many'), (dict(groups=1 << 28, beams=32), 'Too many'),
    (dict(ld=263), 'Row stride'), (dict(pad=264), 'Padding token'), (dict(pad=-1), 'Padding token'),
    (dict(end=264), 'End token'), (dict(logits=None), 'Null'), (dict(scores=None), 'Null'), (dict(out=None), 'Null'),
    (dict(logits=P + 2), 'aligned'), (dict(scores=P + 2), 'aligned'),
    (dict(vocab=5000, ld=5000, work=None), 'Workspace'), (dict(vocab=5000, ld=5000, work_bytes=8), 'Workspace'),
    (dict(vocab=5000, ld=5000, work=P + 8), 'Workspace'),
])
def test_select_refusals(change, text):
    refused(select(**change), text)


def reorder(states=P, row=16, ld=16, groups=2, beams=4, parents=P):
    return library().ng_state_reorder(0, states, row, ld, groups, beams, parents, None)


@pytest.mark.parametrize('change,text', [
    (dict(beams=0), '1..32'), (dict(beams=33), '1..32'), (dict(groups=-1), 'out of range'),
    (dict(row=-4), 'out of range'), (dict(ld=12), 'Row stride'), (dict(states=None), 'Null'),
    (dict(parents=None), 'Null'), (dict(parents=P + 2), 'aligned'),
])
def test_reorder_refusals(change, text):
    refused(reorder(**change), text)


def test_empty_calls_need_no_device():
    assert quantize(rows=0, x=None) == 0 and matmul(m=0, a=None) == 0
    assert select(groups=0, logits=None) == 0 and reorder(groups=0, states=None) == 0 and reorder(row=0, ld=0) == 0


def test_pool_entry_points_refuse_null_handles():
    lib = library()
    z = np.zeros(4, np.int32)
    refused(lib.ng_pool_reorder(None, 2, z), 'Null pool')
    refused(lib.ng_pool_reorder_device(None, 2, P, None), 'Null pool')
    refused(lib.ng_pool_check(None), 'Null pool')
    assert lib.ng_pool_device(None) == -1


def test_workspace_sizes():
    lib = library()
    assert lib.ng_beam_workspace(4, 8, 264) == 0
    assert lib.ng_beam_workspace(4, 8, 50000) > 0
    assert lib.ng_beam_workspace(0, 8, 50000) == 0 and lib.ng_beam_workspace(4, 33, 50000) == 0


@pytest.mark.skipif(gpu_available(), reason='checks the no-GPU failure path')
def test_no_gpu_fails_loudly():
    for call in (quantize, matmul, select, reorder):
        refused(call(), 'CUDA device')


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    q = torch.zeros(4, 16, dtype=torch.uint8).view(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match='CUDA device'):
        blockscale.quantize(x)
    with pytest.raises(ValueError, match='CUDA device'):
        blockscale.matmul(q, torch.zeros(4, 1), q, torch.zeros(1, 1))
    with pytest.raises(ValueError, match='CUDA device'):
        decoding.beam_select(x, torch.zeros(1, 4))
    with pytest.raises(ValueError, match='CUDA device'):
        decoding.reorder(x, torch.zeros((1, 4), dtype=torch.int32))
    with pytest.raises(ValueError, match='rows, columns'):
        blockscale.quantize(torch.zeros(4))


def test_trace_beams():
    """Two steps back through a crossing of two beams, by hand."""
    tokens = np.array([[[10, 11]], [[20, 21]], [[30, 31]]], np.int32)
    parents = np.array([[[0, 0]], [[1, 0]], [[0, 0]]], np.int32)
    assert trace_beams(tokens, parents).tolist() == [[[11, 20, 30], [11, 20, 31]]]


def test_trace_beams_against_copied_sequences():
    rng = np.random.default_rng(0)
    steps, groups, beams = 9, 3, 5
    tokens = rng.integers(0, 264, (steps, groups, beams)).astype(np.int32)
    parents = rng.integers(0, beams, (steps, groups, beams)).astype(np.int32)
    held = [[[] for _ in range(beams)] for _ in range(groups)]
    for t in range(steps):
        held = [[held[g][parents[t, g, w]] + [int(tokens[t, g, w])] for w in range(beams)] for g in range(groups)]
    assert trace_beams(tokens, parents).tolist() == held
