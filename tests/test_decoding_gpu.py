"""Beam selection and state reordering on the GPU, against plain forms in 64 bits, and a whole
beam search over a session pool.

A score is one rounding to fp32 of a 64-bit total, and two 64-bit evaluations of that total differ
by far less than a step of fp32: the tolerance is one fp32 step (2^-23 relative).  Tokens, parents
and flags have one right answer.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from neurogen_b200 import decoding  # noqa: E402
from neurogen_b200.language import LanguageConfig, NativeLanguageModel, SessionPool, init_packed_weights  # noqa: E402

TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


def select_64(logits, scores, finished=None, allowed=None, end=None, pad=256):
    """The definition: every candidate listed, ordered by score, then beam, then logit, then token."""
    groups, beams = scores.shape
    vocab = logits.shape[1]
    x = logits.astype(np.float64).reshape(groups, beams, vocab)
    out_s = np.full((groups, beams), -np.inf, np.float32)
    out_t = np.full((groups, beams), pad, np.int32)
    out_p = np.tile(np.arange(beams, dtype=np.int32), (groups, 1))
    out_f = np.ones((groups, beams), bool)
    ok = np.ones(vocab, bool) if allowed is None else allowed
    for g in range(groups):
        total, beam, logit, token = [], [], [], []
        for w in range(beams):
            s = np.float64(scores[g, w])
            if not np.isfinite(s):
                continue
            if finished is not None and finished[g, w]:
                total.append([s]), beam.append([w]), logit.append([0.0]), token.append([pad])
                continue
            at = np.flatnonzero(ok)
            v = x[g, w, at]
            if not at.size or np.isnan(v).any() or (v == np.inf).any() or (v == -np.inf).all():
                continue
            m = v.max()
            t = s + (v - (m + np.log(np.exp(v - m).sum())))
            keep = np.isfinite(t)
            total.append(t[keep]), beam.append(np.full(keep.sum(), w)), logit.append(v[keep]), token.append(at[keep])
        if not total:
            continue
        total, beam, logit, token = (np.concatenate(v) for v in (total, beam, logit, token))
        order = np.lexsort((token, -logit, beam, -total))[:beams]
        n = order.size
        out_s[g, :n], out_t[g, :n], out_p[g, :n] = total[order], token[order], beam[order]
        out_f[g, :n] = token[order] == (-1 if end is None else end)
        if finished is not None:
            out_f[g, :n] |= finished[g, beam[order]]
    return out_s, out_t, out_p, out_f


def check_select(logits, scores, finished=None, allowed=None, end=None, pad=0):
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    got = decoding.beam_select(logits if logits.is_cuda else logits.cuda(), cuda(scores), cuda(finished), cuda(allowed),
                               end, pad)
    array = lambda t: None if t is None else t.numpy()  # noqa: E731
    want = select_64(logits.float().cpu().numpy(), scores.numpy(), array(finished), array(allowed), end, pad)
    s, t, p, f = (v.cpu().numpy() for v in got)
    assert t.dtype == p.dtype == np.int32 and f.dtype == bool and s.dtype == np.float32
    np.testing.assert_array_equal(t, want[1])
    np.testing.assert_array_equal(p, want[2])
    np.testing.assert_array_equal(f, want[3])
    np.testing.assert_array_equal(np.isfinite(s), np.isfinite(want[0]))
    np.testing.assert_allclose(s, want[0], rtol=2.0 ** -23, atol=0)
    return got


def inputs(seed, groups, beams, vocab, dtype=torch.float32):
    rng = np.random.default_rng(seed)
    logits = torch.from_numpy(2.5 * rng.normal(size=(groups * beams, vocab))).to(dtype)
    scores = torch.from_numpy(-20 * rng.random((groups, beams))).float()
    return rng, logits, scores


VOCABS = [1, 2, 31, 32, 33, 127, 128, 129, 264, 288, 289, 511, 512, 513, 1000, 1024, 1025, 4096, 4097, 8193, 50001,
          131072, 140000]


@pytest.mark.parametrize('vocab', VOCABS)
@pytest.mark.parametrize('groups,beams,dtype', [(3, 1, 'fp32'), (2, 4, 'bf16'), (5, 8, 'fp32'), (2, 7, 'fp16'),
                                                (1, 32, 'fp32'), (2, 31, 'bf16')])
def test_select(groups, beams, dtype, vocab):
    rng, logits, scores = inputs(vocab + beams, groups, beams, vocab, TYPES[dtype])
    check_select(logits, scores)
    scores[0, 1:] = -np.inf   # a search's first step
    finished = torch.from_numpy(rng.random((groups, beams)) < 0.3)
    allowed = torch.from_numpy(rng.random(vocab) < 0.7)
    check_select(logits, scores, finished, allowed, end=int(rng.integers(vocab)), pad=int(rng.integers(vocab)))


@pytest.mark.parametrize('groups,beams,vocab,dtype', [(400, 3, 3000, 'bf16'), (1300, 1, 2500, 'fp32'), (40, 32, 2100, 'fp16'),
                                                      (70, 16, 1200, 'fp32'), (3, 17, 1500, 'fp32'), (130, 2, 5000, 'fp32')])
def test_select_either_side_of_the_two_launch_rule(groups, beams, vocab, dtype):
    """Long rows by one launch (many rows) and by two (few)."""
    rng, logits, scores = inputs(vocab + groups, groups, beams, vocab, TYPES[dtype])
    finished = torch.from_numpy(rng.random((groups, beams)) < 0.2)
    allowed = torch.from_numpy(rng.random(vocab) < 0.9)
    check_select(logits, scores, finished, allowed, end=7)


def test_select_ascending_and_descending_rows():
    """Orders that fill the held-back entries most often: every value above all before it, and none.
    Within a call all rows have one order: a row and its reverse have the same score as real numbers,
    and a 64-bit sum of `vocab` terms, off by up to vocab 2^-53, puts either first."""
    for beams in (1, 6, 32):
        for vocab in (264, 1000, 5000):
            row = torch.arange(vocab).float() / 64
            for order in (row, row.flip(0)):
                logits = order.expand(2 * beams, vocab).contiguous()
                check_select(logits, torch.zeros(2, beams))
                check_select((logits * 2).round(), torch.zeros(2, beams))


def test_select_far_rows():
    """Rows whose offsets pass 32 bits."""
    ld = 40_000_000
    big = torch.empty(64 * ld, dtype=torch.bfloat16, device='cuda').view(64, ld)
    for vocab in (300, 3000):
        rng, logits, scores = inputs(1, 16, 4, vocab, torch.bfloat16)
        big[:, 3:3 + vocab] = logits.cuda()
        check_select(big[:, 3:3 + vocab], scores)


@pytest.mark.parametrize('vocab', [40, 264, 900, 3000, 9000])
def test_select_ties_go_to_the_lower_index(vocab):
    """Equal logits within a beam, equal beams, and both; a vocabulary of one value only."""
    for beams in (1, 4, 9, 32):
        logits = torch.zeros(2 * beams, vocab)
        scores = torch.zeros(2, beams)
        check_select(logits, scores)
        check_select(-0.0 * torch.ones(2 * beams, vocab) * (torch.arange(vocab) % 2), scores)
        rng = np.random.default_rng(vocab + beams)
        row = torch.from_numpy(rng.integers(-2, 3, vocab)).float()
        check_select(row.expand(2 * beams, vocab).contiguous(), scores)
        scores[:, ::2] = -1.0
        check_select(row.expand(2 * beams, vocab).contiguous().bfloat16(), scores)


@pytest.mark.parametrize('vocab', [100, 264, 4000])
@pytest.mark.parametrize('centre', [-2.0 ** 31, -2.0 ** 30, 2.0 ** 24, 2.0 ** 29, 2.0 ** 30 + 64, 2.0 ** 31, 1e30, -1e30])
def test_select_far_from_zero(centre, vocab):
    """Logits whose fp32 steps are of the size of the terms that still count, or larger.

    lse = m + log(sum) is one 64-bit rounding at |m| <= 2^31 + 2^12, and two sums that differ in
    their last bits may round to neighbours, 2^-21 apart; the score's fp32 rounding is 2^-24 of it.
    At 1e30 log(sum) < 9 vanishes on both sides.  Scores 1 apart keep the beams' order clear of it."""
    rng = np.random.default_rng(vocab)
    step = np.spacing(np.float32(abs(centre)))
    beams = 5
    logits = np.float32(centre) + step * rng.integers(-6, 1, (2 * beams, vocab)).astype(np.float32)
    assert logits.dtype == np.float32
    scores = -np.arange(2 * beams, dtype=np.float32).reshape(2, beams) * 1.25
    allowed = rng.random(vocab) < 0.9
    got = decoding.beam_select(torch.from_numpy(logits).cuda(), torch.from_numpy(scores).cuda(), None,
                               torch.from_numpy(allowed).cuda(), None, 0)
    want = select_64(logits, scores, None, allowed, None, 0)
    np.testing.assert_allclose(got[0].cpu().numpy(), want[0], rtol=2.0 ** -23, atol=2.0 ** -20)
    for have, need in zip(got[1:], want[1:]):
        assert np.array_equal(have.cpu().numpy(), need)


@pytest.mark.parametrize('vocab', [70, 264, 5000])
def test_select_masks_and_bad_values(vocab):
    rng, logits, scores = inputs(vocab, 6, 5, vocab)
    big = torch.finfo(torch.float32)
    logits[0, 3] = float('nan')                 # one beam's distribution is undefined
    logits[6] = float('nan')
    logits[8, 1], logits[9, 2] = float('inf'), -float('nan')
    logits[10] = -float('inf')                  # a beam with no token
    logits[11, 1:] = -float('inf')              # a beam with one
    logits[12] = big.min                        # the type's lowest value everywhere
    logits[13, ::2] = big.min
    logits[14, 4] = big.max
    scores[3, 0], scores[3, 1], scores[3, 2] = float('nan'), float('inf'), -float('inf')
    scores[4] = -float('inf')                   # a group with no beam
    scores[5] = torch.tensor([-1e30, -3e38, 0.0, -1e-30, -5.0])
    check_select(logits, scores)
    finished = torch.from_numpy(rng.random((6, 5)) < 0.4)
    check_select(logits, scores, finished, end=3, pad=vocab - 1)
    check_select(logits, scores, finished, torch.zeros(vocab, dtype=torch.bool), end=3, pad=1)   # nothing may follow
    only = torch.zeros(vocab, dtype=torch.bool)
    only[vocab // 2] = True
    check_select(logits, scores, None, only, end=vocab // 2)
    # NaN and infinity where the mask forbids them do not count.
    allowed = torch.ones(vocab, dtype=torch.bool)
    allowed[1:5] = False
    check_select(logits, scores, finished, allowed)
    check_select(logits, scores, torch.ones((6, 5), dtype=torch.bool))


@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('vocab,offset,pad', [(264, 1, 0), (264, 3, 5), (5001, 1, 2), (5001, 2, 2)])
def test_select_strided(vocab, offset, pad, dtype):
    rng, logits, scores = inputs(3, 4, 6, vocab + offset + pad, TYPES[dtype])
    check_select(logits.cuda()[:, offset:offset + vocab], scores)


def test_select_many_groups():
    rng, logits, scores = inputs(11, 700, 3, 264)
    finished = torch.from_numpy(rng.random((700, 3)) < 0.2)
    check_select(logits, scores, finished, end=5)


def test_select_in_place_and_repeats():
    """Scores and flags written over the inputs at the C boundary; the same bits every time."""
    from neurogen_b200 import library
    from neurogen_b200._lib import check
    for vocab in (264, 6000):
        rng, logits, scores = inputs(2, 9, 5, vocab)
        finished = torch.from_numpy(rng.random((9, 5)) < 0.3)
        want = decoding.beam_select(logits.cuda(), scores.cuda(), finished.cuda(), None, 7, 0)
        x, s, f = logits.cuda(), scores.cuda(), finished.cuda()
        tokens, parents = torch.empty((2, 9, 5), dtype=torch.int32, device='cuda')
        need = library().ng_beam_workspace(9, 5, vocab)
        work = torch.empty(max(need, 16), dtype=torch.uint8, device='cuda')
        check(library().ng_beam_select(0, x.data_ptr(), 0, vocab, 9, 5, vocab, s.data_ptr(), f.data_ptr(), None, 7, 0,
                                       s.data_ptr(), tokens.data_ptr(), parents.data_ptr(), f.data_ptr(),
                                       work.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
        for a, b in zip((s, tokens, parents, f), want):
            assert torch.equal(a, b)
        for _ in range(3):
            again = decoding.beam_select(logits.cuda(), scores.cuda(), finished.cuda(), None, 7, 0)
            assert all(torch.equal(a, b) for a, b in zip(again, want))


def test_select_empty():
    s, t, p, f = decoding.beam_select(torch.zeros(0, 264).cuda(), torch.zeros(0, 4).cuda())
    assert s.shape == t.shape == p.shape == f.shape == (0, 4)


def reorder_plain(states, parents):
    groups, beams = parents.shape
    rows = (np.arange(groups)[:, None] * beams + parents).reshape(-1)
    return states[torch.from_numpy(rows)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.uint8, torch.float64])
@pytest.mark.parametrize('groups,beams,size', [(1, 1, 5), (3, 2, 1), (2, 4, 704), (1, 5, 37), (7, 8, 1023), (2, 9, 260),
                                               (3, 16, 513), (2, 17, 4096), (5, 32, 333), (2, 2, 9001), (3, 4, 20000),
                                               (2, 8, 12000), (300, 3, 64)])
def test_reorder(groups, beams, size, dtype):
    rng = np.random.default_rng(size)
    states = torch.from_numpy(rng.integers(0, 200, (groups * beams + 2, size))).to(dtype)
    for parents in (rng.integers(0, beams, (groups, beams)), np.tile(np.arange(beams), (groups, 1)),
                    np.stack([rng.permutation(beams) for _ in range(groups)]), np.zeros((groups, beams), np.int64),
                    np.tile(np.arange(beams)[::-1], (groups, 1))):
        device = states.cuda()
        got = decoding.reorder(device[:groups * beams], torch.from_numpy(parents.copy()).int().cuda())
        assert got.data_ptr() == device.data_ptr()
        assert torch.equal(device[:groups * beams].cpu(), reorder_plain(states[:groups * beams], parents))
        assert torch.equal(device[groups * beams:].cpu(), states[groups * beams:])   # rows behind the last group


def test_reorder_far_rows():
    """Rows whose offsets pass 32 bits."""
    n = 1_500_000_016
    states = torch.zeros((3, n), dtype=torch.uint8, device='cuda')
    at = torch.tensor([0, 1, 77_777, n // 2, n - 2, n - 1], device='cuda')
    for w in range(3):
        states[w, at] = torch.arange(6, dtype=torch.uint8, device='cuda') + 10 * w + 1
    decoding.reorder(states, torch.tensor([[2, 0, 0]], dtype=torch.int32, device='cuda'))
    assert states[:, at].cpu().tolist() == [[21 + i for i in range(6)], [1 + i for i in range(6)], [1 + i for i in range(6)]]
    assert states[0].sum(dtype=torch.int64).item() == sum(21 + i for i in range(6))


def test_reorder_strided_and_shaped():
    rng = np.random.default_rng(1)
    whole = torch.from_numpy(rng.normal(size=(12, 50))).float()
    parents = rng.integers(0, 4, (3, 4))
    for lo, hi in ((0, 50), (1, 50), (4, 40), (3, 4)):
        device = whole.cuda()
        decoding.reorder(device[:, lo:hi], torch.from_numpy(parents).int().cuda())
        want = whole.clone()
        want[:, lo:hi] = reorder_plain(whole[:, lo:hi], parents)
        assert torch.equal(device.cpu(), want)
    cube = torch.arange(12 * 6).view(12, 2, 3)
    got = decoding.reorder(cube.cuda(), torch.from_numpy(parents).int().cuda())
    assert torch.equal(got.cpu(), reorder_plain(cube, parents))


def test_reorder_leaves_rows_with_a_parent_outside_the_group():
    states = torch.arange(8.0).view(4, 2)
    parents = torch.tensor([[1, -1, 4, 2]], dtype=torch.int32)
    got = decoding.reorder(states.cuda(), parents.cuda()).cpu()
    assert torch.equal(got, states[[1, 1, 2, 2]])


def test_streams_and_graphs():
    """A captured step (selection and reordering) replayed on new inputs, and two streams at once."""
    for vocab in (264, 7000):
        rng, logits, scores = inputs(5, 6, 4, vocab)
        other = inputs(6, 6, 4, vocab)[1]
        x, s = logits.cuda(), scores.cuda()
        states = torch.randn(24, 300, device='cuda')
        before = states.clone()
        decoding.reorder(before.clone(), decoding.beam_select(x, s, pad=0)[2])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = decoding.beam_select(x, s, pad=0)
            decoding.reorder(states, out[2])
        for values in (logits, other):
            x.copy_(values)
            states.copy_(before)
            graph.replay()
            want = decoding.beam_select(values.cuda(), s, pad=0)
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            assert torch.equal(states, decoding.reorder(before.clone(), want[2]))
        torch.cuda.synchronize()
        got = []
        for k, values in enumerate((logits.cuda(), other.cuda())):
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got.append([decoding.beam_select(values, s, pad=0) for _ in range(20)])
        torch.cuda.synchronize()
        for values, outs in zip((logits.cuda(), other.cuda()), got):
            want = decoding.beam_select(values, s, pad=0)
            assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want))


def test_refusals():
    x, s = torch.zeros(8, 300, device='cuda'), torch.zeros(2, 4, device='cuda')
    flag = torch.zeros((2, 4), dtype=torch.bool, device='cuda')
    p = torch.zeros((2, 4), dtype=torch.int32, device='cuda')
    for call, text in [
        (lambda: decoding.beam_select(x.double(), s), 'float32'),
        (lambda: decoding.beam_select(x.t(), s), 'adjacent'),
        (lambda: decoding.beam_select(x[:7], s), 'one row of logits'),
        (lambda: decoding.beam_select(x[:1].expand(8, 300), s), 'Row stride'),
        (lambda: decoding.beam_select(x, s.double()), 'scores'),
        (lambda: decoding.beam_select(x, s.t()), 'scores|row of logits'),
        (lambda: decoding.beam_select(torch.zeros(33, 300, device='cuda'), torch.zeros(1, 33, device='cuda')), '1..32'),
        (lambda: decoding.beam_select(x, s, flag.int()), 'finished'),
        (lambda: decoding.beam_select(x, s, None, torch.ones(299, dtype=torch.bool, device='cuda')), 'allowed'),
        (lambda: decoding.beam_select(x, s, end=300), 'End token'), (lambda: decoding.beam_select(x, s, pad=300), 'Padding'),
        (lambda: decoding.beam_select(x[:, :0], s, pad=0), 'Vocabulary'),
        (lambda: decoding.reorder(x, p.long()), 'parents'), (lambda: decoding.reorder(x[:6], p), 'one row of states'),
        (lambda: decoding.reorder(x.t()[:8], p), 'contiguous'),
        (lambda: decoding.reorder(x[:1].expand(8, 300), p), 'Row stride'),
    ]:
        with pytest.raises(ValueError, match=text):
            call()


# -- over a session pool ---------------------------------------------------------------------

CONFIG = LanguageConfig(columns=4, width=32, regions=2, ticks=2, idle_steps=1)


def pool_model(seed=3):
    weights = init_packed_weights(CONFIG, seed=seed)
    rng = np.random.default_rng(seed)
    return NativeLanguageModel(CONFIG, (weights + rng.normal(0, 0.1, weights.size)).astype(np.float32))


def test_pool_reorder():
    model = pool_model()
    pool = SessionPool(model, 6)
    rng = np.random.default_rng(0)
    for _ in range(3):
        pool.step(rng.integers(0, 264, 6))
    before, logits = pool.states(), pool.logits.copy()
    pool.reorder(3, [[2, 0, 0], [1, 1, 2]])
    rows = [2, 0, 0, 4, 4, 5]
    assert np.array_equal(pool.states(), before[rows]) and np.array_equal(pool.logits, logits[rows])
    for beams, parents, text in ((3, [[0, 1, 3], [0, 0, 0]], 'same group'), (3, [[0, -1, 2], [0, 0, 0]], 'same group'),
                                 (4, [[0, 0, 0, 0]], 'divide'), (3, [[0, 0, 0]], 'one parent'), (0, [[]], 'one parent')):
        with pytest.raises(ValueError, match=text):
            pool.reorder(beams, parents)
    assert np.array_equal(pool.states(), before[rows])


@pytest.mark.parametrize('groups,beams,steps', [(1, 4, 12), (3, 2, 7), (2, 1, 5), (5, 8, 6)])
def test_beam_search_equals_a_host_search(groups, beams, steps):
    """The device loop against the same search on the host: batched engine steps, the 64-bit
    selection, states gathered by hand."""
    model = pool_model(groups)
    rng = np.random.default_rng(beams)
    B = groups * beams
    prompts = rng.integers(0, 256, (groups, 4))
    allowed = np.ones(264, bool)
    allowed[256:] = False
    allowed[258] = True
    pool = SessionPool(model, B)
    first = rng.integers(0, 256, B)
    pool.step(first)                       # conversations under way: a group continues its first session
    start = pool.states().reshape(groups, beams, -1)
    tokens, scores = pool.beam_search(prompts, beams, steps, end=258, allowed=allowed)

    states = start[:, :1].repeat(beams, 1).reshape(B, -1)
    for t in range(prompts.shape[1]):
        logits, states, _, _ = model.engine.step_batch(prompts[:, t].repeat(beams), states)
    s = np.full((groups, beams), -np.inf, np.float32)
    s[:, 0] = 0
    done = np.zeros((groups, beams), bool)
    held = np.zeros((groups, beams, 0), np.int32)
    for _ in range(steps):
        s, tok, par, done = select_64(logits, s, done, allowed, 258, 256)
        held = np.concatenate([np.take_along_axis(held, par[:, :, None], 1), tok[:, :, None]], 2)
        rows = (np.arange(groups)[:, None] * beams + par).reshape(-1)
        logits, states, _, _ = model.engine.step_batch(tok.reshape(-1), states[rows])
    assert np.array_equal(tokens, held)
    np.testing.assert_allclose(scores, s, rtol=2.0 ** -22)
    assert np.array_equal(pool.states(), states) and np.array_equal(pool.logits, logits)
    assert len({tuple(row) for row in tokens[0]}) == beams   # different continuations


def test_beam_search_refusals():
    pool = SessionPool(pool_model(), 6)
    before = pool.states()
    for args, text in (((np.zeros((2, 3)), 3, 2, 264), 'End token'), ((np.zeros((2, 3)), 3, 2, None, np.ones(263, bool)), 'allowed'),
                       ((np.zeros((2, 3)), 3, 2, None, np.ones(264, np.int32)), 'allowed'),
                       ((np.zeros((2, 3)), 4, 2), 'divide'), ((np.zeros((2, 3)), 0, 2), 'divide'),
                       ((np.zeros((1, 3)), 3, 2), 'prompts'), ((np.zeros((2, 0)), 3, 2), 'prompts'),
                       ((np.full((2, 3), 264), 3, 2), '0..263'), ((np.zeros((2, 3)), 3, 0), 'one step')):
        with pytest.raises(ValueError, match=text):
            pool.beam_search(*args)
    assert np.array_equal(pool.states(), before)
