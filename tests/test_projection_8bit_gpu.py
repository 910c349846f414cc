"""The engine's opt-in 8-bit projections (NEUROGEN_PROJECTION=fp8).

One advance of a one-region core is recomputed here in 64 bits from the model's equations
(oracle/lang_oracle.c region_step) with the projections' operands rounded to 8 bits as
blockscale.quantize rounds them.  The inputs of the first two projections are known exactly; those of
the output projection are taken from the engine's own next state, so every 8-bit rounding here
is the engine's.  What is left is fp32 arithmetic: a projection's relative error against the
sum of magnitudes is at most (128 + kb + 4) 2^-23 (tests/test_blockscale_gpu.py), below 2e-5 of
it, and the membrane's and LayerNorm's roundings are below 1e-5 of their terms; units whose
potential lies within 1e-3 of the threshold may spike either way and are left out.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from neurogen_b200 import blockscale  # noqa: E402
from neurogen_b200.language import (LanguageConfig, NativeEngine, NativeLanguageModel, SessionPool,  # noqa: E402
                                    canonical_buffers, init_packed_weights, unit_tables)
from test_decoding_gpu import select_64  # noqa: E402


@pytest.fixture
def fp8(monkeypatch):
    monkeypatch.setenv('NEUROGEN_PROJECTION', 'fp8')


def rounded(x, rows):
    """The values that x [m, k] stands for after quantisation, in 64 bits."""
    q, s = blockscale.quantize(torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda(), rows)
    m, k = q.shape
    return (q.double() * s.double().repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]).cpu().numpy()


def unpacked(cfg, packed):
    """The region's parameters from the packed stream (one region)."""
    c, w = cfg.columns, cfg.width
    sizes = dict(emb=264 * w, rec=c * 4096, in_w=c * 12 * w, in_b=c * 12, fb_w=c * 29 * w, out_w=w * c * 100, out_b=w,
                 norm_w=w, norm_b=w, decay=w)
    out, at = {}, 0
    for name, size in sizes.items():
        out[name] = packed[at:at + size].astype(np.float64)
        at += size
    return out


@pytest.mark.parametrize('idle', [False, True])
@pytest.mark.parametrize('columns,width,batch', [(1, 16, 1), (3, 40, 1), (3, 200, 5), (8, 129, 37), (5, 768, 70)])
def test_advance_against_the_equations(columns, width, batch, idle, fp8):
    cfg = LanguageConfig(columns=columns, width=width, regions=1, ticks=1, idle_steps=0)
    c, n = columns, columns * 64
    rng = np.random.default_rng(columns * 1000 + width)
    packed = init_packed_weights(cfg, seed=columns)
    packed = (packed + rng.normal(0, 0.05, packed.size)).astype(np.float32)
    eng = NativeEngine(cfg, packed)
    p = unpacked(cfg, packed)
    f32 = lambda v: v.astype(np.float32)  # noqa: E731
    V, trace = f32(rng.uniform(-0.5, 0.9, (batch, n))), f32(rng.random((batch, n)))
    adapt, last = f32(0.1 * rng.random((batch, n))), f32(rng.random((batch, n)) < 0.2)
    mem, counts = f32(rng.normal(size=(batch, width))), f32(rng.integers(0, 9, (batch, n)))
    state = np.concatenate([V, trace, adapt, last, mem, counts], 1)
    x = f32(rng.normal(size=(batch, width)))
    hidden, after, _ = eng.advance_batch(x, state, idle=idle)
    got = dict(zip(('V', 'trace', 'adapt', 'last', 'mem', 'counts'),
                   np.split(after.astype(np.float64), np.cumsum([n, n, n, n, width]), 1)))

    _, exc, in_ids, fb_ids, out_ids = unit_tables()
    buf = canonical_buffers()
    excs = np.tile(exc, c)
    current = np.tile(np.where(excs, 0.15, 0.35), (batch, 1))
    cols = np.arange(c)[:, None] * 64
    slack = np.zeros((batch, n))
    if not idle:
        w8 = rounded(p['in_w'].reshape(c * 12, width), 128)
        v = rounded(x, 1) @ w8.T + p['in_b']
        size = np.abs(rounded(x, 1)) @ np.abs(w8).T + np.abs(p['in_b'])
        current[:, (cols + in_ids).reshape(-1)] = 3 / (1 + np.exp(-v))
        slack[:, (cols + in_ids).reshape(-1)] += 0.75 * 2e-5 * size
    w8 = rounded(p['fb_w'].reshape(c * 29, width), 128)
    v = rounded(mem, 1) @ w8.T
    size = np.abs(rounded(mem, 1)) @ np.abs(w8).T
    current[:, (cols + fb_ids).reshape(-1)] += 0.5 * np.tanh(v)
    slack[:, (cols + fb_ids).reshape(-1)] += 0.5 * 2e-5 * size
    raw = p['rec'].reshape(c, 64, 64)
    gain = np.logaddexp(0, raw) * buf['mask'].numpy() * buf['sign'].numpy()[None, None, :]
    t = trace.astype(np.float64).reshape(batch, c, 64)
    rec = np.einsum('coi,bci->bco', gain, t).reshape(batch, n)
    near = np.zeros_like(t)
    near[:, 1:] += t[:, :-1]
    near[:, :-1] += t[:, 1:]
    near = near.reshape(batch, n) * excs
    decay = np.where(excs, 0.6, 0.4)
    v = decay * V + (1 - decay) * (current + rec + 0.08 * near)
    margin = v - np.where(excs, 1.0, 0.6) - adapt
    spike = (margin >= 0) * (1 - last)
    sure = np.abs(margin) > 1e-3
    assert sure.mean() > 0.97 and 0.01 < spike.mean() < 0.9
    tol = slack + 1e-5 * (np.abs(v) + np.abs(rec) + 1)
    np.testing.assert_array_equal(got['last'][sure], spike[sure])
    assert (np.abs(got['V'] - v * (1 - spike)) <= tol)[sure].all()
    assert (np.abs(got['trace'] - (0.8 * trace + 0.2 * spike)) <= 1e-6)[sure].all()

    # Output projection, from the engine's own potentials and traces.
    ids = (cols + out_ids).reshape(-1)
    feat = np.concatenate([got['V'][:, ids], got['trace'][:, ids]], 1)
    w8 = rounded(p['out_w'].reshape(width, c * 100), 128)
    raw = rounded(feat, 1) @ w8.T + p['out_b'] + 0.25 * mem
    size = np.abs(rounded(feat, 1)) @ np.abs(w8).T + np.abs(p['out_b']) + 0.25 * np.abs(mem)
    centred = raw - raw.mean(1, keepdims=True)
    inv = 1 / np.sqrt((centred ** 2).mean(1, keepdims=True) + 1e-5)
    h = centred * inv * p['norm_w'] + p['norm_b']
    # A shift of every raw value by up to e moves a normalised one by at most 2 e inv (1 + |h0|).
    e = 2e-5 * size.max(1, keepdims=True)
    tol = 2 * e * inv * (1 + np.abs(centred * inv)) * np.abs(p['norm_w']) + 1e-5 * (1 + np.abs(h))
    assert (np.abs(hidden - h) <= tol).all()
    keep = 0.5 + 0.499 / (1 + np.exp(-p['decay']))
    assert (np.abs(got['mem'] - (keep * mem + (1 - keep) * hidden)) <= 1e-5 * (1 + np.abs(mem) + np.abs(h))).all()


def test_exact_projections_are_the_default(monkeypatch):
    cfg = LanguageConfig(columns=2, width=32, regions=2, ticks=2, idle_steps=1)
    w = init_packed_weights(cfg, seed=1)
    toks, s = np.array([3, 4, 5]), None
    out = {}
    for mode in (None, 'fp8', 'other', None):
        if mode is None:
            monkeypatch.delenv('NEUROGEN_PROJECTION', raising=False)
        else:
            monkeypatch.setenv('NEUROGEN_PROJECTION', mode)
        eng = NativeEngine(cfg, w)
        s = np.zeros((3, eng.state_size), np.float32)
        got = eng.step_batch(toks, s)
        out.setdefault(mode, got)
        if mode is None:
            assert all(np.array_equal(a, b) for a, b in zip(out[None], got))
    assert all(np.array_equal(a, b) for a, b in zip(out[None], out['other']))
    assert not np.array_equal(out[None][3], out['fp8'][3])


@pytest.mark.parametrize('cfg', [LanguageConfig(columns=3, width=17, regions=2, ticks=3, idle_steps=1),
                                 LanguageConfig(columns=4, width=32, regions=5, ticks=2, idle_steps=1), LanguageConfig()])
def test_pools_and_static_steps_agree(cfg, fp8):
    """A pool (captured, replayed) and a host batch of the same size give the same bits; so do ng_step
    and ng_step_static."""
    w = init_packed_weights(cfg, seed=2)
    model = NativeLanguageModel(cfg, w)
    eng = model.engine
    pool = SessionPool(model, 7)
    s = np.zeros((7, eng.state_size), np.float32)
    rng = np.random.default_rng(0)
    for _ in range(4):
        toks = rng.integers(0, 264, 7)
        logits, s, _, _ = eng.step_batch(toks, s)
        assert np.array_equal(pool.step(toks), logits)
    assert np.array_equal(pool.states(), s) and np.isfinite(s).all()
    one, two = np.zeros(eng.state_size, np.float32), np.zeros(eng.state_size, np.float32)
    for token in (257, 104, 9):
        outs = []
        for fn, state in ((eng.lib.ng_step, one), (eng.lib.ng_step_static, two)):
            nxt, logits = np.empty(eng.state_size, np.float32), np.empty(264, np.float32)
            h, a = np.empty(cfg.width, np.float32), np.empty(1, np.float32)
            assert fn(eng.handle, token, state, state.size, nxt, logits, h, a) == 0, eng.lib.ng_error().decode()
            outs.append((nxt, logits, h, a))
        assert all(np.array_equal(x, y) for x, y in zip(*outs))
        one, two = outs[0][0], outs[1][0]


def test_beam_search_with_8bit_projections(fp8):
    """The decoding operators together: 8-bit steps, selection and reordering on the device against the
    same search on the host."""
    cfg = LanguageConfig(columns=4, width=48, regions=2, ticks=2, idle_steps=1)
    rng = np.random.default_rng(5)
    weights = init_packed_weights(cfg, seed=5)
    model = NativeLanguageModel(cfg, (weights + rng.normal(0, 0.1, weights.size)).astype(np.float32))
    groups, beams, steps = 3, 6, 8
    prompts = rng.integers(0, 256, (groups, 5))
    pool = SessionPool(model, groups * beams)
    tokens, scores = pool.beam_search(prompts, beams, steps, end=258)
    states = np.zeros((groups * beams, model.engine.state_size), np.float32)
    for t in range(prompts.shape[1]):
        logits, states, _, _ = model.engine.step_batch(prompts[:, t].repeat(beams), states)
    s = np.full((groups, beams), -np.inf, np.float32)
    s[:, 0] = 0
    done = np.zeros((groups, beams), bool)
    held = np.zeros((groups, beams, 0), np.int32)
    for _ in range(steps):
        s, tok, par, done = select_64(logits, s, done, None, 258, 256)
        held = np.concatenate([np.take_along_axis(held, par[:, :, None], 1), tok[:, :, None]], 2)
        rows = (np.arange(groups)[:, None] * beams + par).reshape(-1)
        logits, states, _, _ = model.engine.step_batch(tok.reshape(-1), states[rows])
    assert np.array_equal(tokens, held) and np.array_equal(pool.states(), states)
    np.testing.assert_allclose(scores, s, rtol=2.0 ** -22)


STALL_CHILD = r'''
import sys
sys.path[:0] = {paths!r}
import torch
from neurogen_b200 import blockscale
w, sw = blockscale.quantize(torch.randn({n}, {k}, device='cuda'), 128)
x = torch.randn({m}, {k}, device='cuda')
blockscale.linear(x, w, sw)
torch.cuda.synchronize()
try:
    blockscale.linear(x, w, sw)
    print('no error')
except ValueError as e:
    print('raised:', e)
q, s = blockscale.quantize(x)
want = (q.double() * s.double().repeat_interleave(128, 1)[:, :{k}]) @ (w.double() * sw.double().repeat_interleave(128, 0)[:{n}].repeat_interleave(128, 1)[:, :{k}]).T
y = blockscale.linear(x, w, sw)
print('after:', bool(((y.double() - want).abs() < 1e-2).all()))
'''


@pytest.mark.parametrize('m,n,k', [(400, 4096, 512), (2048, 4096, 512), (128, 768, 3200)])
def test_a_wait_that_runs_out_is_reported(tmp_path, m, n, k):
    """The tensor-core product's waits are bounded.  A test switch makes the first launch take the
    path of a wait that ran out before it issues any copy or MMA: the next call reports it, and the one
    after runs normally.  The sizes are the tensor-core kernel's (the few-row kernel has no waits): tiles
    walked over, and a k range split over a cluster."""
    import os
    import subprocess
    import sys
    script = tmp_path / 'stall.py'
    script.write_text(STALL_CHILD.format(paths=[str(p) for p in sys.path[:3]], m=m, n=n, k=k))
    env = dict(os.environ, NEUROGEN_TEST_MATMUL_STALL='1')
    out = subprocess.run([sys.executable, str(script)], env=env, capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stderr[-3000:]
    assert 'raised: An 8-bit product timed out' in out.stdout and 'after: True' in out.stdout, out.stdout
