"""A tensor-core product whose bounded wait runs out: who hears of it.

The test switch (NEUROGEN_TEST_MATMUL_STALL=1) makes the process's first tensor-core product take the
path of a wait that ran out, before it issues any copy or MMA, so each case is a process of its own.
A pool's step is captured at its first use, the switched product with it.
"""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

SETUP = r'''
import sys
sys.path[:0] = {paths!r}
import numpy as np, torch
from neurogen_b200 import blockscale
from neurogen_b200.language import LanguageConfig, NativeLanguageModel, SessionPool, init_packed_weights
TIMEOUT = 'An 8-bit product timed out'

def error_of(call):
    try:
        call()
    except ValueError as e:
        return str(e)
    return ''

def product(m=400, n=4096, k=512):
    gen = torch.Generator('cuda').manual_seed(1)
    a, sa = blockscale.quantize(torch.randn((m, k), generator=gen, device='cuda'))
    w, sw = blockscale.quantize(torch.randn((n, k), generator=gen, device='cuda'), 128)
    x = a.double() * sa.double().repeat_interleave(128, 1)
    z = w.double() * sw.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)
    return (a, sa, w, sw), x @ z.T

def right(y, want):   # (128 + 4 + 4) 2^-23 of the sum of magnitudes, below 512 * 0.64 * 3
    return bool(((y.double() - want).abs() < 136 * 2.0 ** -23 * 1000).all())

def model():   # sizes whose projections of 256 sessions go to the tensor cores
    cfg = LanguageConfig(columns=32, width=768, regions=1, ticks=1, idle_steps=0)
    return NativeLanguageModel(cfg, init_packed_weights(cfg, seed=0))

def device_step(pool, stream):
    tokens = torch.full((pool.sessions,), 5, dtype=torch.int32, device='cuda')
    torch.cuda.synchronize()
    assert pool.lib.ng_pool_step_device(pool.h, tokens.data_ptr(), None, stream.cuda_stream) == 0, pool.lib.ng_error()
    stream.synchronize()
'''


def run(tmp_path, body):
    script = tmp_path / 'child.py'
    script.write_text(SETUP.format(paths=[str(p) for p in sys.path[:3]]) + body + "\nprint('done')\n")
    env = dict(os.environ, NEUROGEN_TEST_MATMUL_STALL='1', NEUROGEN_PROJECTION='fp8')
    out = subprocess.run([sys.executable, str(script)], env=env, capture_output=True, text=True, timeout=120)
    assert out.returncode == 0 and out.stdout.endswith('done\n'), out.stdout + out.stderr[-3000:]


def test_a_standalone_product_is_asked_for_by_itself(tmp_path):
    """Without a further product, and once."""
    run(tmp_path, r'''
ops, want = product()
blockscale.check_products()
blockscale.matmul(*ops)
torch.cuda.synchronize()
assert TIMEOUT in error_of(blockscale.check_products)
blockscale.check_products('cuda:0')
assert right(blockscale.matmul(*ops), want)
''')


def test_a_pool_hears_of_its_own_products_only(tmp_path):
    """A standalone product, another pool and a host batch of the same engine run between the failure and
    the pool's check: none of them is refused or blamed, and the pool is told."""
    run(tmp_path, r'''
mod = model()
lost, other, stream = SessionPool(mod, 256), SessionPool(mod, 256), torch.cuda.Stream()
device_step(lost, stream)
ops, want = product()
assert right(blockscale.matmul(*ops), want)
blockscale.check_products()
tokens = np.full(256, 5)
logits = other.step(tokens)
state = np.zeros((256, mod.engine.state_size), np.float32)
assert np.array_equal(mod.engine.step_batch(tokens, state)[0], logits)
assert TIMEOUT in error_of(lambda: lost._check(lost.lib.ng_pool_check(lost.h)))
other._check(other.lib.ng_pool_check(other.h))
assert np.isfinite(other.step(tokens)).all()
''')


def test_a_host_batch_reports_its_own_product(tmp_path):
    run(tmp_path, r'''
mod = model()
tokens, state = np.full(256, 5), np.zeros((256, mod.engine.state_size), np.float32)
assert TIMEOUT in error_of(lambda: mod.engine.step_batch(tokens, state))
logits = mod.engine.step_batch(tokens, state)[0]
pool = SessionPool(mod, 256)
assert np.array_equal(pool.step(tokens), logits)
blockscale.check_products()
''')


@pytest.mark.parametrize('m,n,k', [(35, 2810, 150), (35, 1374, 3293), (304, 124, 4364), (277, 3297, 145), (563, 4070, 141)])
@pytest.mark.parametrize('code,dtype', [(0, 'float32'), (1, 'bfloat16'), (2, 'float16')])
def test_a_lost_result_reads_nan(tmp_path, m, n, k, code, dtype):
    """Tiles walked over and k ranges shared by a cluster; nothing beside or behind the result is written."""
    run(tmp_path, rf'''
m, n, k = {m}, {n}, {k}
from neurogen_b200 import library
a, sa = blockscale.quantize(torch.randn((m, k), device='cuda'))
w, sw = blockscale.quantize(torch.randn((n, k), device='cuda'), 128)
y = torch.full((m + 3, n + 5), 3.5, dtype=torch.{dtype}, device='cuda')
stream = torch.cuda.current_stream().cuda_stream
for lost in (True, False):
    code = library().ng_block_matmul(0, a.data_ptr(), a.stride(0), sa.data_ptr(), w.data_ptr(), w.stride(0), sw.data_ptr(),
                                     m, n, k, None, None, n, 1.0, y.data_ptr(), {code}, n + 5, stream)
    assert code == 0, library().ng_error()
    assert (torch.isnan if lost else torch.isfinite)(y[:m, :n]).all()
    assert (y[m:] == 3.5).all() and (y[:, n:] == 3.5).all()
    if lost:
        torch.cuda.synchronize()
        assert TIMEOUT in error_of(blockscale.check_products)
''')


@pytest.mark.parametrize('host', [True, False])
def test_a_pool_whose_projection_was_lost_refuses_its_states(tmp_path, host):
    """A projection feeds the states, in place: after one that gave up nothing uses them until they are
    set again, and then the pool steps as a fresh one does.  Another pool of the engine is not affected."""
    run(tmp_path, f'HOST = {host}' + r'''
mod = model()
pool, other = SessionPool(mod, 256), SessionPool(mod, 256)
start = np.random.default_rng(0).uniform(0, 0.4, (256, mod.engine.state_size)).astype(np.float32)
pool.set_states(start)
other.set_states(start)
tokens = np.full(256, 5)
if HOST:
    assert TIMEOUT in error_of(lambda: pool.step(tokens))
else:
    device_step(pool, torch.cuda.Stream())
    assert 'lost' in error_of(lambda: pool.step(tokens))   # heard before another step is enqueued
logits = other.step(tokens)
parents = np.zeros((64, 4), np.int32)
d_parents = torch.zeros((64, 4), dtype=torch.int32, device='cuda')
d_tokens = torch.full((256,), 5, dtype=torch.int32, device='cuda')
for call in (lambda: pool.step(tokens), pool.states, lambda: pool.reorder(4, parents),
             lambda: pool.beam_search(np.full((64, 1), 5), 4, 2),
             lambda: pool._check(pool.lib.ng_pool_step_device(pool.h, d_tokens.data_ptr(), None, None)),
             lambda: pool._check(pool.lib.ng_pool_reorder_device(pool.h, 4, d_parents.data_ptr(), None)),
             lambda: pool._check(pool.lib.ng_pool_check(pool.h))):
    message = error_of(call)
    assert 'states are lost' in message and 'load states' in message, message
assert error_of(lambda: pool.set_states(np.full_like(start, np.nan))) and 'lost' in error_of(pool.states)
pool.set_states(start)
assert np.array_equal(pool.states(), start)
assert np.array_equal(pool.step(tokens), logits)
pool._check(pool.lib.ng_pool_check(pool.h))
assert np.array_equal(pool.states(), other.states())
''')
