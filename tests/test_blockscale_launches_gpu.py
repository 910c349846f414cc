"""The 8-bit product on every launch that its plan can choose, each test naming the launch it means to
reach: results of every type with both epilogue terms, y = add, results inside a larger array, two
streams and graphs; and the language core's projections where they go to the tensor cores.

Bounds are those of tests/test_blockscale_gpu.py.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from neurogen_b200 import blockscale, library  # noqa: E402
from neurogen_b200._lib import check, stream_of  # noqa: E402
from neurogen_b200.language import LanguageConfig, NativeEngine, SessionPool, init_packed_weights  # noqa: E402
from neurogen_b200.language import NativeLanguageModel  # noqa: E402
from test_blockscale_gpu import BLOCK, TYPES, held, nearest_e4m3, product_64  # noqa: E402

# Kind (ng_block_matmul_kind): sizes.  Odd and ragged ones; results whose rows start on 16-byte
# boundaries and ones that do not; one block along k to several chunks of scales.
LAUNCHES = {
    8: [(1, 101, 141), (1, 2463, 140), (1, 768, 3200)],
    16: [(10, 1685, 148)],
    32: [(18, 1985, 140), (19, 2613, 140), (256, 384, 768)],
    32001: [(35, 2810, 150), (256, 928, 768)],
    32002: [(35, 1723, 2420), (35, 1724, 2420)],
    32004: [(120, 996, 1257), (120, 997, 1257), (128, 768, 3200)],
    32008: [(304, 124, 4364), (304, 125, 4364)],
    64001: [(150, 2636, 141), (150, 2637, 141)],
    64002: [(10, 4168, 4716), (10, 4167, 4716)],
    64004: [(35, 1374, 3293), (35, 1372, 3293), (256, 768, 3200)],
    64008: [(36, 816, 5984), (36, 815, 5984)],
    128001: [(277, 3297, 145), (277, 3296, 145), (2048, 768, 3200), (300, 3300, 2205)],
    256001: [(563, 4070, 141), (563, 4072, 141), (1020, 4090, 2205), (2300, 4090, 2205)],
}
CASES = [(kind, *size) for kind, sizes in LAUNCHES.items() for size in sizes]


def reached(kind, m, n, k):
    got = library().ng_block_matmul_kind(0, m, n, k)
    assert got == kind, f'{m} x {n} x {k} takes launch {got}, this test means {kind}'


def call(a, sa, w, sw, y, ldy, bias=None, add=None, scale=1.0):
    m, k = a.shape
    n = w.shape[0]
    code = blockscale.ELEMENTS[y.dtype]
    check(library().ng_block_matmul(0, a.data_ptr(), -(-k // 16) * 16, sa.data_ptr(), w.data_ptr(), -(-k // 16) * 16,
                                    sw.data_ptr(), m, n, k, None if bias is None else bias.data_ptr(),
                                    None if add is None else add.data_ptr(), n if add is None else add.stride(0), scale,
                                    y.data_ptr(), code, ldy, stream_of(a.device)))


def operands(m, n, k):
    gen = torch.Generator('cuda').manual_seed(m * n + k)
    x = torch.randn((m, k), generator=gen, device='cuda') * torch.randn((1, k), generator=gen, device='cuda').exp()
    w = torch.randn((n, k), generator=gen, device='cuda') * k ** -0.5
    return (*blockscale.quantize(x), *blockscale.quantize(w, 128)), gen


@pytest.mark.parametrize('kind,m,n,k', CASES)
def test_integers_exact(kind, m, n, k):
    """Small integers under power-of-two scales: every sum is exact in fp32, so the product must be."""
    reached(kind, m, n, k)
    rng = np.random.default_rng(m + 7 * n + 13 * k)
    a, w = rng.integers(-3, 4, (m, k)).astype(np.float64), rng.integers(-3, 4, (n, k)).astype(np.float64)
    kb = -(-k // BLOCK)
    sa, sw = 2.0 ** rng.integers(-2, 3, (m, kb)), 2.0 ** rng.integers(-2, 3, (-(-n // BLOCK), kb))
    x = a * sa.repeat(BLOCK, 1)[:, :k]
    z = w * sw.repeat(BLOCK, 0)[:n].repeat(BLOCK, 1)[:, :k]
    want = (torch.from_numpy(x).cuda() @ torch.from_numpy(z).cuda().T)
    got = blockscale.matmul(held(nearest_e4m3(a), 16), torch.from_numpy(sa).float().cuda(), held(nearest_e4m3(w)),
                            torch.from_numpy(sw).float().cuda())
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize('out', list(TYPES))
@pytest.mark.parametrize('kind,m,n,k', CASES)
def test_every_type_and_epilogue(kind, m, n, k, out):
    """Without an epilogue, with each term and with both; the memory term from a wider array, its rows on
    16-byte boundaries and not."""
    reached(kind, m, n, k)
    (a, sa, w, sw), gen = operands(m, n, k)
    kb = -(-k // BLOCK)
    product, magnitude = product_64(a, sa, w, sw)
    bias = torch.randn(n, generator=gen, device='cuda')
    wide = torch.randn((m, (n + 7) // 4 * 4 + 4), generator=gen, device='cuda')
    for b, start in ((None, None), (bias, None), (None, 4), (bias, 4), (bias, 1)):
        add = None if start is None else wide[:, start:start + n]
        want, size = product, magnitude
        if b is not None:
            want, size = want + b.double(), size + b.double().abs()
        if add is not None:
            want, size = want + 0.25 * add.double(), size + 0.25 * add.double().abs()
        got = blockscale.matmul(a, sa, w, sw, b, add, 0.25, TYPES[out])
        assert got.dtype == TYPES[out]
        bound = (128 + kb + 4) * 2.0 ** -23 * size + torch.finfo(TYPES[out]).eps / 2 * want.abs()
        if out == 'fp16':
            bound = bound + 2.0 ** -25   # half a step of its subnormals
        assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize('kind,m,n,k', CASES)
def test_result_may_overwrite_the_memory_term(kind, m, n, k):
    reached(kind, m, n, k)
    (a, sa, w, sw), gen = operands(m, n, k)
    add = torch.randn((m, n), generator=gen, device='cuda')
    bias = torch.randn(n, generator=gen, device='cuda')
    want = blockscale.matmul(a, sa, w, sw, bias, add, 0.5)
    call(a, sa, w, sw, add, n, bias, add, 0.5)
    assert torch.equal(add, want)


@pytest.mark.parametrize('out', list(TYPES))
@pytest.mark.parametrize('kind,m,n,k', CASES)
def test_rows_beside_and_behind_the_result_stay(kind, m, n, k, out):
    """Row strides that allow 16-byte stores and ones that do not."""
    reached(kind, m, n, k)
    (a, sa, w, sw), _ = operands(m, n, k)
    want = blockscale.matmul(a, sa, w, sw, out_dtype=TYPES[out])
    for ld in (-(-n // 8) * 8 + 8, n + 5):
        y = torch.full((m + 5, ld), 3.5, dtype=TYPES[out], device='cuda')
        call(a, sa, w, sw, y, ld)
        assert torch.equal(y[:m, :n], want)
        assert (y[m:] == 3.5).all() and (y[:, n:] == 3.5).all()


@pytest.mark.parametrize('kind,m,n,k', [(kind, *sizes[0]) for kind, sizes in LAUNCHES.items()])
def test_streams_and_graphs(kind, m, n, k):
    """Two streams at once, and a graph replayed on new inputs."""
    reached(kind, m, n, k)
    (a, sa, w, sw), _ = operands(m, n, k)
    want = blockscale.matmul(a, sa, w, sw)
    torch.cuda.synchronize()
    got = []
    for s in [torch.cuda.Stream() for _ in range(2)]:
        with torch.cuda.stream(s):
            got.append([blockscale.matmul(a, sa, w, sw) for _ in range(20)])
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for ys in got for y in ys)
    graph = torch.cuda.CUDAGraph()
    scale = sa.clone()
    with torch.cuda.graph(graph):
        y = blockscale.matmul(a, scale, w, sw)
    for factor in (1.0, -2.0):   # a power of two: every product and sum scales exactly
        scale.copy_(sa * factor)
        graph.replay()
        assert torch.equal(y, want * factor)


@pytest.fixture
def fp8(monkeypatch):
    monkeypatch.setenv('NEUROGEN_PROJECTION', 'fp8')


@pytest.mark.parametrize('idle', [False, True])
@pytest.mark.parametrize('batch,kinds', [(128, (32, 32, 32004)), (256, (32, 32001, 64004))])
def test_projections_of_many_sessions_against_the_equations(batch, kinds, idle, fp8):
    """The BC-250 region's input, feedback and output projections where the latter two or one go to the
    tensor cores, k range shared, with bias and memory term."""
    from test_projection_8bit_gpu import test_advance_against_the_equations as against_the_equations
    for kind, (n, k) in zip(kinds, ((384, 768), (928, 768), (768, 3200))):
        reached(kind, batch, n, k)
    against_the_equations(32, 768, batch, idle, None)


@pytest.mark.parametrize('batch', [1, 37, 256])
def test_a_token_step_takes_the_embeddings_of_its_tokens(batch, fp8):
    """A step's input projection gathers each session's row of the embedding: the same bits as an
    advance whose input is that row (and an advance is held to the equations)."""
    cfg = LanguageConfig(columns=32, width=768, regions=1, ticks=2, idle_steps=0)
    packed = init_packed_weights(cfg, seed=3)
    eng = NativeEngine(cfg, packed)
    rng = np.random.default_rng(batch)
    packed = np.asarray(packed, np.float32)
    tokens = rng.integers(0, 264, batch)
    state = rng.uniform(0, 0.5, (batch, eng.state_size)).astype(np.float32)
    embedding = packed[:264 * cfg.width].reshape(264, cfg.width)
    _, after_step, _, hidden_step = eng.step_batch(tokens, state)
    hidden, after, _ = eng.advance_batch(embedding[tokens], state, idle=False)
    assert np.array_equal(after_step, after) and np.array_equal(hidden_step, hidden)
    others = eng.step_batch((tokens + 1) % 264, state)[1]
    assert not np.array_equal(others, after_step)


def test_pool_of_256_sessions_equals_host_batches(fp8):
    """The captured step on the tensor-core launches, against host batches of the same size, bit for bit."""
    cfg = LanguageConfig()
    model = NativeLanguageModel(cfg, init_packed_weights(cfg, seed=2))
    pool = SessionPool(model, 256)
    state = np.zeros((256, model.engine.state_size), np.float32)
    rng = np.random.default_rng(0)
    for _ in range(3):
        tokens = rng.integers(0, 264, 256)
        logits, state, _, _ = model.engine.step_batch(tokens, state)
        assert np.array_equal(pool.step(tokens), logits)
    assert np.array_equal(pool.states(), state) and np.isfinite(state).all()
