"""8-bit block-scaled quantisation and product on the GPU, against their definitions in 64 bits.

Quantisation has one right answer, byte for byte: both divisions are single fp32 roundings (a
64-bit quotient of two fp32 numbers, rounded to fp32, is that rounding) and the byte is the
nearest e4m3 value, ties to even.

The product's tolerance: products of two e4m3 values are exact in fp32.  A block of 128 of them
is summed with at most 128 additions, each off by at most 2^-23 of the sum of magnitudes (a
truncating adder; 2^-24 for a rounding one), the scale product and its use are two roundings,
and the kb blocks, bias and memory term kb + 2 more additions: (128 + kb + 4) 2^-23 of the sum of
magnitudes, plus half a step of the result's type.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from neurogen_b200 import blockscale  # noqa: E402

TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
BLOCK = 128

E4M3 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
POSITIVE = E4M3[:127]   # 0 .. 448 ascending; 127 is NaN


def nearest_e4m3(v):
    """Byte of the nearest e4m3 value (ties to the even byte) of finite float64 |v| <= 464."""
    a = np.abs(v)
    hi = np.searchsorted(POSITIVE, a).clip(0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - POSITIVE[lo], POSITIVE[hi] - a
    byte = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (byte | np.where(np.signbit(v), 128, 0)).astype(np.uint8)


def quantize_64(x, rows):
    """(bytes, scale) of a float64 matrix that holds fp32 values."""
    m, k = x.shape
    mb, kb = -(-m // rows), -(-k // BLOCK)
    q, scale = np.zeros((m, k), np.uint8), np.zeros((mb, kb), np.float32)
    for i in range(mb):
        for j in range(kb):
            part = x[i * rows:(i + 1) * rows, j * BLOCK:(j + 1) * BLOCK]
            s = max(np.float32(np.abs(part).max() / 448.0), np.float32(2.0 ** -126))
            scale[i, j] = s
            v = (part / np.float64(s)).astype(np.float32).astype(np.float64)
            q[i * rows:(i + 1) * rows, j * BLOCK:(j + 1) * BLOCK] = nearest_e4m3(v)
    return q, scale


def bytes_of(q):
    return q.contiguous().view(torch.uint8).cpu().numpy()


def wide_values(seed, m, k, dtype):
    rng = np.random.default_rng(seed)
    x = rng.normal(size=(m, k)) * np.exp(rng.normal(size=(m, 1)) + rng.normal(size=(1, k)))
    return torch.from_numpy(x).to(dtype)


@pytest.mark.parametrize('rows', [1, 128])
@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('m,k', [(1, 1), (1, 3), (1, 127), (2, 128), (3, 129), (5, 700), (127, 260), (128, 256),
                                 (129, 131), (300, 1030)])
def test_quantize_is_exact(m, k, dtype, rows):
    x = wide_values(m * 1000 + k, m, k, TYPES[dtype])
    q, scale = blockscale.quantize(x.cuda(), rows)
    want_q, want_scale = quantize_64(x.double().numpy(), rows)
    assert q.shape == (m, k) and q.dtype == torch.float8_e4m3fn and q.data_ptr() % 16 == 0
    assert np.array_equal(scale.cpu().numpy(), want_scale)
    assert np.array_equal(bytes_of(q), want_q)


@pytest.mark.parametrize('rows', [1, 128])
@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('offset,pad', [(1, 0), (3, 4), (4, 4), (2, 1)])
def test_quantize_strided(offset, pad, dtype, rows):
    """Column slices: any start, any stride, and a tensor whose rows lie further apart than its columns."""
    m, k = 37, 389
    x = wide_values(5, m, k + offset + pad, TYPES[dtype])
    view = x.cuda()[:, offset:offset + k]
    q, scale = blockscale.quantize(view, rows)
    want_q, want_scale = quantize_64(x[:, offset:offset + k].double().numpy(), rows)
    assert np.array_equal(scale.cpu().numpy(), want_scale) and np.array_equal(bytes_of(q), want_q)


@pytest.mark.parametrize('rows', [1, 128])
def test_quantize_edges(rows):
    """Zeros, the smallest and largest fp32 numbers, signed zeros, and values on e4m3's ties."""
    x = torch.zeros(6, 256)
    x[1, :128] = 2.0 ** -149 * torch.arange(128)
    x[1, 128:] = 3.4e38 * torch.linspace(-1, 1, 128)
    x[2, 0], x[2, 1] = 448.0, -0.0
    x[2, 2:10] = torch.tensor([17.0, 19.0, 21.0, -17.0, 2.0 ** -10, 3 * 2.0 ** -10, 464.0 / 1.05, 2.0 ** -9])
    x[4, 5] = 1e-37
    q, scale = blockscale.quantize(x.cuda(), rows)
    want_q, want_scale = quantize_64(x.double().numpy(), rows)
    assert np.array_equal(scale.cpu().numpy(), want_scale) and np.array_equal(bytes_of(q), want_q)


@pytest.mark.parametrize('rows', [1, 128])
@pytest.mark.parametrize('dtype', list(TYPES))
def test_quantize_zeros_and_underflow_keep_their_sign(dtype, rows):
    """Zeros of either sign, and values whose quotient rounds to zero, next to values of many scales
    (the reciprocal of a scale may be rounded up or down)."""
    x = wide_values(5, 130, 128 * 40, TYPES[dtype])
    x[:, 3::16] = 0.0
    x[:, 5::16] = -0.0
    x[:, 7::16] *= 2.0 ** -12
    x[:, 9::16] *= torch.finfo(TYPES[dtype]).tiny
    q, scale = blockscale.quantize(x.cuda(), rows)
    want_q, want_scale = quantize_64(x.double().numpy(), rows)
    assert np.array_equal(scale.cpu().numpy(), want_scale)
    assert np.array_equal(bytes_of(q), want_q)


@pytest.mark.parametrize('dtype', list(TYPES))
def test_quantize_16_bit_extremes(dtype):
    """A NaN of either sign, infinities and the type's largest value, in both block shapes."""
    info = torch.finfo(TYPES[dtype])
    x = wide_values(3, 130, 260, TYPES[dtype])
    x[1, 3], x[2, 130], x[129, 259], x[0, 5] = float('nan'), -float('inf'), info.max, -info.max
    x[3, 200] = torch.tensor(-float('nan'))
    for rows in (1, 128):
        for view in (x.cuda(), torch.cat([x[:, :1], x], 1).cuda()[:, 1:]):
            q, s = blockscale.quantize(view, rows)
            bad = torch.zeros(130, 260, dtype=torch.bool)
            bad[1, 3] = bad[2, 130] = bad[3, 200] = True
            per = bad.float().new_zeros(-(-130 // rows) * rows, 384)
            per[:130, :260] = bad.float()
            per = per.view(-1, rows, 3, 128).amax((1, 3)) > 0
            assert torch.equal(torch.isfinite(s.cpu()), ~per)
            want_q, want_s = quantize_64(torch.where(bad, 0, x).double().numpy(), rows)
            ok = ~per.repeat_interleave(rows, 0)[:130].repeat_interleave(128, 1)[:, :260].numpy()
            assert np.array_equal(bytes_of(q)[ok], want_q[ok])
            assert np.array_equal(s.cpu().numpy()[~per.numpy()], want_s[~per.numpy()])


def test_matmul_far_rows():
    """A result whose offsets pass 32 bits, against 64 bits at its corners."""
    m, n, k = 70_000, 40_000, 32
    gen = torch.Generator(device='cuda').manual_seed(1)
    a, sa = blockscale.quantize(torch.randn((m, k), generator=gen, device='cuda'))
    w, sw = blockscale.quantize(torch.randn((n, k), generator=gen, device='cuda'), 128)
    y = blockscale.matmul(a, sa, w, sw, out_dtype=torch.bfloat16)
    for rows in (slice(0, 200), slice(35_000, 35_100), slice(m - 130, m)):
        want, size = product_64(a[rows], sa[rows], w, sw)
        assert ((y[rows].double() - want).abs() <= (128 + 1 + 4) * 2.0 ** -23 * size + 2.0 ** -8 * want.abs()).all()


def test_quantize_non_finite():
    x = wide_values(1, 4, 300, torch.float32)
    x[1, 10] = float('nan')
    x[2, 200] = float('-inf')
    q, scale = blockscale.quantize(x.cuda())
    s, v = scale.cpu(), q.float().cpu()
    assert torch.isnan(s[1, 0]) and torch.isnan(v[1, :128]).all()
    assert torch.isinf(s[2, 1]) and torch.isnan(v[2, 200]) and (v[2, 128:200] == 0).all()
    keep = torch.ones_like(s, dtype=torch.bool)
    keep[1, 0] = keep[2, 1] = False
    assert torch.isfinite(s[keep]).all()
    w, ws = blockscale.quantize(wide_values(2, 50, 300, torch.float32).cuda(), 128)
    y = blockscale.matmul(q, scale, w, ws).cpu()
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 3]]).all()


def held(values_u8, pad=0):
    """Bytes with rows on 16-byte boundaries; `pad` more columns of NaN bytes between the rows."""
    m, k = values_u8.shape
    ld = -(-(k + pad) // 16) * 16
    t = torch.full((m, ld), 0x7F, dtype=torch.uint8)
    t[:, :k] = torch.from_numpy(values_u8)
    return t.cuda()[:, :k].view(torch.float8_e4m3fn)


SHAPES = [(1, 1, 1), (1, 16, 16), (1, 17, 31), (1, 768, 3200), (2, 129, 100), (3, 264, 768), (5, 127, 129),
          (7, 128, 128), (8, 400, 255), (9, 33, 700), (16, 384, 768), (17, 65, 1000), (31, 130, 260), (33, 264, 96),
          (64, 928, 768), (100, 203, 17), (127, 300, 385), (128, 256, 512), (129, 257, 640), (256, 1024, 256),
          (300, 100, 4100), (515, 1290, 384), (1200, 400, 900), (2000, 2100, 300), (4100, 130, 200)]


@pytest.mark.parametrize('m,n,k', SHAPES)
def test_matmul_integers_exact(m, n, k):
    """Small integers under power-of-two scales: every sum is exact in fp32, so the product must be."""
    rng = np.random.default_rng(m + 7 * n + 13 * k)
    a, w = rng.integers(-3, 4, (m, k)).astype(np.float64), rng.integers(-3, 4, (n, k)).astype(np.float64)
    kb = -(-k // BLOCK)
    sa = 2.0 ** rng.integers(-2, 3, (m, kb))
    sw = 2.0 ** rng.integers(-2, 3, (-(-n // BLOCK), kb))
    want = np.zeros((m, n))
    for j in range(kb):
        at = slice(j * BLOCK, (j + 1) * BLOCK)
        want += (a[:, at] * sa[:, j:j + 1]) @ (w[:, at] * sw.repeat(BLOCK, 0)[:n, j:j + 1]).T
    got = blockscale.matmul(held(nearest_e4m3(a), 16), torch.from_numpy(sa).float().cuda(), held(nearest_e4m3(w)),
                            torch.from_numpy(sw).float().cuda())
    assert np.array_equal(got.cpu().double().numpy(), want)


def product_64(a, sa, w, sw):
    """(sum, sum of magnitudes) of a block-scaled product, on the GPU in 64 bits."""
    m, k = a.shape
    n = w.shape[0]
    x = a.double() * sa.double().repeat_interleave(BLOCK, 1)[:, :k]
    z = w.double() * sw.double().repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    return x @ z.T, x.abs() @ z.abs().T


@pytest.mark.parametrize('out', list(TYPES))
@pytest.mark.parametrize('m,n,k', SHAPES)
def test_matmul_against_64_bits(m, n, k, out):
    gen = torch.Generator(device='cuda').manual_seed(m * n + k)
    x = torch.randn((m, k), generator=gen, device='cuda') * torch.randn((1, k), generator=gen, device='cuda').exp()
    w = torch.randn((n, k), generator=gen, device='cuda') * k ** -0.5
    a, sa = blockscale.quantize(x)
    b, sb = blockscale.quantize(w, 128)
    bias = torch.randn(n, generator=gen, device='cuda')
    add = torch.randn((m, n + 3), generator=gen, device='cuda')[:, 1:1 + n]
    want, size = product_64(a, sa, b, sb)
    kb = -(-k // BLOCK)
    half_step = torch.finfo(TYPES[out]).eps / 2
    for extra in (False, True):
        if extra:
            got = blockscale.matmul(a, sa, b, sb, bias, add, 0.25, TYPES[out])
            want = want + bias.double() + 0.25 * add.double()
            size = size + bias.double().abs() + 0.25 * add.double().abs()
        else:
            got = blockscale.matmul(a, sa, b, sb, out_dtype=TYPES[out])
        assert got.dtype == TYPES[out] and got.shape == (m, n)
        bound = (128 + kb + 4) * 2.0 ** -23 * size + half_step * want.abs()
        if out == 'fp16':
            bound = bound + 2.0 ** -25   # half a step of its subnormals
        assert ((got.double() - want).abs() <= bound).all()


def test_linear_is_quantize_then_matmul_and_repeats():
    gen = torch.Generator(device='cuda').manual_seed(3)
    for m in (1, 40, 700):
        x = torch.randn((m, 1500), generator=gen, device='cuda', dtype=torch.bfloat16)
        w, sw = blockscale.quantize(torch.randn((900, 1500), generator=gen, device='cuda'), 128)
        y = blockscale.linear(x, w, sw, out_dtype=torch.bfloat16)
        q, s = blockscale.quantize(x)
        for _ in range(3):
            assert torch.equal(y, blockscale.matmul(q, s, w, sw, out_dtype=torch.bfloat16))


def test_empty_batch():
    w, sw = blockscale.quantize(torch.randn(20, 40).cuda(), 128)
    q, s = blockscale.quantize(torch.zeros(0, 40).cuda())
    assert q.shape == (0, 40) and s.shape == (0, 1)
    assert blockscale.matmul(q, s, w, sw).shape == (0, 20)


def test_result_may_overwrite_the_memory_term():
    """y = add at the C boundary: an in-place update."""
    from neurogen_b200 import library
    from neurogen_b200._lib import check
    gen = torch.Generator(device='cuda').manual_seed(8)
    for m, n, k in ((1, 300, 500), (200, 300, 1500)):
        a, sa = blockscale.quantize(torch.randn((m, k), generator=gen, device='cuda'))
        w, sw = blockscale.quantize(torch.randn((n, k), generator=gen, device='cuda'), 128)
        add = torch.randn((m, n), generator=gen, device='cuda')
        want = blockscale.matmul(a, sa, w, sw, None, add, 0.5)
        check(library().ng_block_matmul(0, a.data_ptr(), -(-k // 16) * 16, sa.data_ptr(), w.data_ptr(),
                                        -(-k // 16) * 16, sw.data_ptr(), m, n, k, None, add.data_ptr(), n, 0.5,
                                        add.data_ptr(), 0, n, torch.cuda.current_stream().cuda_stream))
        assert torch.equal(add, want)


def test_rows_behind_the_result_stay():
    """A result in a wider and longer array: nothing beside or behind it is written."""
    from neurogen_b200 import library
    from neurogen_b200._lib import check
    gen = torch.Generator(device='cuda').manual_seed(9)
    for m, n, k in ((1, 77, 300), (3, 130, 129), (70, 129, 1000), (300, 500, 260)):
        for code, dtype in ((0, torch.float32), (1, torch.bfloat16), (2, torch.float16)):
            a, sa = blockscale.quantize(torch.randn((m, k), generator=gen, device='cuda'))
            w, sw = blockscale.quantize(torch.randn((n, k), generator=gen, device='cuda'), 128)
            y = torch.full((m + 5, n + 7), 3.5, dtype=dtype, device='cuda')
            check(library().ng_block_matmul(0, a.data_ptr(), -(-k // 16) * 16, sa.data_ptr(), w.data_ptr(),
                                            -(-k // 16) * 16, sw.data_ptr(), m, n, k, None, None, n, 1.0,
                                            y.data_ptr(), code, n + 7, torch.cuda.current_stream().cuda_stream))
            assert torch.equal(y[:m, :n], blockscale.matmul(a, sa, w, sw, out_dtype=dtype))
            assert (y[m:] == 3.5).all() and (y[:, n:] == 3.5).all()


def test_streams_and_graphs():
    """On a side stream, two calls at once, and captured into a graph that is replayed on new inputs."""
    gen = torch.Generator(device='cuda').manual_seed(4)
    x = torch.randn((90, 700), generator=gen, device='cuda')
    w, sw = blockscale.quantize(torch.randn((500, 700), generator=gen, device='cuda'), 128)
    want = blockscale.linear(x, w, sw)
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in sides:
        with torch.cuda.stream(s):
            got.append([blockscale.linear(x, w, sw) for _ in range(20)])
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for ys in got for y in ys)
    graph = torch.cuda.CUDAGraph()
    held_x = x.clone()
    with torch.cuda.graph(graph):
        y = blockscale.linear(held_x, w, sw)
    for scale in (1.0, -2.0):
        held_x.copy_(x * scale)
        graph.replay()
        assert torch.equal(y, blockscale.linear(x * scale, w, sw))


def test_refusals():
    x = torch.zeros(4, 32, device='cuda')
    q, s = blockscale.quantize(x)
    w, sw = blockscale.quantize(x, 128)
    for call, text in [
        (lambda: blockscale.quantize(x.double()), 'float32'), (lambda: blockscale.quantize(x, 64), '1 or 128'),
        (lambda: blockscale.quantize(x.t()), 'adjacent columns'), (lambda: blockscale.quantize(x[:, :0]), 'column'),
        (lambda: blockscale.quantize(x[:1].expand(4, 32)), 'Row stride'),
        (lambda: blockscale.matmul(x, s, w, sw), 'e4m3'), (lambda: blockscale.matmul(q[:, :16], s, w, sw), 'columns'),
        (lambda: blockscale.matmul(q, s, w, sw.double()), 'w_scale'),
        (lambda: blockscale.matmul(q, s[:2], w, sw), 'a_scale'),
        (lambda: blockscale.matmul(q, s, w, sw, bias=torch.zeros(5, device='cuda')), 'bias'),
        (lambda: blockscale.matmul(q, s, w, sw, add=torch.zeros(3, 4, device='cuda')), 'add'),
        (lambda: blockscale.matmul(q, s, w, sw, out_dtype=torch.float64), 'out_dtype'),
        (lambda: blockscale.matmul(torch.zeros(4, 31, dtype=torch.uint8, device='cuda').view(q.dtype),
                                   s, torch.zeros(4, 31, dtype=torch.uint8, device='cuda').view(q.dtype), sw),
         '16-byte'),
        (lambda: blockscale.matmul(q, s, w.cpu(), sw), 'CUDA device'),
    ]:
        with pytest.raises(ValueError, match=text):
            call()
