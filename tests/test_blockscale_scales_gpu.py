"""The 8-bit product under scales whose own product leaves fp32's range though the result does not.

A block's sum d is an integer multiple of 2^-18 below 2^25, so s d with s = a_scale * w_scale can be an
ordinary number (or zero) where s overflows or is subnormal.  The definition multiplies each
operand by its scale, so such a result is as good as any other.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from neurogen_b200 import blockscale  # noqa: E402
from test_blockscale_gpu import BLOCK, held, nearest_e4m3, product_64  # noqa: E402

# Sizes of every launch: a few rows (8, 16, 32 a CTA, one and several CTAs an SM), tiles of 32, 64, 128
# and 256 columns, and a k range shared by 2, 4 and 8 CTAs.
SIZES = [(1, 101, 141), (1, 2463, 140), (10, 1685, 148), (18, 1985, 140), (19, 2613, 140), (35, 2810, 150),
         (35, 1723, 2420), (120, 996, 1257), (304, 124, 4364), (150, 2636, 141), (10, 4168, 4716), (35, 1374, 3293),
         (36, 816, 5984), (277, 3297, 145), (563, 4070, 141)]


@pytest.mark.parametrize('m,n,k', SIZES)
def test_powers_of_two_across_the_range(m, n, k):
    """Small integers under powers of two from 2^-140 to 2^127: results that fp32 holds are exact, zeros
    included; below its subnormals' step each of the kb additions rounds once, by half of 2^-149; where a
    block's term overflows the result is not finite."""
    rng = np.random.default_rng(m + 3 * n + 5 * k)
    a, w = rng.integers(-3, 4, (m, k)).astype(np.float64), rng.integers(-3, 4, (n, k)).astype(np.float64)
    w[rng.random(n) < 0.2] = 0   # block sums of exactly zero
    kb, nb = -(-k // BLOCK), -(-n // BLOCK)
    rows = np.array([-100, 0, 127, -140, 60, -126, 100, -60, -30, 90])
    cols = np.array([60, -126, 0, -60, 127, -40, -140, 30])
    e, f = np.resize(np.roll(rows, -(n % 10)), m), np.resize(np.roll(cols, -(k % 8)), nb)
    sa, sw = np.broadcast_to(2.0 ** e[:, None], (m, kb)), np.broadcast_to(2.0 ** f[:, None], (nb, kb))
    power = e[:, None] + np.repeat(f, BLOCK)[None, :n]
    whole, most = np.zeros((m, n)), np.zeros((m, n))
    for j in range(kb):
        at = slice(j * BLOCK, (j + 1) * BLOCK)
        part = a[:, at] @ w[:, at].T
        whole += part
        most = np.maximum(np.maximum(most, np.abs(part)), np.abs(whole))
    got = blockscale.matmul(held(nearest_e4m3(a)), torch.from_numpy(sa.astype(np.float32)).cuda(), held(nearest_e4m3(w)),
                            torch.from_numpy(sw.astype(np.float32)).cuda()).cpu().double().numpy()
    fits = np.ldexp(most, power) < 2.0 ** 127
    exact = fits & (power >= -149)
    assert exact.any()
    np.testing.assert_array_equal(got[exact], np.ldexp(whole, power)[exact])
    small = fits & ~exact
    assert (np.abs(got - np.ldexp(whole, power))[small] <= kb * 2.0 ** -150).all()
    over = np.ldexp(most, power) >= 2.0 ** 128
    assert not np.isfinite(got[over & (kb == 1)]).any()


@pytest.mark.parametrize('m,n,k', SIZES)
@pytest.mark.parametrize('ea,ew,small', [(-70, -70, False), (-126, -10, False), (111, -135, False), (60, 68, True),
                                         (116, 12, True)])
def test_scale_products_out_of_range_against_64_bits(m, n, k, ea, ew, small):
    """Any scales around 2^ea and 2^ew, whose products are subnormal or overflow, with block sums that
    bring the results back into range (`small`: bytes of 2^-9 and a few times that).  The bound is
    tests/test_blockscale_gpu.py's, and half a step of the subnormals for each addition."""
    gen = torch.Generator('cuda').manual_seed(m + n + k)
    kb, nb = -(-k // BLOCK), -(-n // BLOCK)

    def operand(rows):
        bits = torch.randint(0, 256, (rows, k), generator=gen, device='cuda', dtype=torch.int32)
        bits = bits % 4 + (bits // 128) * 128 if small else bits - (bits % 128 == 127).int()
        buffer = torch.zeros((rows, -(-k // 16) * 16), dtype=torch.uint8, device='cuda')
        buffer[:, :k] = bits.to(torch.uint8)
        return buffer[:, :k].view(torch.float8_e4m3fn)

    a, w = operand(m), operand(n)
    sa = torch.ldexp(1 + torch.rand((m, kb), generator=gen, device='cuda').double(), torch.tensor(ea, device='cuda'))
    sw = torch.ldexp(1 + torch.rand((nb, kb), generator=gen, device='cuda').double(), torch.tensor(ew, device='cuda'))
    sa, sw = sa.float(), sw.float()
    want, size = product_64(a, sa, w, sw)
    got = blockscale.matmul(a, sa, w, sw).double()
    assert size.max() < 2.0 ** 127 and size.max() > 2.0 ** -126
    assert ((got - want).abs() <= (128 + kb + 4) * 2.0 ** -23 * size + (kb + 3) * 2.0 ** -150).all()


@pytest.mark.parametrize('m', [1, 300])
def test_scales_that_are_zero_or_not_finite(m):
    """A zero scale makes its block nothing; an infinite or NaN scale makes a NaN of zero values, and an
    infinite one an infinity of others, as multiplying the operands out does."""
    k, n = 256, 200
    a = held(nearest_e4m3(np.ones((m, k))))
    w = held(nearest_e4m3(np.ones((n, k))))
    sa, sw = torch.full((m, 2), 2.0 ** 100, device='cuda'), torch.full((2, 2), 2.0 ** 20, device='cuda')
    sa[:, 0] = 0
    assert (blockscale.matmul(a, sa, w, sw) == 128 * 2.0 ** 120).all()
    sw[0, 0] = 2.0 ** -140
    assert (blockscale.matmul(a, sa, w, sw) == 128 * 2.0 ** 120).all()
    for bad in (float('inf'), float('nan')):
        sa[:, 0], sw[0, 0] = bad, 2.0 ** -140
        y = blockscale.matmul(a, sa, w, sw)
        assert (torch.isnan(y) if bad != bad else y == bad).all()
