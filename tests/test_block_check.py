"""Asking for a lost 8-bit product without a GPU: no product has run, so there is none; a device that
cannot exist is refused."""
import pytest

from neurogen_b200 import blockscale, library


def test_check_products():
    assert library().ng_block_check(0) == 0
    for device in (-1, 64):
        assert library().ng_block_check(device) == -1 and 'out of range' in library().ng_error().decode()
    blockscale.check_products('cuda:0')
    with pytest.raises(ValueError, match='out of range'):
        blockscale.check_products('cuda:64')


def test_matmul_kind_refusals():
    lib = library()
    for size in ((0, 4, 4), (4, 0, 4), (4, 4, 0), (1 << 31, 4, 4), (4, 1 << 31, 4), (4, 4, 1 << 31)):
        assert lib.ng_block_matmul_kind(0, *size) == -1 and 'out of range' in lib.ng_error().decode()
    assert lib.ng_block_matmul_kind(64, 4, 4, 4) == -1 and 'device' in lib.ng_error().decode()
