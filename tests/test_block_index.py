"""Index arithmetic of the 8-bit operators on matrices of many blocks: on the CPU for every block a
launch forms, and on the GPU one case just above 2^24 blocks with a ragged last CTA."""
import shutil
import subprocess

import pytest
import torch

from conftest import ROOT

CSRC = ROOT / 'neurogen-2.5_b200' / 'csrc'


@pytest.mark.skipif(shutil.which('g++') is None, reason='no C++ compiler')
def test_blocks_past_the_last_one_read_nothing(tmp_path):
    exe = tmp_path / 'block_index'
    cmd = ['g++', '-std=c++17', '-O2', '-Wall', '-Werror', '-fsanitize=undefined', '-fno-sanitize-recover', f'-I{CSRC}',
           '-I/usr/local/cuda/include', str(ROOT / 'tests' / 'native' / 'block_index.cpp'), '-o', str(exe)]
    out = subprocess.run(cmd, capture_output=True, text=True)
    assert out.returncode == 0, out.stderr[-3000:]
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr[-2000:]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype,m,k', [(torch.bfloat16, (1 << 24) + 1, 16), (torch.float32, (1 << 24) + 35, 3)])
def test_quantize_more_than_2_24_blocks(dtype, m, k):
    """One block a row.  The definition in 64 bits (a 64-bit quotient of two fp32 numbers, rounded to
    fp32, is the fp32 division) at the ends and in the middle; the rows behind the result stay."""
    from neurogen_b200 import blockscale, library
    from neurogen_b200._lib import check, stream_of
    x = torch.randn((m, k), generator=torch.Generator('cuda').manual_seed(2), device='cuda', dtype=dtype)
    q = torch.full((m + 70, 16), 0x55, dtype=torch.uint8, device='cuda')
    scale = torch.full((m + 70,), 7.0, device='cuda')
    check(library().ng_block_quantize(0, x.data_ptr(), blockscale.ELEMENTS[dtype], m, k, k, 1, q.data_ptr(), 16,
                                      scale.data_ptr(), stream_of(x.device)))
    assert (q[m:] == 0x55).all() and (q[:, k:] == 0x55).all() and (scale[m:] == 7.0).all()
    for rows in (slice(0, 1000), slice(m // 2, m // 2 + 1000), slice(m - 1000, m)):
        part = x[rows].double()
        want = (part.abs().amax(1) / 448.0).float().clamp(min=2.0 ** -126)
        assert torch.equal(scale[rows], want)
        values = (part / want.double()[:, None]).float().to(torch.float8_e4m3fn)
        assert torch.equal(q[rows, :k], values.view(torch.uint8))
