"""8-bit block-scaled matrices on the GPU (include/neurogen_b200.h part 5).

A matrix is e4m3 bytes with one fp32 scale for each block of 128 columns and one row
(activations) or 128 rows (weights).  ``matmul`` multiplies two of them on the tensor cores; the
engine's opt-in 8-bit projections (``NEUROGEN_PROJECTION=fp8``) are these operators.  They take
CUDA tensors, run on the current stream of the tensors' device and do not synchronise; of a call's
data nothing is kept.  Inference only: no gradients flow through them.
"""
import torch

from ._lib import library, F32_CODE, check, stream_of

BLOCK = 128
ELEMENTS = {torch.float32: F32_CODE, torch.bfloat16: 1, torch.float16: 2}
E4M3 = torch.float8_e4m3fn


# The wrappers are on the path of calls that take a few microseconds on the device: each check is one
# attribute, and results are made by empty_strided, the cheapest of torch's constructors.

def _matrix(x, what):
    if not isinstance(x, torch.Tensor) or x.dim() != 2:
        raise ValueError(f'{what} must be a tensor [rows, columns]')
    if not x.is_cuda:
        raise ValueError(f'{what} must be on a CUDA device; there is no CPU fallback')
    shape = x.shape
    if x.stride(1) != 1 and shape[1] > 1:
        raise ValueError(f'{what} must have adjacent columns')
    return shape


def _row_stride(x, rows, cols):
    """Elements from a row to the next; a single row has no next."""
    return x.stride(0) if rows > 1 else cols


def _vector(x, shape, dtype, device, what):
    if (not isinstance(x, torch.Tensor) or x.dtype is not dtype or x.shape != shape or x.device != device
            or not x.is_contiguous()):
        raise ValueError(f'{what} must be contiguous {dtype} {list(shape)} on {device}')


def quantize(x, rows=1):
    """``x`` [m, k] (float32, bfloat16 or float16) as (e4m3 [m, k], scale): a scale for each 1 x 128
    block (``rows=1``) or 128 x 128 block (``rows=128``).

    scale = max(amax / 448, 2^-126) and byte = e4m3(x / scale), rounded to nearest even.  The bytes'
    rows start on 16-byte boundaries (their row stride is k rounded up to 16).
    """
    m, k = _matrix(x, 'x')
    code = ELEMENTS.get(x.dtype)
    if code is None:
        raise ValueError('x must be float32, bfloat16 or float16')
    if rows != 1 and rows != BLOCK:
        raise ValueError('A scale covers 1 or 128 rows')
    if k < 1:
        raise ValueError('x must have at least one column')
    device = x.device
    ldq, kb = -(-k // 16) * 16, -(-k // BLOCK)
    q = torch.empty_strided((m, k), (ldq, 1), dtype=E4M3, device=device)
    scale = torch.empty_strided((-(-m // rows), kb), (kb, 1), dtype=torch.float32, device=device)
    check(library().ng_block_quantize(device.index, x.data_ptr(), code, m, k, _row_stride(x, m, k), rows,
                                      q.data_ptr(), ldq, scale.data_ptr(), stream_of(device)))
    return q, scale


def matmul(a, a_scale, w, w_scale, bias=None, add=None, add_scale=1.0, out_dtype=torch.float32):
    """``a @ w.T`` (+ ``bias``) (+ ``add_scale * add``) of two block-scaled matrices.

    ``a`` e4m3 [m, k] with scales for 1 x 128 blocks, ``w`` e4m3 [n, k] with scales for 128 x 128
    blocks (``quantize(w, 128)``); rows on 16-byte boundaries.  ``bias`` float32 [n], ``add``
    float32 [m, n].  fp32 sums, rounded once to ``out_dtype`` (float32, bfloat16 or float16).
    """
    m, k = _matrix(a, 'a')
    n, kw = _matrix(w, 'w')
    if a.dtype is not E4M3 or w.dtype is not E4M3:
        raise ValueError('a and w must be float8_e4m3fn')
    if kw != k:
        raise ValueError(f'a has {k} columns and w {kw}')
    if k < 1 or n < 1:
        raise ValueError('w must not be empty')
    code = ELEMENTS.get(out_dtype)
    if code is None:
        raise ValueError('out_dtype must be float32, bfloat16 or float16')
    device = a.device
    if w.device != device:
        raise ValueError('a and w must be on the same device')
    k16, kb = -(-k // 16) * 16, -(-k // BLOCK)
    _vector(a_scale, (m, kb), torch.float32, device, 'a_scale')
    _vector(w_scale, (-(-n // BLOCK), kb), torch.float32, device, 'w_scale')
    if bias is not None:
        _vector(bias, (n,), torch.float32, device, 'bias')
    if add is not None and (_matrix(add, 'add') != (m, n) or add.dtype is not torch.float32 or add.device != device):
        raise ValueError(f'add must be float32 [{m}, {n}] on {device}')
    y = torch.empty_strided((m, n), (n, 1), dtype=out_dtype, device=device)
    check(library().ng_block_matmul(device.index, a.data_ptr(), _row_stride(a, m, k16), a_scale.data_ptr(), w.data_ptr(),
                                    _row_stride(w, n, k16), w_scale.data_ptr(), m, n, k,
                                    None if bias is None else bias.data_ptr(),
                                    None if add is None else add.data_ptr(),
                                    n if add is None else _row_stride(add, m, n), add_scale, y.data_ptr(),
                                    code, n, stream_of(device)))
    return y


def check_products(device=None):
    """Raise ValueError when a product on ``device`` (default: the current one) has given up a wait since
    the last call that reported one; synchronise before.  ``matmul`` asks the same before it starts:
    this is for callers that replay a graph or have no further product to make.
    """
    index = None if device is None else torch.device(device).index
    check(library().ng_block_check(torch.cuda.current_device() if index is None else index))


def linear(x, w, w_scale, bias=None, add=None, add_scale=1.0, out_dtype=torch.float32):
    """``quantize(x)`` times the block-scaled weights ``w``: a projection in 8 bits."""
    return matmul(*quantize(x), w, w_scale, bias, add, add_scale, out_dtype)
