"""edgegan_amd.ops and its C entries at the limits of what they take: pitches of single rows, derivatives at exactly zero, the largest and smallest
finite values and temperatures, workspaces of exactly the size asked for.  References, tolerances and their derivation: test_rowops_gpu."""
import ctypes as C
import math

import pytest
import torch

import test_rowops_gpu as R
from test_rowops_gpu import BF16, F16, F32, TYPES, U, half, near, rnd, tiny

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops(built_lib):
    from edgegan_amd import ops as o
    return o


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('norm', [0, 1])
@pytest.mark.parametrize('cols', [5, 37, 100, 1021, 4096, 20005])
def test_quantize_one_row_at_any_pitch(ops, cols, norm, dtype):
    """A single row's distance to the next one says nothing: all of the row is written whatever it is, zeros behind it only as far as it reaches."""
    lib = ops._library()
    x = rnd(1, cols, seed=cols, dtype=dtype, scale=2.0).cuda()
    want, want_s = ops.quantize_rows(x, norm=(None, None, 1e-5) if norm else None)
    whole = (cols + 15) // 16 * 16
    for ldq in sorted({0, 1, cols - 1, cols, cols + 3, whole, whole + 16}):
        q, s = torch.full((whole + 64,), 77, dtype=torch.int8, device='cuda'), torch.zeros(1, device='cuda')
        assert lib.eg_quantize_rows(0, stream(), R_TYPES[dtype], x.data_ptr(), 0, norm, None, None, 1e-5, 1, cols, q.data_ptr(), ldq, s.data_ptr()) == 0
        end = max(cols, min(whole, ldq))
        assert torch.equal(q[:cols], want[0]) and torch.equal(s, want_s), ldq
        assert (q[cols:end] == 0).all() and (q[end:] == 77).all(), ldq


R_TYPES = {F32: 0, BF16: 1, F16: 2}


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('act', ['relu', 'lrelu'])
@pytest.mark.parametrize('rows,cols', [(4, 3), (4, 24), (300, 100), (5, 1000), (40, 1001), (3, 5001), (3, 9000), (3, 20003)])
def test_gradient_of_activations_at_zero(ops, rows, cols, act, dtype):
    """Rows of one value (padding, mostly) have xh = 0, so with no shift or one of zeros every pre-activation is exactly 0: the derivative there is LeakyReLU's slope
    (ReLU: 0), in every kernel, as in torch."""
    x, dy = rnd(rows, cols, seed=1, dtype=dtype), rnd(rows, cols, seed=2, dtype=dtype)
    x[0], x[1::3], x[2] = 0, 3.5, -0.25
    w = rnd(cols, seed=3, dtype=dtype, scale=0.2, shift=1.0)
    zero = torch.zeros(cols, dtype=dtype)
    for weight, bias in ((w, None), (w, zero), (None, zero), (zero, zero), (None, None)):
        y, dx, dw, db = R.check_norm(ops, x, dy, weight, bias, 1e-5, act)
        assert (y[:3] == 0).all()
    if act == 'relu':
        assert (dx[:3] == 0).all()
