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


def check_statistics(ops, x, w, b, eps=1e-5, act=None):
    """y and the statistics against 64 bits.  A rstd below the normal numbers is a multiple of 2^-149: off by half of one, which y sees relative to rstd."""
    y, mean, rstd = ops.layer_norm(x.cuda(), w.cuda(), b.cuda(), eps=eps, act=act, statistics=True)
    m64, r64, xh, z = R.norm64(x, w, b, eps)
    low = 2.0 ** -150 / r64
    ex = R.xhat_error(x, m64, r64) + xh.abs() * low[:, None]
    near(mean.cpu(), m64, 2 * U * m64.abs() + ex.amax(1) / r64, 'mean')
    near(rstd.cpu(), r64, r64 * (R.chain(x.shape[1]) + 8 * U + 2 * ex.amax(1) ** 2 + low), 'rstd')
    want = torch.where(z > 0, z, R.ACT_SLOPE[act] * z)
    ez = ex * w.double().abs() + 3 * U * (z.abs() + b.double().abs() + (xh * w.double()).abs())
    near(y.cpu(), want, ez * (1 + half(x.dtype)) + half(x.dtype) * want.abs() + tiny(x.dtype), 'y')
    return z, ez


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('cols', [2, 3, 17, 40, 128, 1000, 1024, 3001, 5000, 9000, 17000, 40001])
def test_layer_norm_of_large_values(ops, cols, dtype):
    """Rows of the type's lowest and highest value, masked in parts by the lowest one, and of numbers whose squares 32 bits do not hold: the
    statistics are those of the definition, alone and in front of the quantisation."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    big = [1.0, 1e15, 1e19, 3e19, 1e25, 1e37] if dtype != F16 else [1.0, 1e3, 1e4]
    rows = [torch.full((cols,), low), torch.full((cols,), high)]
    for i, s in enumerate(big):
        rows.append((rnd(cols, seed=i).clamp(-4, 4) * s))
    masked = rnd(cols, seed=20)
    masked[cols // 2:] = low
    rows.append(masked)
    masked = rnd(cols, seed=21)
    masked[-1] = low
    rows.append(masked)
    rows.append(rnd(cols, seed=22))          # an ordinary row between them
    x = torch.stack(rows).to(dtype)
    w, b = rnd(cols, seed=30, scale=0.2, shift=1.0), rnd(cols, seed=31, scale=0.2)
    z, ez = check_statistics(ops, x, w, b, act='lrelu')
    z, ez = check_statistics(ops, x, w, b)
    how = (w.cuda(), b.cuda(), 1e-5)
    q, s = ops.quantize_rows(x.cuda(), norm=how)
    amax = z.abs().amax(1)
    near(s.cpu(), amax / 127, ez.amax(1) / 127 + U * amax / 127, 'scale')
    off = (q.cpu().double() - 127 * z / amax[:, None]).abs()
    assert (off <= 0.5 + 127 * (ez + ez.amax(1, keepdim=True)) / amax[:, None] + 1e-9).all()
    # few rows and short ones in one launch are the two calls
    qw, sw = ops.quantize_rows(rnd(33, cols, seed=32).cuda())
    for part in (x[:1], x[2:6], x, x[[-1, 0]], x[[0, -1]], x[[-1, -1, 0, -1]], x[[0, -1, -1, -1]], x[[-1, 6, 1]]):
        got = ops.int8_linear(part.cuda(), qw, sw, norm=how)
        assert torch.equal(got, ops.int8_matmul(*ops.quantize_rows(part.cuda(), norm=how), qw, sw, out_dtype=dtype))
    # a row's neighbours do not matter
    y = ops.layer_norm(x.cuda(), w.cuda(), b.cuda())
    for r in range(len(rows)):
        assert torch.equal(ops.layer_norm(x[r:r + 1].cuda(), w.cuda(), b.cuda())[0], y[r]), r
    # many of them in the hands of each team, in place
    many, wd, bd = x.repeat(900, 1).cuda(), w.cuda(), b.cuda()
    assert ops._library().eg_layer_norm(0, stream(), R_TYPES[dtype], many.data_ptr(), cols, 0, wd.data_ptr(), bd.data_ptr(), len(many), cols, 1e-5, 0, many.data_ptr(), cols, None,
                                        None) == 0
    assert torch.equal(many, y.repeat(900, 1))


@pytest.mark.parametrize('dtype', [F32, BF16], ids=str)
@pytest.mark.parametrize('rows,cols', [(6, 40), (300, 100), (5, 1001), (3, 9000), (3, 20003)])
def test_gradient_of_large_values(ops, rows, cols, dtype):
    """The gradient at rows of size 10^25 (rstd is a normal number and dx of size 10^-25)."""
    x = (rnd(rows, cols, seed=1, scale=1e25)).to(dtype)
    R.check_norm(ops, x, rnd(rows, cols, seed=2, dtype=dtype), rnd(cols, seed=3, shift=1.0, scale=0.2), rnd(cols, seed=4, scale=0.2), 1e-5, 'lrelu')


@pytest.mark.parametrize('cols', [*range(1, 40), 127, 250, 1001, 1002, 1003, 1023, 3001, 5001, 5002, 5003, 8191, 16383, 20001])
def test_rows_of_one_value(ops, cols):
    """xh is exactly 0, whatever the value and the length: y is the shift."""
    for dtype in TYPES:
        x = torch.tensor([0.1, 1000.1, -3.3e-7, 65503.0, 1 / 3, -0.7, 2.0 ** -14 * 1.1], dtype=dtype)[:, None].expand(7, cols).contiguous()
        b = rnd(cols, seed=1, dtype=dtype).cuda()
        y, mean, _ = ops.layer_norm(x.cuda(), None, b, statistics=True)
        assert torch.equal(mean.cpu(), x[:, 0].float()) and torch.equal(y, b.expand(7, cols)), dtype


@pytest.mark.parametrize('cols', [14, 300, 5000, 40000, 70001])
@pytest.mark.parametrize('t', [1e-25, 1e-12, 1e-3])
def test_distill_at_small_temperatures(ops, t, cols):
    """T^2 may be below every 32-bit number where T^2 KL is not: both distributions are one class, and the loss is T times the student's distance to it."""
    rows = 5
    z = rnd(rows, cols, seed=cols, scale=2.0)
    z[:, 3] = 20.0                                   # the student's choice, ahead by more than 1e-3 of anything
    idx, u = torch.tensor([[0, 1, 2, 3, 4]] * rows), rnd(rows, 5, seed=2)
    u[:, 1] = 9.0                                    # the teacher's
    loss, grad = ops.distill_loss(z.cuda(), idx.cuda(), u.cuda(), temperature=t)
    want = t * (z[:, 3] - z[:, 1]).double()
    near(loss.cpu(), want, 16 * U * want, 'loss')    # (a difference, 1 / T, three products)
    g = torch.zeros(rows, cols, dtype=torch.float64)
    g[:, 3], g[:, 1] = t, -t
    near(grad.cpu(), g, 4 * U * g.abs(), 'grad')


@pytest.mark.parametrize('cols', [14, 300, 5000, 40000, 70001])
@pytest.mark.parametrize('t', [1e12, 1e18, 1e25])
def test_distill_at_large_temperatures(ops, t, cols):
    """Both distributions are even: T^2 log(classes / kept) where f32 holds it, infinity where not, and a gradient of size T."""
    z, idx, u = rnd(3, cols, seed=cols), torch.tensor([[0, 3], [5, 1], [2, 13]]), rnd(3, 2, seed=2)
    loss, grad = ops.distill_loss(z.cuda(), idx.cuda(), u.cuda(), temperature=t)
    want = torch.full((3,), t * t * math.log(cols / 2), dtype=torch.float64)
    if t < 1e19:   # the log-sums of `cols` and two exponentials, each off by a sum and a rounding; three products
        near(loss.cpu(), want, t * t * (R.chain(cols) + 40 * U + 4 * U * math.log(cols)) + 4 * U * want, 'loss')
    else:
        assert (loss == math.inf).all()
    g = torch.full((3, cols), t / cols, dtype=torch.float64)
    g.scatter_add_(1, idx, torch.full((3, 2), -t / 2, dtype=torch.float64))
    near(grad.cpu(), g, t * (R.chain(cols) + 40 * U) * (1 / cols + 0.5 * (g < 0)) + 4 * U * g.abs(), 'grad')


def test_tensors_without_plain_memory_are_refused(ops):
    """Sparse tensors, and tensors whose sign torch applies when they are read."""
    from edgegan_amd import EdgeGANLibError
    x = torch.randn(4, 32, device='cuda')
    column = torch.randn(4, 1, dtype=torch.complex64, device='cuda').conj().imag     # the values of minus its memory
    one = torch.randn(1, dtype=torch.complex64, device='cuda').conj().imag
    assert column.is_neg() and one.is_neg()
    v = torch.ones(32, device='cuda')
    for f in (lambda: ops.layer_norm(x.to_sparse()), lambda: ops.layer_norm(x.to_sparse_csr()), lambda: ops.layer_norm(column), lambda: ops.layer_norm(one),
              lambda: ops.layer_norm(x, v.to_sparse()), lambda: ops.layer_norm(column.clone(), one), lambda: ops.layer_norm(x, eps=10 ** 400),
              lambda: ops.quantize_rows(column), lambda: ops.distill_loss(column, torch.zeros(4, 1, dtype=torch.int64, device='cuda'), torch.zeros(4, 1, device='cuda')),
              lambda: ops.distill_loss(x, torch.zeros(4, 1, dtype=torch.int64, device='cuda'), column)):
        with pytest.raises(EdgeGANLibError):
            f()
    assert ops.layer_norm(column.resolve_neg()).shape == (4, 1)


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,cols', [(129, 32), (33, 100), (700, 100), (5000, 128), (17, 1000), (600, 1000), (1100, 1024), (3, 5001), (700, 4096), (600, 8193), (3, 20003), (300, 16500), (70, 33000)])
def test_gradient_writes_inside_its_workspace(ops, rows, cols, dtype):
    """The workspace of eg_layer_norm_workspace's size is enough for every type, and what lies behind it stays."""
    lib = ops._library()
    x, dy, w = rnd(rows, cols, seed=1, dtype=dtype).cuda(), rnd(rows, cols, seed=2, dtype=dtype).cuda(), rnd(cols, seed=3, dtype=dtype).cuda()
    _, m, r = ops.layer_norm(x, w, w, statistics=True)
    size = lib.eg_layer_norm_workspace(rows, cols)
    assert size > 0
    ws = torch.full((size + (8 << 20),), 77, dtype=torch.uint8, device='cuda')   # (room for twice the blocks and more)
    out = torch.empty(2, cols, dtype=dtype, device='cuda')
    e = R_TYPES[dtype]
    assert lib.eg_layer_norm_backward(0, stream(), e, dy.data_ptr(), cols, x.data_ptr(), cols, m.data_ptr(), r.data_ptr(), e, w.data_ptr(), w.data_ptr(), rows, cols, 0,
                                      None, 0, out[0].data_ptr(), out[1].data_ptr(), ws.data_ptr(), size) == 0
    assert (ws[size:] == 77).all()
    _, dw, db = ops.layer_norm_backward(dy, x, m, r, w, w)
    assert torch.equal(out[0], dw) and torch.equal(out[1], db)
