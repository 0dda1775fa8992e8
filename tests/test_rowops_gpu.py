"""edgegan_amd.ops against 64-bit restatements of its formulas.

Tolerances are derived per element: U = 2^-24 is half a step of a 32-bit number of size one (every 32-bit operation rounds by at most that,
relative to its result), `half(t)` the same for the result's type.  A sum of n numbers that a lane adds one after the other (at most n / 32 of
them: a row has at least 32 lanes, or is short) and a tree joins is off by at most (n / 32 + 16) U times the sum of the magnitudes."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):   # a value below the normal range is rounded to a multiple of the smallest number
    return torch.finfo(t).tiny * torch.finfo(t).eps


def chain(n):
    return (n / 32 + 16) * U


def near(got, want, tol, what=''):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    if bad.any():
        i = int(torch.argmax((err / tol.clamp(min=1e-300)).flatten()))
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.numel()} values off; worst got {got.flatten()[i].item()!r}, want '
                             f'{want.flatten()[i].item()!r}, tolerance {tol.expand(want.shape).flatten()[i].item():.3e}')


@pytest.fixture(scope='module')
def ops(built_lib):
    from edgegan_amd import ops as o
    return o


def rnd(*shape, seed=0, dtype=F32, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype)


def affine32(x, mean, rstd, w, b):
    """The pre-activation by the kernels' own three 32-bit operations: its sign is the activation's."""
    z = (x.float() - mean[:, None]) * rstd[:, None]
    if w is not None:
        z = z * w.float()
    return z if b is None else z + b.float()


def norm64(x, w, b, eps):
    x = x.double()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = (d.square().mean(1) + eps).rsqrt()
    xh = d * rstd[:, None]
    z = xh * (1 if w is None else w.double()) + (0 if b is None else b.double())
    return mean, rstd, xh, z


def xhat_error(x, mean, rstd):
    """Bound on the error of (x - mean) rstd: the mean off by its rounding and that of its sum, the difference rounded, rstd off by a sum."""
    n = x.shape[1]
    spread = 1 / rstd
    e_mean = 2 * U * mean.abs() + chain(n) ** 2 * x.double().abs().mean(1) + chain(n) * U * n + 4 * U * spread
    d = (x.double() - mean[:, None]).abs()
    return ((U * d + e_mean[:, None]) + d * (chain(n) + 4 * U + 2 * (e_mean * rstd)[:, None])) * rstd[:, None]


ACT_SLOPE = {None: 1.0, 'relu': 0.0, 'lrelu': 0.2}
SIZES = [(1, 1), (3, 2), (5, 7), (2, 8), (33, 16), (9, 31), (130, 64), (7, 100), (67, 128), (3, 129), (5, 255), (21, 256), (2, 513), (4, 1000),
         (37, 1024), (3, 2048), (6, 4096), (3, 5001), (2, 8192), (2, 20000), (3, 70001)]


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,cols', SIZES)
def test_layer_norm_and_gradient(ops, rows, cols, dtype):
    act = [None, 'relu', 'lrelu'][(rows + cols) % 3]
    wtype = dtype if (rows + cols) % 2 else F32
    x = rnd(rows, cols, seed=rows * 7 + cols, dtype=dtype, scale=1.5, shift=0.75)
    dy = rnd(rows, cols, seed=rows * 7 + cols + 1, dtype=dtype)
    w, b = rnd(cols, seed=cols, dtype=wtype, scale=0.2, shift=1.0), rnd(cols, seed=cols + 1, dtype=wtype, scale=0.2)
    check_norm(ops, x, dy, w, b, 1e-5, act)


def check_norm(ops, x, dy, w, b, eps, act, x_dev=None, dy_dev=None):
    cu = lambda t: None if t is None else t.cuda()
    xd, dyd = (x.cuda() if x_dev is None else x_dev), (dy.cuda() if dy_dev is None else dy_dev)
    wd, bd = cu(w), cu(b)
    y, mean, rstd = ops.layer_norm(xd, wd, bd, eps=eps, act=act, statistics=True)
    assert torch.equal(ops.layer_norm(xd, wd, bd, eps=eps, act=act), y), 'with and without statistics'
    assert y.dtype == x.dtype and mean.dtype == F32
    slope, cols, rows = ACT_SLOPE[act], x.shape[1], x.shape[0]
    m64, r64, xh, z = norm64(x, w, b, eps)
    ex = xhat_error(x, m64, r64)
    aw = torch.ones(cols, dtype=torch.float64) if w is None else w.double().abs()
    ab = torch.zeros(cols, dtype=torch.float64) if b is None else b.double().abs()
    near(mean.cpu(), m64, 2 * U * m64.abs() + ex.amax(1) / r64, 'mean')
    # rstd: relative error half of the variance's, plus the root's and the division's
    near(rstd.cpu(), r64, r64 * (chain(cols) + 8 * U + 2 * ((ex.amax(1)) ** 2)), 'rstd')
    want = torch.where(z > 0, z, slope * z)
    ez = ex * aw + 3 * U * (z.abs() + ab + (xh.abs() * aw))
    near(y.cpu(), want, ez * (1 + half(x.dtype)) + half(x.dtype) * want.abs() + tiny(x.dtype), 'y')

    dx, dw, db = ops.layer_norm_backward(dyd, xd, mean, rstd, wd, bd, act=act)
    m, r = mean.cpu(), rstd.cpu()                     # the gradient's inputs are the statistics as stored
    xh = (x.double() - m.double()[:, None]) * r.double()[:, None]
    exh = 3 * U * xh.abs()
    passed = affine32(x, m, r, w, b) > 0 if act else torch.ones_like(xh, dtype=torch.bool)
    g = dy.double() * torch.where(passed, 1.0, slope)
    gw = g * (1 if w is None else w.double())
    a, c = gw.mean(1, keepdim=True), (gw * xh).mean(1, keepdim=True)
    want = (gw - a - xh * c) * r.double()[:, None]
    mag_a, mag_c = gw.abs().mean(1, keepdim=True), (gw * xh).abs().mean(1, keepdim=True)
    e = 4 * U * gw.abs() + (chain(cols) + 4 * U) * mag_a + xh.abs() * (chain(cols) + 8 * U) * mag_c + exh * c.abs() + 3 * U * (gw.abs() + a.abs() + (xh * c).abs())
    near(dx.cpu(), want, e * r.double()[:, None] * (1 + half(x.dtype)) + half(x.dtype) * want.abs() + tiny(x.dtype), 'dx')
    if w is not None:
        assert dw.dtype == w.dtype
        want = (g * xh).sum(0)
        near(dw.cpu(), want, (chain(rows) + 8 * U) * (g * xh).abs().sum(0) + half(w.dtype) * want.abs() + tiny(w.dtype), 'dweight')
    if b is not None:
        assert db.dtype == b.dtype
        want = g.sum(0)
        near(db.cpu(), want, (chain(rows) + 2 * U) * g.abs().sum(0) + half(b.dtype) * want.abs() + tiny(b.dtype), 'dbias')
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    return y, dx, dw, db


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,cols', [(128, 32), (129, 32), (128, 3), (64, 64), (65, 33), (32, 128), (33, 100), (16, 1024), (17, 1000), (13, 701), (1, 8192), (2, 8192), (3, 8192), (2, 5001), (2, 8193), (1, 1)])
def test_layer_norm_gradient_of_few_rows(ops, rows, cols, dtype):
    """On both sides of the rule by which one block does it all; the parameters' gradients one by one are the same, and the rows' sum is the sum of single rows'."""
    x, dy, w, b = (rnd(*shape, seed=i + rows, dtype=dtype).cuda() for i, shape in enumerate([(rows, cols), (rows, cols), (cols,), (cols,)]))
    _, m, r = ops.layer_norm(x, w, b, act='lrelu', statistics=True)
    dx, dw, db = ops.layer_norm_backward(dy, x, m, r, w, b, act='lrelu')
    assert torch.equal(ops.layer_norm_backward(dy, x, m, r, w, None)[1], ops.layer_norm_backward(dy, x, m, r, w, torch.zeros_like(b))[1])
    xh = (x.double() - m.double()[:, None]) * r.double()[:, None]
    z = xh * w.double() + b.double()
    g = dy.double() * torch.where(z > 0, 1.0, 0.2)
    near_kink = (z.abs() < 1e-4 * (1 + xh.abs())).any(0)      # (32 bits may put such an element on the other side)
    for got, want, terms in ((dw, (g * xh).sum(0), (g * xh).abs().sum(0) + (g.abs() * (1 + xh.abs())).sum(0)), (db, g.sum(0), g.abs().sum(0))):
        tol = (chain(rows) + 8 * U) * terms * (1 + half(dtype)) + half(dtype) * want.abs() + tiny(dtype)
        near(got.cpu()[~near_kink.cpu()], want.cpu()[~near_kink.cpu()], tol.cpu()[~near_kink.cpu()], 'sums')


@pytest.mark.parametrize('weight,bias,act', [(False, False, None), (True, False, 'lrelu'), (False, True, 'relu')])
@pytest.mark.parametrize('rows,cols', [(5, 96), (3, 1030), (2, 9000)])
def test_layer_norm_without_parameters(ops, rows, cols, weight, bias, act):
    x, dy = rnd(rows, cols, seed=1), rnd(rows, cols, seed=2)
    check_norm(ops, x, dy, rnd(cols, seed=3) if weight else None, rnd(cols, seed=4) if bias else None, 1e-3, act)


@pytest.mark.parametrize('rows', [1, 2, 63, 257, 1025, 20011])
@pytest.mark.parametrize('cols', [24, 320])
def test_layer_norm_many_rows(ops, rows, cols):
    check_norm(ops, rnd(rows, cols, seed=5), rnd(rows, cols, seed=6), rnd(cols, seed=7), rnd(cols, seed=8), 1e-5, 'lrelu')


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('cols', [128, 130, 1024, 5000])
def test_layer_norm_strides(ops, cols, dtype):
    """Columns sliced out of wider rows at an odd element, several leading dimensions, results consecutive."""
    wide = rnd(2, 9, cols + 5, seed=9, dtype=dtype)
    wide_dy = rnd(2, 9, cols + 11, seed=10, dtype=dtype)
    x, dy = wide[..., 3:3 + cols], wide_dy[..., 1:1 + cols]
    w, b = rnd(cols, seed=11, dtype=dtype), rnd(cols, seed=12, dtype=dtype)
    xd, dyd = wide.cuda()[..., 3:3 + cols], wide_dy.cuda()[..., 1:1 + cols]
    y, mean, rstd = ops.layer_norm(xd, w.cuda(), b.cuda(), act='lrelu', statistics=True)
    assert y.shape == x.shape and y.is_contiguous() and mean.shape == (2, 9)
    y2, m2, r2 = ops.layer_norm(x.reshape(18, cols).cuda(), w.cuda(), b.cuda(), act='lrelu', statistics=True)
    near(y.reshape(18, cols).cpu(), y2.cpu().double(), 2 * half(dtype) * y2.cpu().double().abs() + 64 * U, 'strided')
    got = ops.layer_norm_backward(dyd, xd, mean, rstd, w.cuda(), b.cuda(), act='lrelu')
    check_norm(ops, x.reshape(18, cols), dy.reshape(18, cols), w, b, 1e-5, 'lrelu')
    want = ops.layer_norm_backward(dy.reshape(18, cols).cuda(), x.reshape(18, cols).cuda(), m2, r2, w.cuda(), b.cuda(), act='lrelu')
    for u, v in zip(got, want):
        v = v.cpu().double()
        near(u.reshape(v.shape).cpu(), v, 3 * half(dtype) * v.abs() + 2e3 * U * v.abs().mean(), 'strided gradient')


def test_layer_norm_edges(ops):
    """Constant rows (variance 0), a large level beside a small spread, the largest finite values' neighbourhood, NaN and infinities."""
    x = torch.zeros(6, 200)
    x[1] = 1000.1
    x[2] = rnd(200, seed=13) * 1e-3 + 4096
    x[3] = rnd(200, seed=14) * 1e15
    x[4] = rnd(200, seed=15)
    x[4, 17] = float('nan')
    x[5] = rnd(200, seed=16)
    x[5, 3] = float('inf')
    y, mean, rstd = ops.layer_norm(x.cuda(), eps=1e-5, statistics=True)
    y, mean, rstd = y.cpu(), mean.cpu(), rstd.cpu()
    assert (y[0] == 0).all() and (mean[0] == 0) and abs(rstd[0] * math.sqrt(1e-5) - 1) < 1e-6
    # a constant row: the mean is off by at most half a step of 1000.1 (2^-15), times 1 / sqrt(eps)
    assert (y[1].abs() <= 2.0 ** -15 * 317).all()
    m, r, xh, _ = norm64(x[2:4], None, None, 1e-5)
    near(y[2:4], xh, xhat_error(x[2:4], m, r) + 4 * U * xh.abs(), 'level and spread')
    assert torch.isnan(y[4]).all() and torch.isnan(rstd[4]) and torch.isnan(y[5]).all()
    # other rows are not touched by a NaN row; relu keeps a NaN
    assert torch.isnan(ops.layer_norm(x.cuda(), act='relu').cpu()[4]).all()


def test_layer_norm_no_rows(ops):
    x = torch.empty(0, 40, device='cuda')
    w = torch.ones(40, device='cuda')
    y, mean, rstd = ops.layer_norm(x, w, w, statistics=True)
    dx, dw, db = ops.layer_norm_backward(x, x, mean, rstd, w, w)
    assert y.shape == (0, 40) and dx.shape == (0, 40) and (dw == 0).all() and (db == 0).all()


def test_layer_norm_gradient_by_differences(ops):
    """Directional differences of sum(y v) in 64-bit arithmetic on the inputs, at a smooth point (no activation)."""
    rows, cols = 6, 50
    x, w, b, v = rnd(rows, cols, seed=20), rnd(cols, seed=21), rnd(cols, seed=22), rnd(rows, cols, seed=23)
    f = lambda x, w, b: float((norm64(x, w, b, 1e-5)[3] * v.double()).sum())
    _, mean, rstd = ops.layer_norm(x.cuda(), w.cuda(), b.cuda(), statistics=True)
    grads = ops.layer_norm_backward(v.cuda(), x.cuda(), mean, rstd, w.cuda(), b.cuda())
    for i, (p, g) in enumerate(zip((x, w, b), grads)):
        d = rnd(*p.shape, seed=30 + i).double()
        h = 1e-5
        args = [x.double(), w.double(), b.double()]
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + h * d, args[i] - h * d
        slope = (f(*up) - f(*down)) / (2 * h)
        got = float((g.cpu().double() * d).sum())
        # the differences' own error is O(h^2) ~ 1e-9 of the third derivative; the gradient's about 1e-6 of its terms
        assert abs(slope - got) <= 2e-5 * float((g.cpu().double() * d).abs().sum()), (i, slope, got)


# ---- 8 bits ----------------------------------------------------------------------------------------------------------------------

def quantize64(x):
    amax = x.double().abs().amax(1)
    q = torch.round(127 * x.double() / torch.where(amax > 0, amax, torch.ones_like(amax))[:, None])
    return q.to(torch.int8), (amax / 127).float()


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,cols', SIZES)
def test_quantize_rows(ops, rows, cols, dtype):
    x = rnd(rows, cols, seed=cols, dtype=dtype, scale=3.0)
    x[0, 0] = x[0].abs().max()
    if cols > 1:
        x[0, 1] = -x[0, 0] / 2        # exactly between -63 and -64
    q, s = ops.quantize_rows(x.cuda())
    q64, s64 = quantize64(x)
    assert torch.equal(q.cpu(), q64) and torch.equal(s.cpu(), s64)
    assert q.stride(0) % 16 == 0 or rows == 1
    whole = torch.as_strided(q, (rows, (cols + 15) // 16 * 16), ((cols + 15) // 16 * 16, 1))
    assert (whole[:, cols:] == 0).all(), 'the gap behind a row is zeros'


def test_quantize_rows_edges(ops):
    x = torch.zeros(7, 37)
    x[1, 5] = 1e-45                                # the smallest number
    x[2] = rnd(37, seed=1) * 1e38
    x[3] = rnd(37, seed=2)
    x[3, 36] = float('nan')
    x[4] = rnd(37, seed=3)
    x[4, 0] = -float('inf')
    x[5] = torch.arange(37) * 1e-40                 # below the normal numbers
    x[6] = -3.0
    q, s = ops.quantize_rows(x.cuda())
    q, s = q.cpu(), s.cpu()
    want, ws = quantize64(x)
    for r in (0, 1, 2, 5, 6):
        assert torch.equal(q[r], want[r]), r
        assert s[r] == ws[r], r
    for r in (3, 4):
        assert torch.isnan(s[r]) and (q[r] == 0).all(), r


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,cols', [(1, 1), (4, 17), (9, 64), (3, 1000), (2, 4096), (2, 30001)])
def test_quantize_rows_behind_norm(ops, rows, cols, dtype):
    x = rnd(rows, cols, seed=cols + 5, dtype=dtype, scale=2.0, shift=1.0)
    w, b = rnd(cols, seed=6, scale=0.3, shift=1.0), rnd(cols, seed=7, scale=0.3)
    q, s = ops.quantize_rows(x.cuda(), norm=(w.cuda(), b.cuda(), 1e-5))
    m, r, xh, z = norm64(x, w, b, 1e-5)
    ez = xhat_error(x, m, r) * w.double().abs() + 3 * U * (z.abs() + b.double().abs() + (xh * w.double()).abs())
    amax = z.abs().amax(1)
    near(s.cpu(), amax / 127, ez.amax(1) / 127 + U * amax / 127, 'scale')
    off = (q.cpu().double() - 127 * z / amax[:, None]).abs()
    assert (off <= 0.5 + 127 * (ez + ez.amax(1, keepdim=True)) / amax[:, None] + 1e-9).all()


def int8_case(ops, m, n, k, out_dtype, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed + 1000 * m + 10 * n + k)
    a = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    sa, sw = torch.rand(m, generator=g) * 0.01 + 1e-3, torch.rand(n, generator=g) * 0.01 + 1e-3
    b = torch.randn(n, generator=g) if bias else None
    return a, w, sa, sw, b


def check_int8(ops, a, w, sa, sw, b, out_dtype, ad=None, wd=None):
    ad, wd = (a.cuda() if ad is None else ad), (w.cuda() if wd is None else wd)
    got = ops.int8_matmul(ad, sa.cuda(), wd, sw.cuda(), None if b is None else b.cuda(), out_dtype)
    total = a.double() @ w.double().t()
    prod = total * sa.double()[:, None] * sw.double()
    want = prod if b is None else prod + b.double()
    # the sum to 32 bits, two products, the bias
    tol = 3.01 * U * prod.abs() + U * want.abs()
    near(got.cpu(), want, tol * (1 + half(out_dtype)) + half(out_dtype) * want.abs() + tiny(out_dtype), f'{tuple(a.shape)} x {tuple(w.shape)}')
    assert got.dtype == out_dtype
    return got


@pytest.mark.parametrize('out_dtype', TYPES, ids=str)
@pytest.mark.parametrize('m,n,k', [(1, 1, 1), (1, 64, 64), (1, 1000, 4096), (2, 17, 33), (3, 40, 15), (5, 250, 16), (16, 128, 128), (17, 129, 257), (23, 70, 2050),
                                   (31, 33, 1000), (33, 64, 127), (64, 64, 64), (100, 300, 96), (128, 128, 144), (129, 257, 1040), (200, 136, 64),
                                   (256, 256, 256), (300, 520, 272), (513, 255, 640), (700, 1030, 384)])
def test_int8_matmul(ops, m, n, k, out_dtype):
    check_int8(ops, *int8_case(ops, m, n, k, out_dtype, bias=(m + n + k) % 2 == 0), out_dtype)


@pytest.mark.parametrize('m,n,k', [(1, 96, 100), (20, 96, 100), (70, 200, 300), (300, 300, 516), (1, 513, 2048), (260, 260, 1024)])
def test_int8_matmul_strides(ops, m, n, k):
    """Rows at odd distances and odd addresses; rows as quantize_rows lays them out; garbage in every gap."""
    a, w, sa, sw, b = int8_case(ops, m, n, k, F32)
    base = check_int8(ops, a, w, sa, sw, b, F32)
    for pad, shift in ((1, 0), (5, 3), (16 - k % 16, 0), (64, 16), (12, 4)):
        def spread(t):
            store = torch.full((t.shape[0], k + pad + shift), 113, dtype=torch.int8)
            store[:, shift:shift + k] = t
            return store.cuda()[:, shift:shift + k]
        for ad, wd in ((spread(a), None), (None, spread(w)), (spread(a), spread(w))):
            got = ops.int8_matmul(a.cuda() if ad is None else ad, sa.cuda(), w.cuda() if wd is None else wd, sw.cuda(), b.cuda())
            assert torch.equal(got, base), (pad, shift)


def test_int8_matmul_extremes(ops):
    """The largest sums: every product 127^2 or -127 * 128, as many terms as are allowed."""
    for m, n, k in ((3, 5, 131071), (130, 70, 20000)):
        a, w = torch.full((m, k), -128, dtype=torch.int8), torch.full((n, k), -128, dtype=torch.int8)
        w[1:] = 127
        check_int8(ops, a, w, torch.ones(m), torch.ones(n), None, F32)
    # a scale of NaN (a row that quantize_rows could not hold) reaches its own row alone; zero scales give the bias
    a, w, sa, sw, b = int8_case(ops, 40, 50, 64, F32)
    sa[3], sa[5] = float('nan'), 0.0
    got = ops.int8_matmul(a.cuda(), sa.cuda(), w.cuda(), sw.cuda(), b.cuda()).cpu()
    assert torch.isnan(got[3]).all() and torch.equal(got[5], b) and torch.isfinite(got[[0, 1, 2, 4, 6]]).all()


@pytest.mark.parametrize('m,n', [(40, 70), (31, 9000), (520, 1030), (1000, 1500), (50, 20000), (2000, 1900), (100, 34000), (4000, 2000), (66000, 70), (4100, 2100)])
@pytest.mark.parametrize('k', [16, 100, 256, 513])
def test_int8_matmul_tile_sizes(ops, m, n, k):
    """One output shape for each of the tile sizes and of the reasons for which it is taken; k that ends in every part of a step."""
    a, w, sa, sw, b = int8_case(ops, m, n, k, BF16, bias=k % 2 == 0, seed=k)
    padded = []
    for t in (a, w):   # rows 16 bytes apart, and no zeros behind them
        store = torch.full((t.shape[0], -(-k // 16) * 16), 113, dtype=torch.int8, device='cuda')
        store[:, :k] = t.cuda()
        padded.append(store[:, :k])
    check_int8(ops, a, w, sa, sw, b, BF16, *padded)


def test_int8_matmul_empty(ops):
    z = lambda *s: torch.zeros(*s, dtype=torch.int8, device='cuda')
    f = lambda n: torch.ones(n, device='cuda')
    assert ops.int8_matmul(z(0, 8), f(0), z(5, 8), f(5)).shape == (0, 5)
    assert ops.int8_matmul(z(4, 8), f(4), z(0, 8), f(0)).shape == (4, 0)
    assert (ops.int8_matmul(z(4, 0), f(4), z(3, 0), f(3), bias=2 * f(3)) == 2).all()


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,inner,cols,norm', [(1, 4096, 512, True), (1, 100, 40, False), (4, 1000, 96, True), (23, 2050, 130, False), (300, 64, 128, False), (500, 520, 300, True),
                                                  (2, 20000, 33, True)])
def test_int8_linear(ops, rows, inner, cols, norm, dtype):
    """The layer as its two calls, bit for bit; leading dimensions kept; near the unquantised layer."""
    x = rnd(rows, inner, seed=inner, dtype=dtype)
    weight = rnd(cols, inner, seed=inner + 1, scale=1 / math.sqrt(inner))
    bias, w, b = rnd(cols, seed=3).cuda(), rnd(inner, seed=4, scale=0.1, shift=1.0).cuda(), rnd(inner, seed=5, scale=0.1).cuda()
    qw, sw = ops.quantize_rows(weight.cuda())
    how = (w, b, 1e-5) if norm else None
    got = ops.int8_linear(x.cuda(), qw, sw, bias, norm=how)
    q, s = ops.quantize_rows(x.cuda(), norm=how)
    assert got.dtype == dtype and torch.equal(got, ops.int8_matmul(q, s, qw, sw, bias, dtype))
    assert torch.equal(ops.int8_linear(x.cuda().view(1, rows, 1, inner), qw, sw, bias, norm=how), got.view(1, rows, 1, cols))
    feats = norm64(x, w.cpu(), b.cpu(), 1e-5)[3] if norm else x.double()
    full = feats @ weight.double().t() + bias.cpu().double()
    # each operand is off by at most half a step of amax / 127, independent of the rest: the sum's deviation, five times
    step = (feats.abs().amax(1, keepdim=True) / 254) * weight.double().norm(dim=1) + feats.norm(dim=1, keepdim=True) * (weight.double().abs().amax(1) / 254)
    near(got.cpu(), full, 5 * step + half(dtype) * full.abs() + 1e-4, 'against the unquantised layer')


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,inner,cols', [(5, 8, 1), (31, 16, 33), (33, 24, 127), (129, 32, 128), (1000, 40, 129), (300, 56, 5000), (257, 64, 300), (16384, 128, 128), (16411, 72, 100)])
def test_int8_linear_short_rows(ops, rows, inner, cols, dtype):
    """Rows that are quantised where they are multiplied give the bits of the two calls; rows with NaN and infinities, of zeros and of tiny values among them."""
    g = torch.Generator().manual_seed(rows + inner)
    store = torch.randn(rows, inner + 16, generator=g).to(dtype)
    x = store[:, :inner]
    x[1], x[2, 1], x[3, 2], x[4] = 0, float('nan'), float('-inf'), x[4] * torch.finfo(dtype).tiny
    store[:, inner:] = float('nan')   # behind the rows
    qw, sw = ops.quantize_rows(torch.randn(cols, inner, generator=g).cuda())
    bias = torch.randn(cols, generator=g).cuda()
    xd = store.cuda()[:, :inner]
    out = ops.int8_linear(xd, qw, sw, bias)
    want = ops.int8_matmul(*ops.quantize_rows(xd), qw, sw, bias, dtype)
    assert torch.equal(out.view(torch.uint8), want.view(torch.uint8)) and out[2:4].isnan().all() and not out[4:].isnan().any()
    q, s = quantize64(torch.where(x.isfinite(), x, torch.zeros_like(x)))   # (the two rows that are not finite are left out below)
    exact = (q.double() @ qw.cpu().double().t()) * s.double()[:, None] * sw.cpu().double() + bias.cpu().double()
    fine = [r for r in range(min(rows, 300)) if r not in (2, 3)]
    close = exact[fine]
    near(out.cpu()[fine], close, 4 * U * ((exact - bias.cpu().double())[fine].abs() + close.abs()) * (1 + half(dtype)) + half(dtype) * close.abs() + tiny(dtype), 'short rows')


# ---- distillation ----------------------------------------------------------------------------------------------------------------

def distill64(z, idx, u, t, w, dtype=torch.float64):
    z, u = z.to(dtype) / t, u.to(dtype) / t
    cols = z.shape[1]
    kept = (idx >= 0) & (idx < cols)
    u = torch.where(kept, u, torch.full_like(u, -math.inf))
    safe = torch.where(kept, idx, torch.zeros_like(idx)).long()
    dead = (w == 0) | (u.amax(1) == -math.inf)
    u0 = torch.where(dead[:, None], torch.zeros_like(u), u)
    z0 = torch.where(dead[:, None], torch.zeros_like(z), z)
    logp, logq = u0.log_softmax(1), z0.log_softmax(1)
    p = logp.exp()
    term = torch.where(p > 0, p * (logp - logq.gather(1, safe)), torch.zeros_like(p))
    loss = t * t * term.sum(1) * w.to(dtype)
    pz = torch.zeros_like(z).scatter_add_(1, safe, torch.where(kept, p, torch.zeros_like(p)))
    grad = (logq.exp() - pz) * (w.to(dtype) * t)[:, None]
    dead = dead | (w == 0)
    return torch.where(dead, torch.zeros_like(loss), loss), torch.where(dead[:, None], torch.zeros_like(grad), grad), logq, pz


def check_distill(ops, z, idx, u, t, w, z_dev=None, **kw):
    zd = z.cuda() if z_dev is None else z_dev
    loss, grad = ops.distill_loss(zd, idx.cuda(), u.cuda(), temperature=t, row_weight=None if w is None else w.cuda(), **kw)
    w64 = torch.ones(z.shape[0]) if w is None else w
    want, want_g, logq, pz = distill64(z, idx, u, t, w64)
    cols, top = z.shape[1], idx.shape[1]
    zmax = torch.where(torch.isfinite(z.double()), z.double(), torch.zeros(1, dtype=torch.float64)).abs().amax(1) / t
    umax = torch.where(torch.isfinite(u.double()), u.double(), torch.zeros(1, dtype=torch.float64)).abs().amax(1) / t
    # the log-sum: a sum's error and four roundings of numbers of the logits' size, each exp good to a few units of its argument
    e_q = chain(cols) + U * (8 * zmax + 16 + 2 * math.log(cols))
    e_p = chain(top) + U * (8 * umax + 16 + 2 * math.log(max(top, 1)))
    aw = w64.double().abs()
    lmax = torch.where(torch.isfinite(logq), logq, torch.zeros(1, dtype=torch.float64)).abs().amax(1)
    near(loss.cpu(), want, aw * t * t * (e_q + e_p * (2 + lmax + 2 * umax + 4) + chain(top) * (lmax + 2 * umax + 4)) + 4 * U * want.abs(), 'loss')
    if grad is not None:
        assert grad.dtype == z.dtype
        fw = (aw * t)[:, None]
        q = logq.exp()
        argq = torch.where(torch.isfinite(logq), logq, torch.zeros(1, dtype=torch.float64)).abs()
        tol = fw * (q * (e_q[:, None] + 4 * U * (1 + argq)) + pz * (e_p[:, None] * 2 + chain(top) + 4 * U)) + 4 * U * want_g.abs()
        near(grad.cpu(), want_g, tol * (1 + half(z.dtype)) + half(z.dtype) * want_g.abs() + tiny(z.dtype), 'grad')
    return loss, grad


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,cols,top', [(1, 1, 1), (3, 2, 2), (64, 14, 5), (5, 14, 14), (9, 63, 7), (2, 64, 64), (7, 300, 20), (130, 1000, 33), (3, 1024, 1024), (5, 4099, 128),
                                           (2, 10007, 64), (3, 32000, 300), (1, 65536, 64), (2, 70001, 50), (2, 131072, 64), (1, 262147, 100), (40, 20000, 10)])
def test_distill(ops, rows, cols, top, dtype):
    z = rnd(rows, cols, seed=rows + cols, dtype=dtype, scale=2.0)
    u, idx = torch.topk(0.5 * z.float() + rnd(rows, cols, seed=cols, scale=2.0), top, dim=1)
    t = [1.0, 2.0, 1.5][(rows + cols) % 3]
    w = torch.rand(rows, generator=torch.Generator().manual_seed(5)) + 0.5 if rows % 2 else None
    loss, grad = check_distill(ops, z, idx, u, t, w)
    again, _ = check_distill(ops, z, idx.int(), u, t, w, grad=False)
    assert torch.equal(loss, again), 'without the gradient, 4-byte indexes'


@pytest.mark.parametrize('dtype', TYPES, ids=str)
@pytest.mark.parametrize('rows,cols', [(65, 32769), (64, 32769), (66, 65536), (3, 32768), (5, 16385)])
def test_distill_on_both_sides_of_the_chunk_rule(ops, rows, cols, dtype):
    z = rnd(rows, cols, seed=rows + cols, dtype=dtype, scale=2.0)
    u, idx = torch.topk(z.float() + rnd(rows, cols, seed=cols), 40, dim=1)
    check_distill(ops, z, idx, u, 2.0, None)


@pytest.mark.parametrize('cols', [14, 500, 5000, 40000, 150000])
def test_distill_padding_and_ignored_rows(ops, cols):
    """Padding indexes, the same index twice, rows without a teacher, rows of weight 0 that hold NaN, masked classes (-inf), -inf in the teacher."""
    rows, top = 12, 6
    z = rnd(rows, cols, seed=cols, scale=2.0)
    idx = torch.randint(0, cols, (rows, top), generator=torch.Generator().manual_seed(1))
    u = rnd(rows, top, seed=2)
    idx[0, 2] = -1
    idx[1, 3:] = cols                       # just outside
    idx[1, 0] = 2 ** 40
    idx[2] = idx[2, 0]                      # one class, six times
    idx[3] = -100                           # no teacher at all
    u[4] = -math.inf                        # none with a probability
    u[5, 1:] = -math.inf                    # all of it on one class
    z[6] = math.nan                         # a padded row: weight 0
    z[7, 1::2] = -math.inf                  # masked classes, none of them kept
    idx[7] = idx[7] // 2 * 2 % (cols - cols % 2)
    u[8] = -3e38                            # as low as finite numbers go
    z[9, 1:] = -3e38                        # the type's lowest value as a mask
    idx[9] = 0
    u[3] = math.nan                         # (padding hides it)
    w = torch.ones(rows)
    w[6] = 0
    w[10] = -2.5
    loss, grad = check_distill(ops, z, idx, u, 2.0, w)
    loss, grad = loss.cpu(), grad.cpu()
    for r in (3, 4, 6):
        assert loss[r] == 0 and (grad[r] == 0).all(), r
    assert (grad[7, 1::2] == 0).all()
    # a kept class that the student gives no chance at all: the loss is infinite, the gradient finite
    z[0, idx[0, 0]] = -math.inf
    loss, grad = ops.distill_loss(z.cuda(), idx.cuda(), u.cuda(), 2.0, w.cuda())
    assert loss[0] == math.inf and torch.isfinite(grad[0]).all()
    # NaN in a row that counts stays in that row
    z[11, 5] = math.nan
    loss2, grad2 = ops.distill_loss(z.cuda(), idx.cuda(), u.cuda(), 2.0, w.cuda())
    assert torch.isnan(loss2[11]) and torch.isnan(grad2[11]).all() and torch.equal(loss2[:11], loss[:11]) and torch.equal(grad2[:11], grad[:11])


@pytest.mark.parametrize('cols', [14, 1000, 9001, 66000])
def test_distill_strides(ops, cols):
    z = rnd(2, 3, cols + 3, seed=3)
    idx = torch.randint(0, cols, (2, 3, 9), generator=torch.Generator().manual_seed(2))
    u = rnd(2, 3, 9, seed=4)
    zd, idd, ud = z.cuda()[..., 1:1 + cols], idx.cuda()[..., 2:7], u.cuda()[..., 1:6]
    loss, grad = ops.distill_loss(zd, idd, ud, 1.5)
    assert loss.shape == (2, 3) and grad.shape == (2, 3, cols)
    want, want_g, _, _ = distill64(z[..., 1:1 + cols].reshape(6, cols), idx[..., 2:7].reshape(6, 5), u[..., 1:6].reshape(6, 5), 1.5, torch.ones(6))
    near(loss.cpu().view(6), want, 1e-5 * (1 + want.abs()), 'loss')
    near(grad.cpu().view(6, cols), want_g, 1e-5 * want_g.abs() + 1e-6, 'grad')


def test_distill_gradient_by_differences(ops):
    rows, cols, top, t = 4, 40, 6, 2.0
    z, idx, u = rnd(rows, cols, seed=8), torch.randint(0, cols, (rows, top), generator=torch.Generator().manual_seed(4)), rnd(rows, top, seed=9)
    w = torch.rand(rows, generator=torch.Generator().manual_seed(6)) + 0.5
    _, grad = ops.distill_loss(z.cuda(), idx.cuda(), u.cuda(), t, w.cuda())
    d = rnd(rows, cols, seed=10).double()
    f = lambda x: float(distill64(x, idx, u, t, w)[0].sum())
    slope = (f(z.double() + 1e-5 * d) - f(z.double() - 1e-5 * d)) / 2e-5
    got = float((grad.cpu().double() * d).sum())
    assert abs(slope - got) <= 2e-5 * float((grad.cpu().double() * d).abs().sum())


def test_distill_empty(ops):
    z = torch.zeros(0, 9, device='cuda')
    loss, grad = ops.distill_loss(z, torch.zeros(0, 3, dtype=torch.int64, device='cuda'), torch.zeros(0, 3, device='cuda'))
    assert loss.shape == (0,) and grad.shape == (0, 9)
    z = torch.zeros(2, 9, device='cuda')          # no teacher logits at all: nothing to learn from
    loss, grad = ops.distill_loss(z, torch.zeros(2, 0, dtype=torch.int64, device='cuda'), torch.zeros(2, 0, device='cuda'))
    assert (loss == 0).all() and (grad == 0).all()


# ---- far offsets -----------------------------------------------------------------------------------------------------------------

def test_offsets_past_32_bits(ops):
    """Rows 2^30 + 24 elements apart: the last one begins past 2^31 elements, 2^32 bytes."""
    cols, ld = 96, (1 << 30) + 24
    store = torch.zeros(3 * ld, dtype=BF16, device='cuda')
    x = torch.as_strided(store, (3, cols), (ld, 1))
    val = rnd(3, cols, seed=1, dtype=BF16)
    x.copy_(val)
    c = val.cuda()
    y, m, r = ops.layer_norm(x, statistics=True)
    y2, m2, r2 = ops.layer_norm(c, statistics=True)
    assert torch.equal(y, y2) and torch.equal(m, m2) and torch.equal(r, r2)
    assert torch.equal(ops.layer_norm_backward(x, x, m, r)[0], ops.layer_norm_backward(c, c, m, r)[0])
    q, s = ops.quantize_rows(x)
    q2, s2 = ops.quantize_rows(c)
    assert torch.equal(q, q2) and torch.equal(s, s2)
    idx, u = torch.randint(0, cols, (3, 4), device='cuda'), torch.randn(3, 4, device='cuda')
    for a, b in zip(ops.distill_loss(x, idx, u), ops.distill_loss(c, idx, u)):
        assert torch.equal(a, b)
    qs = torch.as_strided(store.view(torch.int8), (3, cols), (2 * ld, 1))
    qs.copy_(q)
    w, ws = ops.quantize_rows(torch.randn(40, cols, device='cuda'))
    assert torch.equal(ops.int8_matmul(qs, s, w, ws), ops.int8_matmul(q, s, w, ws))
    assert torch.equal(ops.int8_matmul(w, ws, qs, s), ops.int8_matmul(w, ws, q, s))


def test_far_rows_of_products(ops):
    """Operands and results past 2^32 bytes, in the one-launch form for short rows and in the tiles."""
    m, k, n = (1 << 25) + 77, 64, 70
    x = torch.zeros(m, k, dtype=BF16, device='cuda')
    ends = torch.cat([torch.arange(3), torch.arange(m - 300, m)]).cuda()
    x[ends] = rnd(303, k, seed=1, dtype=BF16).cuda()
    w, ws = ops.quantize_rows(rnd(n, k, seed=2).cuda())
    bias = rnd(n, seed=3).cuda()
    out = ops.int8_linear(x, w, ws, bias)
    assert torch.equal(out[ends], ops.int8_linear(x[ends], w, ws, bias))
    assert torch.equal(out[m // 2], bias.to(BF16))
    del out
    q, s = ops.quantize_rows(x)
    assert torch.equal(q[ends], ops.quantize_rows(x[ends])[0])
    w, ws = ops.quantize_rows(rnd(130, k, seed=4).cuda())
    out = ops.int8_matmul(q, s, w, ws, out_dtype=BF16)
    assert torch.equal(out[ends], ops.int8_matmul(q[ends], s[ends], w, ws, out_dtype=BF16))
    assert not out[m // 2].any()


# ---- together, on streams, in graphs ---------------------------------------------------------------------------------------------

def head_step(ops, feats, gamma, beta, W, teacher_q, teacher_s, teacher_norm, top, t):
    """A student head learns from a teacher head that is served in 8 bits: norm, projection, loss, and all gradients."""
    logits_t = ops.int8_linear(feats, teacher_q, teacher_s, norm=teacher_norm, out_dtype=F32)
    u, idx = torch.topk(logits_t, top, dim=1)
    h, mean, rstd = ops.layer_norm(feats, gamma, beta, act='lrelu', statistics=True)
    logits = h @ W.t()
    w = torch.full((feats.shape[0],), 1 / feats.shape[0], device='cuda')
    loss, dlogits = ops.distill_loss(logits, idx, u, temperature=t, row_weight=w)
    dW = dlogits.t().contiguous() @ h
    dh = dlogits @ W
    dfeats, dgamma, dbeta = ops.layer_norm_backward(dh, feats, mean, rstd, gamma, beta, act='lrelu')
    return loss, dfeats, dgamma, dbeta, dW


@pytest.mark.parametrize('rows,cols,classes', [(64, 512, 14), (9, 300, 250)])
def test_head_learns_from_an_8bit_teacher(ops, rows, cols, classes):
    feats, gamma, beta = rnd(rows, cols, seed=1, scale=2.0), rnd(cols, seed=2, scale=0.2, shift=1.0), rnd(cols, seed=3, scale=0.2)
    W, Wt = rnd(classes, cols, seed=4, scale=cols ** -0.5), rnd(classes, cols, seed=5, scale=2 * cols ** -0.5)
    tq, ts = ops.quantize_rows(Wt.cuda())
    tn = (rnd(cols, seed=6, shift=1.0, scale=0.1).cuda(), None, 1e-5)
    args = (feats.cuda(), gamma.cuda(), beta.cuda(), W.cuda(), tq, ts, tn, 5, 2.0)
    got = head_step(ops, *args)
    # the same by autograd in 64 bits, from the same teacher logits
    u, idx = torch.topk(ops.int8_linear(args[0], tq, ts, norm=tn, out_dtype=F32), 5, dim=1)
    p = [t.double().requires_grad_() for t in (feats, gamma, beta, W)]
    m, r, xh, z = norm64(p[0], p[1], p[2], 1e-5)
    h = torch.nn.functional.leaky_relu(z, 0.2)
    loss = distill64(h @ p[3].t(), idx.cpu(), u.cpu(), 2.0, torch.full((rows,), 1 / rows))[0]
    loss.sum().backward()
    near(got[0].cpu(), loss.detach(), 1e-4 * loss.detach().abs() + 1e-6, 'loss')
    for name, g, q in zip(('features', 'gamma', 'beta', 'W'), got[1:], p):
        near(g.cpu(), q.grad, 2e-4 * q.grad.abs() + 2e-5 * q.grad.abs().max(), name)


def test_on_another_stream_and_in_a_graph(ops):
    rows, cols, classes = 70, 260, 1000
    feats, gamma, beta = rnd(rows, cols, seed=1).cuda(), rnd(cols, seed=2).cuda(), rnd(cols, seed=3).cuda()
    wide = rnd(rows, 40000, seed=7).cuda()           # a row over several blocks
    W = rnd(classes, cols, seed=4, scale=0.1).cuda()
    tq, ts = ops.quantize_rows(rnd(classes, cols, seed=5).cuda())
    xq, xs = ops.quantize_rows(feats)
    idx, u = torch.randint(0, 40000, (rows, 8), device='cuda'), torch.randn(rows, 8, device='cuda')
    lidx = torch.randint(0, classes, (rows, 8), device='cuda')

    def work():
        h, mean, rstd = ops.layer_norm(feats, gamma, beta, act='relu', statistics=True)
        out = [h, *ops.layer_norm_backward(h, feats, mean, rstd, gamma, beta, act='relu')]
        logits = ops.int8_linear(h, tq, ts)
        out += [logits, ops.int8_linear(h[:1], tq, ts), *ops.distill_loss(logits, lidx, u), *ops.distill_loss(wide[:3], idx[:3], u[:3])]
        out += ops.quantize_rows(feats, norm=(gamma, beta, 1e-5))
        return out

    eager = [t.clone() for t in work()]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for a, b in zip(work(), eager):
            assert torch.equal(a, b)
    torch.cuda.current_stream().wait_stream(s)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    with torch.cuda.graph(other):
        held2 = work()
    for step in range(4):
        feats.copy_(rnd(rows, cols, seed=50 + step))
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        now = work()
        for i, (a, b, c) in enumerate(zip(held, held2, now)):
            assert torch.equal(a, c) and torch.equal(b, c), (step, i)


def test_products_in_a_graph(ops):
    """Every form of the 8-bit linear layer, captured twice and replayed between eager calls."""
    shapes = [(1, 256, 40), (3, 256, 9000), (20, 256, 70), (300, 40, 300), (600, 256, 1030), (70, 130, 20000), (2000, 136, 1900), (4000, 256, 2000), (4100, 256, 2100), (16384, 128, 100)]
    data = []
    for i, (m, k, n) in enumerate(shapes):
        data.append((rnd(m, k, seed=i, dtype=BF16).cuda(), *ops.quantize_rows(rnd(n, k, seed=100 + i).cuda())))

    def work():
        return [ops.int8_linear(*d) for d in data]
    work()
    graphs, held = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            held.append(work())
    for step in range(3):
        for i, d in enumerate(data):
            d[0].copy_(rnd(*d[0].shape, seed=1000 * step + i, dtype=BF16))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b, c, shape in zip(*held, work(), shapes):
            assert torch.equal(a, c) and torch.equal(b, c), (step, shape)


def test_two_threads(ops):
    """Calls of two threads on streams of their own, each with the results of a call alone."""
    import threading
    sets = []
    for i in range(2):
        x, w = rnd(300, 1000 + 24 * i, seed=i).cuda(), rnd(1000 + 24 * i, seed=5 + i).cuda()
        q, s = ops.quantize_rows(rnd(500, 1000 + 24 * i, seed=7 + i).cuda())
        sets.append((x, w, q, s, torch.randint(0, 1000, (300, 9), device='cuda'), rnd(300, 9, seed=9 + i).cuda()))

    def work(x, w, q, s, idx, u):
        y, m, r = ops.layer_norm(x, w, None, act='relu', statistics=True)
        return [y, *ops.layer_norm_backward(y, x, m, r, w, None, act='relu')[:2], ops.int8_linear(x, q, s), *ops.distill_loss(x, idx, u)]
    want = [work(*d) for d in sets]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = work(*sets[i])
            stream.synchronize()
        if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
            wrong.append(i)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_repeats_bit_for_bit(ops):
    x, dy = rnd(5000, 700, seed=1).cuda(), rnd(5000, 700, seed=2).cuda()
    w = rnd(700, seed=3).cuda()
    _, m, r = ops.layer_norm(x, w, w, statistics=True)
    first = ops.layer_norm_backward(dy, x, m, r, w, w)
    z, idx, u = rnd(3, 90000, seed=4).cuda(), torch.randint(0, 90000, (3, 16), device='cuda'), torch.randn(3, 16, device='cuda')
    idx[0] = idx[0, 0]
    d = ops.distill_loss(z, idx, u)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.layer_norm_backward(dy, x, m, r, w, w)))
        assert all(torch.equal(a, b) for a, b in zip(d, ops.distill_loss(z, idx, u)))


# ---- refusals --------------------------------------------------------------------------------------------------------------------

def test_refusals(ops):
    from edgegan_amd import EdgeGANLibError
    x, v = torch.randn(4, 32, device='cuda'), torch.ones(32, device='cuda')
    m = torch.ones(4, device='cuda')
    q, s = ops.quantize_rows(x)
    idx, u = torch.zeros(4, 3, dtype=torch.int64, device='cuda'), torch.zeros(4, 3, device='cuda')
    bad = [
        lambda: ops.layer_norm(x.cpu()), lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x.t()), lambda: ops.layer_norm(x, v[:31]),
        lambda: ops.layer_norm(x, v.cpu()), lambda: ops.layer_norm(x, v.half()), lambda: ops.layer_norm(x, v, v.bfloat16()), lambda: ops.layer_norm(x, eps=0.0),
        lambda: ops.layer_norm(x, eps=math.nan), lambda: ops.layer_norm(x, eps=None), lambda: ops.layer_norm(x, act=['relu']), lambda: ops.distill_loss(x, idx, u, temperature='2'), lambda: ops.layer_norm(x, act='tanh'), lambda: ops.layer_norm(torch.empty(3, 0, device='cuda')),
        lambda: ops.layer_norm(torch.zeros((), device='cuda')), lambda: ops.layer_norm(x.view(2, 2, 32).transpose(0, 1)), lambda: ops.layer_norm(x[:1].expand(4, 32)),
        lambda: ops.layer_norm_backward(x[:3], x, m, m), lambda: ops.layer_norm_backward(x.half(), x, m, m), lambda: ops.layer_norm_backward(x, x, m[:3], m),
        lambda: ops.layer_norm_backward(x, x, None, m), lambda: ops.layer_norm_backward(x, x, m.half(), m),
        lambda: ops.quantize_rows(x.int()), lambda: ops.quantize_rows(x, norm=(v, v)), lambda: ops.quantize_rows(x, norm=(v.half(), None, 1e-5)),
        lambda: ops.quantize_rows(x, norm=(v, v, -1.0)), lambda: ops.quantize_rows(torch.empty(2, 0, device='cuda')),
        lambda: ops.int8_matmul(x, s, q, s), lambda: ops.int8_matmul(q, s, q[:, :16], s), lambda: ops.int8_matmul(q, s, q, s[:3]),
        lambda: ops.int8_matmul(q, None, q, s), lambda: ops.int8_matmul(q, s, q, s, bias=v), lambda: ops.int8_matmul(q, s, q, s, out_dtype=torch.float64),
        lambda: ops.int8_matmul(q, s, q.view(2, 2, 32), s), lambda: ops.int8_matmul(q, s, q.cpu(), s),
        lambda: ops.int8_matmul(*[torch.zeros(1, 131072, dtype=torch.int8, device='cuda'), torch.ones(1, device='cuda')] * 2),
        lambda: ops.distill_loss(x, idx, u[:, :2]), lambda: ops.distill_loss(x, idx.float(), u), lambda: ops.distill_loss(x, idx, u.half()),
        lambda: ops.distill_loss(x, idx[:3], u[:3]), lambda: ops.distill_loss(x, idx, u, temperature=0.0), lambda: ops.distill_loss(x, idx, u, temperature=-1.0),
        lambda: ops.distill_loss(x, idx, u, temperature=math.inf), lambda: ops.distill_loss(x, idx, u, row_weight=m[:3]), lambda: ops.distill_loss(x, idx.cpu(), u),
        lambda: ops.distill_loss(x, torch.zeros(4, 1025, dtype=torch.int64, device='cuda'), torch.zeros(4, 1025, device='cuda')),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(EdgeGANLibError):
            f()
            pytest.fail(f'case {i} was taken')
    lib = ops._library()                             # a device that is not there: an error code, and the current device stays
    before = torch.cuda.current_device()
    assert lib.eg_layer_norm(63, None, 0, x.data_ptr(), 32, 0, None, None, 4, 32, 1e-5, 0, x.data_ptr(), 32, None, None) != 0
    assert torch.cuda.current_device() == before
    assert torch.isfinite(ops.layer_norm(x)).all()   # nothing is left behind


def test_in_place(ops):
    """The C entries may write over x, dy and the logits (same distance between rows)."""
    lib, st = ops._library(), torch.cuda.current_stream().cuda_stream
    for rows, cols in ((9, 100), (5, 1001), (3, 5000), (2, 40003), (2, 70000)):
        x, dy, w = rnd(rows, cols, seed=1).cuda(), rnd(rows, cols, seed=2).cuda(), rnd(cols, seed=3).cuda()
        y, m, r = ops.layer_norm(x, w, w, act='lrelu', statistics=True)
        dx, dw, db = ops.layer_norm_backward(dy, x, m, r, w, w, act='lrelu')
        z = x.clone()
        assert lib.eg_layer_norm(0, st, 0, z.data_ptr(), cols, 0, w.data_ptr(), w.data_ptr(), rows, cols, 1e-5, 2, z.data_ptr(), cols, None, None) == 0
        assert torch.equal(z, y), (rows, cols)
        g, gw = dy.clone(), torch.empty(2, cols, device='cuda')
        size = lib.eg_layer_norm_workspace(rows, cols)
        ws = torch.empty(size, dtype=torch.uint8, device='cuda')
        assert lib.eg_layer_norm_backward(0, st, 0, g.data_ptr(), cols, x.data_ptr(), cols, m.data_ptr(), r.data_ptr(), 0, w.data_ptr(), w.data_ptr(), rows, cols, 2,
                                          g.data_ptr(), cols, gw[0].data_ptr(), gw[1].data_ptr(), ws.data_ptr(), size) == 0
        assert torch.equal(g, dx) and torch.equal(gw[0], dw) and torch.equal(gw[1], db), (rows, cols)
        idx, u = torch.randint(0, cols, (rows, 6), device='cuda'), torch.randn(rows, 6, device='cuda')
        loss, grad = ops.distill_loss(x, idx, u, 2.0)
        z, l2 = x.clone(), torch.empty(rows, device='cuda')
        size = lib.eg_distill_loss_workspace(rows, cols, 6)
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device='cuda')
        assert lib.eg_distill_loss(0, st, 0, z.data_ptr(), cols, 8, idx.data_ptr(), 6, u.data_ptr(), 6, None, rows, cols, 6, 2.0, l2.data_ptr(), z.data_ptr(), cols,
                                   ws.data_ptr(), size) == 0
        assert torch.equal(z, grad) and torch.equal(l2, loss), (rows, cols)


def test_gradient_parts(ops):
    """dx alone and the parameters' gradients alone, through the C entry; both are the whole call's."""
    lib, st = ops._library(), torch.cuda.current_stream().cuda_stream
    for rows, cols in ((300, 70), (4, 3001), (2, 50001)):
        x, dy, w = rnd(rows, cols, seed=1).cuda(), rnd(rows, cols, seed=2).cuda(), rnd(cols, seed=3).cuda()
        _, m, r = ops.layer_norm(x, w, None, statistics=True)
        dx, dw, _ = ops.layer_norm_backward(dy, x, m, r, w, None)
        size = lib.eg_layer_norm_workspace(rows, cols)
        ws = torch.empty(size, dtype=torch.uint8, device='cuda')
        a, b = torch.empty_like(x), torch.empty(cols, device='cuda')
        args = (0, st, 0, dy.data_ptr(), cols, x.data_ptr(), cols, m.data_ptr(), r.data_ptr(), 0, w.data_ptr(), None, rows, cols, 0)
        assert lib.eg_layer_norm_backward(*args, a.data_ptr(), cols, None, None, None, 0) == 0
        assert lib.eg_layer_norm_backward(*args, None, 0, b.data_ptr(), None, ws.data_ptr(), size) == 0
        assert torch.equal(a, dx) and torch.equal(b, dw), (rows, cols)
