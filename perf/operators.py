"""The row operators of edgegan_amd.ops as cases that can be timed and compared: layer norm and its gradient, linear
layers in 8-bit integers, distillation from a teacher's top logits.

`run` computes a case in elementary torch operations (own = False) or through edgegan_amd.ops (own = True)."""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SIZE = {'f32': 4, 'bf16': 2, 'f16': 2}
EPS = 1e-5
SLOPE = 0.2   # LeakyReLU of the discriminators


def listed():
    return [
        # the norm behind the patch discriminators' second convolution at batch 64: 32 x 32 positions of 128 channels
        dict(name='norm_maps', kind='norm', rows=65536, cols=128, dtype='f32', wtype='f32', act='lrelu'),
        # one position's features while a head answers a single request
        dict(name='norm_single', kind='norm', rows=1, cols=4096, dtype='bf16', wtype='bf16', act='none'),
        # features of an odd width, as a concatenation leaves them
        dict(name='norm_odd', kind='norm', rows=1023, cols=5001, dtype='f16', wtype='f16', act='relu'),
        # the gradient of norm_maps
        dict(name='norm_backward_maps', kind='norm_backward', rows=65536, cols=128, dtype='f32', wtype='f32', act='lrelu'),
        # wide features in half precision, with parameters kept in 32 bits: the largest map of a wide model
        dict(name='norm_backward_wide', kind='norm_backward', rows=16384, cols=4096, dtype='bf16', wtype='f32', act='none'),
        # a head's linear layer behind its norm, for a single request: the weights' bytes count
        dict(name='linear_single', kind='linear', rows=1, inner=4096, cols=4096, dtype='bf16', norm=True, bias=True),
        # the same for a small batch of requests, odd sizes
        dict(name='linear_few', kind='linear', rows=23, inner=2050, cols=8190, dtype='f16', norm=False, bias=True),
        # the encoder's first shortcut (64 to 128 channels, 32 x 32 positions) at batch 64
        dict(name='linear_shortcut', kind='linear', rows=65536, inner=64, cols=128, dtype='f32', norm=False, bias=True),
        # a large batch through a wide layer: the matrix cores count
        dict(name='linear_large', kind='linear', rows=8192, inner=4096, cols=8192, dtype='bf16', norm=False, bias=False),
        # the classifier's 14 logits at batch 64, from a teacher's five best
        dict(name='distill_classes', kind='distill', rows=64, cols=14, top=5, dtype='f32', temperature=2.0, ignored=False),
        # an output layer of an odd size
        dict(name='distill_odd', kind='distill', rows=511, cols=10007, top=20, dtype='f16', temperature=1.0, ignored=False),
        # a large output layer, with a part of the rows left out
        dict(name='distill_large', kind='distill', rows=4096, cols=65536, top=64, dtype='bf16', temperature=1.5, ignored=True),
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    def odd(n):   # half of the sizes end where a vector of 16 bytes does
        return max(16, n // 16 * 16) if n >= 16 and rng.random() < 0.5 else n

    kind = rng.choice(['norm', 'norm_backward', 'linear', 'distill'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    if kind in ('norm', 'norm_backward'):
        cols = odd(size(16, 8192))
        rows = size(1, max(1, min(65536, (1 << 26) // cols)))
        return dict(kind=kind, rows=rows, cols=cols, dtype=dtype, wtype=rng.choice(['f32', dtype]), act=rng.choice(['none', 'relu', 'lrelu']))
    if kind == 'linear':
        inner, cols = odd(size(32, 8192)), odd(size(16, 8192))
        # (a norm's last bit decides which of two neighbouring 8-bit values a number halfway between them takes: no case in 32 bits)
        return dict(kind=kind, rows=size(1, max(1, min(8192, (1 << 38) // (inner * cols)))), inner=inner, cols=cols, dtype=dtype,
                    norm=dtype != 'f32' and rng.random() < 0.5, bias=rng.random() < 0.5)
    cols = size(10, 65536)
    rows = size(1, max(1, min(8192, (1 << 28) // cols)))
    return dict(kind=kind, rows=rows, cols=cols, top=size(1, min(cols, 128)), dtype=dtype, temperature=rng.choice([1.0, 1.5, 2.0, 4.0]),
                ignored=rng.random() < 0.5)


def features(g, rows, cols, dtype):
    """Rows as a convolution or a linear layer leaves them: channels of unlike level and spread."""
    level = torch.randn(cols, generator=g, device='cuda') * 0.5
    spread = torch.rand(cols, generator=g, device='cuda') + 0.5
    x = torch.randn(rows, cols, generator=g, device='cuda')
    return x.mul_(spread).add_(level).to(TYPES[dtype])


def parameters(g, cols, dtype):
    return ((1 + 0.1 * torch.randn(cols, generator=g, device='cuda')).to(TYPES[dtype]),
            (0.1 * torch.randn(cols, generator=g, device='cuda')).to(TYPES[dtype]))


def padded(q):
    """8-bit rows at a pitch of whole 16-byte groups: how a program keeps a quantised filter."""
    p = torch.zeros(q.shape[0], (q.shape[1] + 15) // 16 * 16, dtype=torch.int8, device=q.device)
    p[:, :q.shape[1]] = q
    return p[:, :q.shape[1]]


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    kind, rows, cols = case['kind'], case['rows'], case['cols']
    s = dict(case)
    if kind in ('norm', 'norm_backward'):
        s['x'] = features(g, rows, cols, case['dtype'])
        s['weight'], s['bias'] = parameters(g, cols, case['wtype'])
        if kind == 'norm_backward':
            s['dy'] = torch.randn(rows, cols, generator=g, device='cuda').to(TYPES[case['dtype']])
            _, s['mean'], s['rstd'] = plain_statistics(s['x'].float())
    elif kind == 'linear':
        inner = case['inner']
        s['x'] = features(g, rows, inner, case['dtype'])
        s['gamma'], s['beta'] = parameters(g, inner, 'f32') if case['norm'] else (None, None)
        w = torch.randn(cols, inner, generator=g, device='cuda') / math.sqrt(inner)
        q, s['wscale'] = plain_quantize(w)
        s['w'] = padded(q.to(torch.int8))
        s['bias_'] = (0.1 * torch.randn(cols, generator=g, device='cuda')) if case['bias'] else None
    else:
        s['x'] = (2 * torch.randn(rows, cols, generator=g, device='cuda')).to(TYPES[case['dtype']])
        teacher = torch.randn(rows, cols, generator=g, device='cuda').mul_(2).add_(s['x'].float(), alpha=0.5)
        s['teacher'], s['index'] = torch.topk(teacher, case['top'], dim=1)
        # the mean over the rows; in f16 with a loss scale, as training in that type has one
        weight = torch.full((rows,), (4096.0 if case['dtype'] == 'f16' else 1.0) / rows, device='cuda')
        if case['ignored']:
            weight *= (torch.rand(rows, generator=g, device='cuda') < 0.9)
        s['row_weight'] = weight
    return s


def plain_statistics(x):
    mean = x.mean(1)
    d = x - mean[:, None]
    return d, mean, 1 / torch.sqrt((d * d).mean(1) + EPS)


def plain_act(z, act):
    if act == 'none':
        return z
    return torch.where(z > 0, z, z * (SLOPE if act == 'lrelu' else 0.0))


def plain_quantize(x):
    """The 8-bit rows (as floats) and their scales: whole numbers nearest to 127 x / max |x|, a tie to the even one. In 64 bits,
    since a value next to a border decides by its last bit."""
    d = x.double()
    amax = d.abs().amax(1)
    q = torch.round(d * 127 / torch.where(amax > 0, amax, torch.ones_like(amax))[:, None])
    return q.float(), (amax / 127).float()


def plain(s):
    kind, x = s['kind'], s['x'].float()
    if kind == 'norm':
        d, mean, rstd = plain_statistics(x)
        y = plain_act(d * rstd[:, None] * s['weight'].float() + s['bias'].float(), s['act'])
        return dict(y=y.to(s['x'].dtype), mean=mean, rstd=rstd)
    if kind == 'norm_backward':
        w, g = s['weight'].float(), s['dy'].float()
        xh = (x - s['mean'][:, None]) * s['rstd'][:, None]
        if s['act'] != 'none':
            g = torch.where(xh * w + s['bias'].float() > 0, g, g * (SLOPE if s['act'] == 'lrelu' else 0.0))
        gw = g * w
        dx = (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True)) * s['rstd'][:, None]
        return dict(dx=dx.to(s['x'].dtype), dweight=(g * xh).sum(0).to(s['weight'].dtype), dbias=g.sum(0).to(s['weight'].dtype))
    if kind == 'linear':
        if s['norm']:
            d, _, rstd = plain_statistics(x)
            x = d * rstd[:, None] * s['gamma'] + s['beta']
        q, scale = plain_quantize(x)
        y = torch.matmul(q, s['w'].float().t()) * scale[:, None] * s['wscale']
        if s['bias_'] is not None:
            y = y + s['bias_']
        return dict(y=y.to(s['x'].dtype))
    t = s['temperature']
    z, u = x / t, s['teacher'] / t
    zmax, umax = z.amax(1, keepdim=True), u.amax(1, keepdim=True)
    logq = z - zmax - torch.log(torch.exp(z - zmax).sum(1, keepdim=True))
    logp = u - umax - torch.log(torch.exp(u - umax).sum(1, keepdim=True))
    p, w = torch.exp(logp), s['row_weight']
    loss = w * t * t * (p * (logp - torch.gather(logq, 1, s['index']))).sum(1)
    grad = torch.exp(logq).scatter_add_(1, s['index'], -p) * (w * t)[:, None]
    return dict(loss=loss, grad=grad.to(s['x'].dtype))


def run(state):
    if not own:
        return plain(state)
    from edgegan_amd import ops
    s, kind = state, state['kind']
    if kind == 'norm':
        y, mean, rstd = ops.layer_norm(s['x'], s['weight'], s['bias'], eps=EPS, act=s['act'], statistics=True)
        return dict(y=y, mean=mean, rstd=rstd)
    if kind == 'norm_backward':
        dx, dweight, dbias = ops.layer_norm_backward(s['dy'], s['x'], s['mean'], s['rstd'], s['weight'], s['bias'], act=s['act'])
        return dict(dx=dx, dweight=dweight, dbias=dbias)
    if kind == 'linear':
        norm = (s['gamma'], s['beta'], EPS) if s['norm'] else None
        return dict(y=ops.int8_linear(s['x'], s['w'], s['wscale'], s['bias_'], norm=norm))
    loss, grad = ops.distill_loss(s['x'], s['index'], s['teacher'], temperature=s['temperature'], row_weight=s['row_weight'])
    return dict(loss=loss, grad=grad)


def work(case):
    kind, rows, cols = case['kind'], case['rows'], case['cols']
    e = SIZE[case['dtype']]
    n = rows * cols
    if kind == 'norm':
        return dict(bytes=2 * n * e + 2 * cols * SIZE[case['wtype']] + 8 * rows, flops=8 * n)
    if kind == 'norm_backward':
        return dict(bytes=3 * n * e + 4 * cols * SIZE[case['wtype']] + 8 * rows, flops=14 * n)
    if kind == 'linear':
        k = case['inner']
        return dict(bytes=rows * k * e + cols * k + 4 * cols * (2 if case['bias'] else 1) + n * e + (8 * k if case['norm'] else 0), flops=2 * n * k)
    return dict(bytes=2 * n * e + rows * case['top'] * 12 + 8 * rows, flops=6 * n)


def exact(case, seed):
    """The definitions, row by row in matrices of 64-bit numbers."""
    s = prepare(case, seed)
    kind, x = case['kind'], s['x'].double()
    slope = {'none': 1.0, 'relu': 0.0, 'lrelu': SLOPE}[case.get('act', 'none')]
    if kind == 'norm':
        var, mean = torch.var_mean(x, dim=1, correction=0)
        rstd = (var + EPS) ** -0.5
        z = torch.addcmul(s['bias'].double(), (x - mean.unsqueeze(1)) * rstd.unsqueeze(1), s['weight'].double())
        return dict(y=z.clamp(min=0) + slope * z.clamp(max=0), mean=mean, rstd=rstd)
    if kind == 'norm_backward':
        r = s['rstd'].double().unsqueeze(1)
        xhat = (x - s['mean'].double().unsqueeze(1)) * r
        passed = ((xhat * s['weight'].double() + s['bias'].double()) > 0).double()
        g = s['dy'].double() * (passed + slope * (1 - passed))
        dxhat = g * s['weight'].double()
        a = dxhat.sum(1, keepdim=True) / x.shape[1]
        b = (dxhat * xhat).sum(1, keepdim=True) / x.shape[1]
        return dict(dx=r * (dxhat - a - b * xhat), dweight=torch.mul(g, xhat).sum(0), dbias=g.sum(0))
    if kind == 'linear':
        if case['norm']:
            var, mean = torch.var_mean(x, dim=1, correction=0)
            x = (x - mean.unsqueeze(1)) / torch.sqrt(var + EPS).unsqueeze(1) * s['gamma'].double() + s['beta'].double()
        amax = x.abs().max(dim=1).values
        scale = amax / 127
        y = torch.round(127 * x / amax.unsqueeze(1)) @ s['w'].double().t().contiguous()   # whole numbers: exact
        y = y * torch.outer(scale, s['wscale'].double())
        return dict(y=y if s['bias_'] is None else y + s['bias_'].double())
    t, w = case['temperature'], s['row_weight'].double()
    logq = (x / t).log_softmax(dim=1)
    logp = (s['teacher'].double() / t).log_softmax(dim=1)
    p = torch.zeros_like(x)
    for k in range(case['top']):   # one column of the teacher's at a time, an index given twice counting twice
        p[torch.arange(len(x), device=x.device), s['index'][:, k]] += logp[:, k].exp()
    loss = t ** 2 * w * sum(logp[:, k].exp() * (logp[:, k] - logq.gather(1, s['index'][:, k:k + 1])[:, 0]) for k in range(case['top']))
    return dict(loss=loss, grad=t * w.unsqueeze(1) * (logq.exp() - p))
