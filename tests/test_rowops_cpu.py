"""The row operators' C entries on the host: every refusal is an error code and a message, before any device is touched."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

from edgegan_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20      # an address that is never read


def norm(lib, device=0, dtype=0, x=P, ldx=8, wtype=0, rows=2, cols=8, eps=1e-5, act=0, y=P, ldy=8, mean=None, rstd=None):
    return lib.eg_layer_norm(device, None, dtype, x, ldx, wtype, None, None, rows, cols, eps, act, y, ldy, mean, rstd)


def backward(lib, rows=2, cols=8, ws=P, size=1 << 20, mean=P, dgamma=P, x=P, lddx=8):
    return lib.eg_layer_norm_backward(0, None, 0, P, 8, x, 8, mean, P, 0, P, P, rows, cols, 0, P, lddx, dgamma, P, ws, size)


def quantize(lib, rows=2, cols=8, q=P, ldq=16, scale=P, norm=0, gamma=None, eps=1e-5):
    return lib.eg_quantize_rows(0, None, 0, P, 8, norm, gamma, None, eps, rows, cols, q, ldq, scale)


def product(lib, a=P, lda=64, sa=P, m=4, n=4, k=64, out_type=0, ldo=4):
    return lib.eg_int8_matmul(0, None, a, lda, sa, P, 64, P, None, m, n, k, out_type, P, ldo)


def linear(lib, dtype=0, x=P, ldx=64, norm=0, gamma=None, eps=1e-5, w=P, ldw=64, ws=P, rows=2, cols=4, inner=64, out_type=0, out=P, ldo=4, work=P, size=1 << 20):
    return lib.eg_int8_linear(0, None, dtype, x, ldx, norm, gamma, None, eps, w, ldw, ws, None, rows, cols, inner, out_type, out, ldo, work, size)


def distill(lib, rows=2, cols=8, top=3, t=1.0, loss=P, index_bytes=8, index=P, ldi=3, ldg=8):
    return lib.eg_distill_loss(0, None, 0, P, 8, index_bytes, index, ldi, P, 3, None, rows, cols, top, t, loss, P, ldg, P, 1 << 20)


CASES = [
    (norm, dict(dtype=3), 'type'), (norm, dict(wtype=-1), 'type'), (norm, dict(x=None), 'null'), (norm, dict(y=None), 'null'), (norm, dict(ldx=7), 'elements apart'),
    (norm, dict(ldy=-8), 'elements apart'), (norm, dict(rows=-1), 'rows'), (norm, dict(cols=(1 << 24) + 1), 'columns'), (norm, dict(cols=0), 'without columns'),
    (norm, dict(eps=0.0), 'eps'), (norm, dict(eps=float('inf')), 'eps'), (norm, dict(act=3), 'activation'), (norm, dict(mean=P), 'together'), (norm, dict(x=P + 2), 'misaligned'),
    (norm, dict(ldx=1 << 62), 'too large'),
    (norm, dict(wtype=1), 'beside'), (norm, dict(dtype=2, wtype=1), 'beside'), (norm, dict(mean=P + 2, rstd=P), 'misaligned'),
    (backward, dict(ws=None), 'workspace'), (backward, dict(size=4), 'workspace'), (backward, dict(ws=P + 4), 'workspace'), (backward, dict(mean=None), 'statistics'),
    (backward, dict(x=None), 'null'), (backward, dict(lddx=3), 'elements apart'), (backward, dict(cols=0), 'without columns'),
    (quantize, dict(q=None), 'null'), (quantize, dict(ldq=7), 'elements apart'), (quantize, dict(scale=None), 'scale'), (quantize, dict(gamma=P), 'norm'),
    (quantize, dict(norm=1, eps=-1.0), 'eps'), (quantize, dict(cols=0), 'without columns'), (quantize, dict(scale=P + 1), 'misaligned'), (product, dict(sa=P + 2), 'misaligned'), (distill, dict(loss=P + 2), 'misaligned'),
    (product, dict(k=131072, lda=131072), 'overflow'), (product, dict(m=-1), 'sizes'), (product, dict(n=1 << 30), 'sizes'), (product, dict(a=None), 'null'), (product, dict(lda=63), 'elements apart'),
    (product, dict(sa=None), 'scale'), (product, dict(out_type=7), 'type'), (product, dict(ldo=3), 'elements apart'),
    (linear, dict(dtype=9), 'type'), (linear, dict(x=None), 'null'), (linear, dict(ldx=63), 'elements apart'), (linear, dict(gamma=P), 'norm'), (linear, dict(norm=1, eps=0.0), 'eps'),
    (linear, dict(w=None), 'null'), (linear, dict(ldw=1), 'elements apart'), (linear, dict(ws=None), 'scale'), (linear, dict(inner=0), 'without columns'), (linear, dict(inner=1 << 17, ldx=1 << 17, ldw=1 << 17), 'overflow'),
    (linear, dict(work=None), 'workspace'), (linear, dict(size=100), 'workspace'), (linear, dict(out=None), 'null'), (linear, dict(ldo=2), 'elements apart'), (linear, dict(rows=-1), 'sizes'),
    (distill, dict(top=1025, ldi=1025), 'teacher logits'), (distill, dict(t=0.0), 'temperature'), (distill, dict(t=float('nan')), 'temperature'), (distill, dict(t=1e-45), 'temperature'),
    (distill, dict(loss=None), 'loss'), (distill, dict(index_bytes=2), 'bytes'), (distill, dict(index=P + 4), 'misaligned'), (distill, dict(ldi=2), 'elements apart'), (distill, dict(ldg=7), 'elements apart'),
    (distill, dict(cols=0), 'without columns'),
]


@pytest.mark.parametrize('call,args,message', CASES, ids=[f'{c.__name__}-{next(iter(a))}-{i}' for i, (c, a, _) in enumerate(CASES)])
def test_refusals(built_lib, call, args, message):
    assert call(built_lib, **args) == 1
    assert message in built_lib.eg_last_error(None).decode()


def test_nothing_to_do_is_no_error(built_lib):
    """Zero rows: no device is asked for."""
    assert norm(built_lib, rows=0, x=None, y=None) == 0
    assert quantize(built_lib, rows=0) == 0
    assert product(built_lib, m=0, a=None) == 0
    assert distill(built_lib, rows=0) == 0
    assert linear(built_lib, rows=0, x=None) == 0 and linear(built_lib, cols=0, w=None) == 0


def test_workspace_sizes(built_lib):
    assert built_lib.eg_layer_norm_workspace(-1, 8) == -1 and built_lib.eg_layer_norm_workspace(8, (1 << 24) + 1) == -1
    assert built_lib.eg_layer_norm_workspace(0, 8) == 0
    assert built_lib.eg_int8_linear_workspace(1, 131072) == -1 and built_lib.eg_int8_linear_workspace(3, 100) >= 3 * 116
    assert built_lib.eg_distill_loss_workspace(1, -1, 1) == -1 and built_lib.eg_distill_loss_workspace(1, 8, 1025) == -1
    assert built_lib.eg_distill_loss_workspace(4, 1000, 8) >= 0


def test_two_runtimes_are_refused(built_lib):
    """The engine loaded before torch runs on another HIP runtime: the operators say so instead of mixing the two."""
    code = ('import sys; sys.path.insert(0, %r)\n'
            'from edgegan_amd import _lib\n'
            '_lib.load_library()\n'
            'from edgegan_amd import ops\n'
            'runtimes = {l.split()[-1] for l in open("/proc/self/maps") if "libamdhip64" in l}\n'
            'try:\n    ops._library()\n    print("taken", len(runtimes))\n'
            'except _lib.EdgeGANLibError as e:\n    print("refused", len(runtimes))\n' % ROOT)
    out = subprocess.run([sys.executable, '-c', code], capture_output=True, text=True, timeout=300).stdout.split()
    assert out in (['refused', '2'], ['taken', '1']), out


@pytest.mark.parametrize('flags', [dict(G_norm='layernorm'), dict(E_norm='layernorm', D_norm='layernorm'), dict(E_norm='layernorm', G_norm='layernorm', D_norm='layernorm', num_classes=0)])
def test_registry_layer_norm_flags(built_lib, flags):
    """E_norm / G_norm / D_norm = 'layernorm': every normalised block gains a scale and a shift, and nothing else changes."""
    import edgegan_amd as ea
    import edgegan_oracle as O
    cfg = ea.Config(batch_size=2, **flags)
    got = [(s.name, tuple(s.shape), s.trainable) for s in ea.variable_specs(cfg)]
    assert got == [(s.name, tuple(s.shape), s.trainable) for s in O.variable_specs(O.Config(batch_size=2, **flags))]
    names = {n: sh for n, sh, _ in got}
    assert ('G2/g_dconv_3/layer_norm/LayerNorm/gamma' in names) == (cfg.G_norm == 'layernorm')
    assert ('D/d_conv_4/layer_norm/LayerNorm/beta' in names) == (cfg.D_norm == 'layernorm')
    assert ('E/e_resnet_512_4/res2/layer_norm/LayerNorm/gamma' in names) == (cfg.E_norm == 'layernorm')
    assert 'D/d_conv_0/layer_norm/LayerNorm/beta' not in names
    v = ea.init_variables(cfg, seed=1)
    for n in names:
        if n.endswith('LayerNorm/gamma'):
            assert np.all(v[n] == 1)
        elif n.endswith('LayerNorm/beta'):
            assert np.all(v[n] == 0)


def test_layer_norm_flag_reaches_the_engine():
    from edgegan_amd import flags as F, train as TR
    fl = TR.update_flags(F.parse(['--D_norm=layernorm', '--E_norm', 'layernorm'], F.TRAIN_FLAGS))
    F.check_supported(fl)


def test_linear_in_one_launch(built_lib):
    """Which calls need no workspace, and that the others do not go without one."""
    def one(dtype=0, x=P, ldx=64, norm=0, gamma=None, w=P, ldw=64, rows=2, cols=4, inner=64, out_type=0, ldo=4):
        return built_lib.eg_int8_linear_in_one(dtype, x, ldx, norm, gamma, None, w, ldw, rows, cols, inner, out_type, ldo)
    assert one() and one(norm=1) and one(rows=4) and one(rows=100) and one(rows=1, ldx=3, inner=4096, ldw=4096)
    assert one(rows=100000, inner=128, ldx=128, ldw=128, cols=100, ldo=100)
    for no in (dict(x=P + 4), dict(ldx=65), dict(w=P + 8), dict(ldw=72), dict(out_type=1), dict(inner=66, ldx=68, ldw=80), dict(rows=100, norm=1), dict(norm=1, gamma=P + 4),
               dict(rows=100, inner=128, ldx=128, ldw=128), dict(rows=5, inner=4096, ldx=4096, ldw=4096), dict(rows=3, cols=20000, norm=1), dict(dtype=7), dict(rows=-1), dict(inner=0),
               dict(inner=131072), dict(cols=-1), dict(cols=1 << 40)):
        assert not one(**no), no
    assert linear(built_lib, rows=100, norm=1, work=None, size=0) != 0 and b'workspace' in built_lib.eg_last_error(None)


def test_gradient_workspace_sizes(built_lib):
    """Few rows need none, and take none in its place; the others do not go without."""
    size = built_lib.eg_layer_norm_workspace
    for rows, cols in ((128, 32), (64, 64), (32, 128), (16, 1024), (2, 8192), (0, 5), (7, 0)):
        assert size(rows, cols) == 0, (rows, cols)
    for rows, cols in ((129, 32), (65, 64), (33, 128), (17, 1024), (3, 8192), (1, 8193), (1 << 40, 7)):
        assert size(rows, cols) > 0 and size(rows, cols) % 4 == 0, (rows, cols)
    assert backward(built_lib, rows=1000, ws=None, size=0) != 0 and b'workspace' in built_lib.eg_last_error(None)
