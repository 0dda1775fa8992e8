"""The row operators where the engine itself runs them: E_norm / G_norm / D_norm = 'layernorm', the classifier's teacher, inference in 8 bits."""
import math

import numpy as np
import pytest
import torch

import edgegan_amd as ea
import edgegan_oracle as O
import parity

pytestmark = pytest.mark.gpu


def _assert(rows):
    bad = [r for r in rows if not r[1] <= r[2]]
    assert not bad, '\n'.join(f'{n}: err {e:.3e} > tol {t:.1e}' for n, e, t in sorted(bad, key=lambda r: -r[1])[:20])


def moved_parameters(cfg, seed):
    """Initial values with every norm's scale / shift moved off 1 / 0, so that a wrong gradient of theirs shows."""
    values = ea.init_variables(cfg, seed)
    rng = np.random.RandomState(seed + 1)
    for n in values:
        if n.endswith('Norm/gamma'):
            values[n] = (1.0 + 0.2 * rng.standard_normal(values[n].shape)).astype(np.float32)
        elif n.endswith('Norm/beta'):
            values[n] = (0.1 * rng.standard_normal(values[n].shape)).astype(np.float32)
    return values


LN = dict(E_norm='layernorm', G_norm='layernorm', D_norm='layernorm')


@pytest.mark.parametrize('flags', [dict(D_norm='layernorm'), dict(LN, num_classes=0), dict(E_norm='layernorm', G_norm='batch'), dict(LN, compute_dtype='f32x3', num_classes=0),
                                   dict(LN, compute_dtype='bf16', num_classes=0)], ids=['D', 'all_single_class', 'E_with_G_batch', 'all_f32x3', 'all_bf16'])
def test_substeps_layer_norm(flags):
    """Every sub-step against the 64-bit oracle, the gradients of the norms' scale and shift included; in the discriminators that runs the
    layer norm's tangent and the reverse of it (the gradient penalty's second derivative).  Then a whole concurrent iteration and the evaluation."""
    cfg = ea.Config(batch_size=3, **flags)
    values = moved_parameters(cfg, 21)
    net = ea.EdgeGAN(cfg, values)
    bf = cfg.compute_dtype == 'bf16'   # (the tolerances of the other norms' test of this mode)
    rows = parity.substep_checks(net, values, ea.synthetic_batch(cfg, seed=37), bf16=bf, self_consistency=True, grad_tol=0.1 if bf else 1e-2, loss_tol=1e-2 if bf else 1e-4)
    checked = {r[0] for r in rows}
    if cfg.D_norm == 'layernorm':
        for g in ('gamma', 'beta'):
            assert any(f'D_patch2/d_conv_3/layer_norm/LayerNorm/{g}' in r for r in checked)
    _assert(rows)
    net.set_variables(values)
    net.train_step()
    assert all(np.isfinite(v) for v in net.losses().values())
    assert all(np.isfinite(v) for v in net.evaluate().values() if np.isscalar(v))
    net.close()


@pytest.mark.parametrize('flags', [dict(E_norm='layernorm', G_norm='layernorm'), dict(E_norm='layernorm')], ids=['E_G', 'E'])
def test_inference_layer_norm(flags):
    cfg = ea.Config(batch_size=2, **flags)
    values = moved_parameters(cfg, 4)
    net = ea.EdgeGAN(cfg, values)
    om = O.OracleModel(parity.oracle_config(cfg), values, dtype=torch.float64)
    imgs = np.random.RandomState(1).uniform(-1, 1, size=(3, 64, 128, 3)).astype(np.float32)
    cls = np.arange(3, dtype=np.int32)
    e_ref, i_ref = om.infer(parity.t64(imgs), torch.tensor(cls), 0.4, -1.1)
    e, i = net.infer(imgs, cls, eps2=[0.4, -1.1])
    assert parity.relerr(e, e_ref.numpy()) < 1e-4 and parity.relerr(i, i_ref.numpy()) < 1e-4
    net.close()


def test_teacher_of_the_classifier():
    """Sub-step 4's gradient with a teacher against autograd of (focal loss + weight x mean distillation loss) in 64 bits; without one the bits of before."""
    cfg = ea.Config(batch_size=4)
    values = ea.init_variables(cfg, 3)
    batch = ea.synthetic_batch(cfg, seed=5)
    net = ea.EdgeGAN(cfg, values)
    net.upload_batch(**batch)
    specs = [s for s in ea.variable_specs(cfg) if s.name.startswith('D2/') and s.trainable]

    def grads():
        net.substep(4, apply=False)
        out = {}
        for s in specs:
            try:
                out[s.name] = net.get_variable(s.name + '/grad')
            except ea.EdgeGANLibError:   # (never receives one)
                pass
        return out

    plain = grads()
    rng = np.random.RandomState(8)
    T, weight, top = 2.0, 0.7, 5
    u = (2 * rng.standard_normal((4, 14))).astype(np.float32)
    index = np.argsort(-u, axis=1)[:, :top].astype(np.int32)
    logits = np.take_along_axis(u, index, 1)
    index[1, 3:] = -1                              # padding
    net.set_teacher(index, logits, temperature=T, weight=weight)
    got = grads()
    # the oracle
    om = O.OracleModel(parity.oracle_config(cfg), values, dtype=torch.float64)
    p = om._leaf_params()
    inp = O.StepInputs(*[parity.t64(batch[k]) for k in ('images', 'z', 'alpha', 'eps')])
    student = O.classifier(p, inp.images[:, :, cfg.width // 2:, :], om.cfg)
    idx = torch.tensor(index, dtype=torch.int64)
    t = torch.tensor(logits, dtype=torch.float64) / T
    t = torch.where(idx >= 0, t, torch.full_like(t, -math.inf)).log_softmax(1)
    logq = (student / T).log_softmax(1).gather(1, idx.clamp(min=0))
    kl = torch.where(idx >= 0, t.exp() * (t.clamp(min=-1e3) - logq), torch.zeros_like(logq)).sum(1)
    extra = weight * T * T * kl.mean()
    loss = O.forward_graph(p, inp, om.cfg, inp.eps[0], want=['loss_d_ac'])['loss_d_ac'] + extra
    names = [n for n in got]
    want = torch.autograd.grad(loss, [p[n] for n in names], allow_unused=True)
    assert len(names) > 20
    # (slopes of the PReLUs are single cancelling sums: the tolerance that the other tests of them use.  The floor: a bias in front of the min-max
    #  gate (y - min) / (max - min) shifts y, min and max alike where no LeakyReLU lies between signs, so its gradient is zero and 32 bits leave rounding noise
    #  of the gradients' scale, the rule of parity.substep_checks)
    gmax = max(float(w.abs().max()) for w in want)
    _assert([(n, parity.rel_l2(got[n], w.numpy(), 1e-5 * gmax), 5e-2 if 'prelu' in n else 1e-2) for n, w in zip(names, want)])
    assert abs(net.teacher_loss() - float(extra.detach())) <= 1e-4 * abs(float(extra.detach()))
    assert any(not np.array_equal(got[n], plain[n]) for n in names)
    # a whole iteration with it, another teacher for the next batch (more logits), then none: as before
    net.train_step()
    assert np.isfinite(net.teacher_loss())
    net.set_teacher(np.tile(np.arange(14, dtype=np.int32), (4, 1)), u, temperature=1.0, weight=weight)
    net.train_step()
    assert np.isfinite(net.teacher_loss())
    net.set_variables(values)
    net.set_teacher(None)
    with pytest.raises(ea.EdgeGANLibError):
        net.teacher_loss()
    net.set_variables(values)
    again = grads()
    assert all(np.array_equal(again[n], plain[n]) for n in names)
    net.close()


def test_teacher_refusals():
    net = ea.EdgeGAN(ea.Config(batch_size=2), ea.init_variables(ea.Config(batch_size=2), 1))
    i, u = np.zeros((2, 3), np.int32), np.zeros((2, 3), np.float32)
    for bad in (lambda: net.set_teacher(i, u[:, :2]), lambda: net.set_teacher(i[:1], u[:1]), lambda: net.set_teacher(i, u, temperature=0.0),
                lambda: net.set_teacher(i, u, weight=float('nan')), lambda: net.set_teacher(np.zeros((2, 1025), np.int32), np.zeros((2, 1025), np.float32)),
                lambda: net.infer_precision(4)):
        with pytest.raises(ea.EdgeGANLibError):
            bad()
    net.close()
    cfg = ea.Config(batch_size=2, num_classes=0)
    net = ea.EdgeGAN(cfg, ea.init_variables(cfg, 1))
    with pytest.raises(ea.EdgeGANLibError):
        net.set_teacher(i, u)
    net.close()


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_inference_in_8_bits(dtype):
    """Near the unquantised graph, the same bits from every slot and lane schedule, changed variables honoured, and the old bits once it is off."""
    cfg = ea.Config(batch_size=4, compute_dtype=dtype)
    values = ea.init_variables(cfg, 2)
    net = ea.EdgeGAN(cfg, values)
    imgs = np.random.RandomState(3).uniform(-1, 1, size=(4, 64, 128, 3)).astype(np.float32)
    cls = np.array([0, 3, 7, 13], dtype=np.int32)
    full = net.infer(imgs, cls, eps2=[0.4, -1.1])
    net.infer_precision(8)
    q = net.infer(imgs, cls, eps2=[0.4, -1.1])
    for a, b in zip(q, full):
        # an operand is off by under 1/254 of its row's largest value (about 3 spreads): some 0.7 % of a product's spread per layer; outputs are in [-1, 1]
        assert not np.array_equal(a, b) and np.sqrt(np.mean((a - b) ** 2)) < 0.05 * np.sqrt(np.mean(b ** 2)) + 1e-3
    net.infer_upload(imgs, cls, eps2=[0.4, -1.1])
    for runs in (1, 2, 5, 9):
        for _ in range(runs):
            net.infer_run()
        e, i = net.infer_download()
        assert np.array_equal(e, q[0]) and np.array_equal(i, q[1]), runs
    w = values['E/e_resnet_256_2/shortcut/conv2d/w']
    net.set_variable('E/e_resnet_256_2/shortcut/conv2d/w', 3 * w)
    changed = net.infer(imgs, cls, eps2=[0.4, -1.1])
    assert not np.array_equal(changed[0], q[0])
    net.set_variable('E/e_resnet_256_2/shortcut/conv2d/w', w)
    back = net.infer(imgs, cls, eps2=[0.4, -1.1])
    assert np.array_equal(back[0], q[0]) and np.array_equal(back[1], q[1])
    net.upload_batch(**ea.synthetic_batch(cfg, seed=1))
    net.train_step()                                    # (training is not affected, and moves the filters)
    net.infer(imgs, cls, eps2=[0.4, -1.1])
    net.set_variables(values)
    net.infer_precision(0)
    again = net.infer(imgs, cls, eps2=[0.4, -1.1])
    assert np.array_equal(again[0], full[0]) and np.array_equal(again[1], full[1])
    net.close()
