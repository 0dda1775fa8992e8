"""'layernorm' block norms and the classifier's teacher under data parallelism, two ranks on the one device over the loop-back collective (see test_dp_gpu): a
rank's gradients depend on its own samples alone, so their mean is the whole batch's."""
import os
import subprocess
import sys

import numpy as np
import pytest

import dp_rowops_worker as W
import edgegan_amd as ea
from test_dp_gpu import _env, _replicated, shim  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run_ranks(shim, tmp, mode, key, **extra):
    out = tmp / key
    out.mkdir()
    procs = [subprocess.Popen([sys.executable, os.path.join(ROOT, 'tests', 'dp_rowops_worker.py'), str(r), '2', str(out), mode], env=_env(shim, tmp, key, **extra),
                              stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True) for r in range(2)]
    logs = [p.communicate(timeout=100)[0] for p in procs]
    for r, p in enumerate(procs):
        assert p.returncode == 0, f'rank {r} failed:\n{logs[r][-3000:]}'
    return [dict(np.load(out / f'rank{r}.npz')) for r in range(2)]


def gradients(net, batch, teacher, k, names):
    net.upload_batch(**batch)
    net.set_teacher(*teacher, temperature=W.TEMPERATURE, weight=W.WEIGHT)
    net.substep(k, apply=False)
    out = {}
    for n in names:
        try:
            out[n] = net.get_variable(n + '/grad').astype(np.float64)
        except ea.EdgeGANLibError:   # (never receives one)
            pass
    return out


@pytest.mark.parametrize('k,group', [(1, 'D/'), (4, 'D2/')])
def test_two_ranks_average_their_shards(shim, tmp_path, k, group):
    """Sub-step 1 (the joint discriminator's layer norms, their tangents and the reverse of them) and sub-step 4 (the teacher): both replicas have RMSProp's update for the mean
    of the shards' gradients."""
    ranks = run_ranks(shim, tmp_path, f'substep{k}', f's{k}')
    for n in filter(_replicated, ranks[0]):
        if n != 'teacher_loss':
            assert np.array_equal(ranks[0][n], ranks[1][n]), f'replicas differ in {n}'
    cfg, values = W.config(), W.values()
    net = ea.EdgeGAN(cfg, values)
    names = [s.name for s in net.specs if s.trainable and s.name.startswith(group)]
    shards = [gradients(net, W.shard(r), W.teacher(r), k, names) for r in range(2)]
    losses = [float(net.teacher_loss())] if k == 4 else []
    net.close()
    names = list(shards[0])
    assert len(names) > 8 and (k == 4 or any('LayerNorm/gamma' in n for n in names))
    for n in names:
        g = 0.5 * (shards[0][n] + shards[1][n])
        ms = 1.0 + (g * g - 1.0) * 0.1                        # (the slot starts at 1, decay 0.9)
        step = cfg.learning_rate * g / np.sqrt(ms + 1e-10)
        got = values[n].astype(np.float64).reshape(g.shape) - ranks[0][n].astype(np.float64).reshape(g.shape)
        # a weight is rounded at 2^-24 of its size
        assert np.abs(got - step).max() <= 2e-4 * np.abs(step).max() + 2.0 ** -23 * np.abs(values[n]).max(), n
        np.testing.assert_allclose(ranks[0][n + '/RMSProp'].reshape(g.shape), ms, rtol=2e-6, atol=0)
    assert any(np.abs(shards[0][n] - shards[1][n]).max() > 1e-3 * np.abs(shards[0][n]).max() for n in names), 'the shards must differ for this test to mean anything'
    if k == 4:
        assert abs(losses[0] - ranks[1]['teacher_loss']) <= 1e-5 * abs(losses[0])
        # ... which is the gradient of one process with the whole batch
        net = ea.EdgeGAN(W.config(4), values)
        batch = [W.shard(r) for r in range(2)]
        axis = {n: [i for i in range(v.ndim) if v.shape[i] == W.SHARD][0] for n, v in batch[0].items() if n != 'eps'}
        whole = {n: np.concatenate([b[n] for b in batch], axis[n]) if n in axis else batch[0][n] for n in batch[0]}
        t = [np.concatenate(a) for a in zip(*(W.teacher(r) for r in range(2)))]
        one = gradients(net, whole, t, 4, names)
        assert abs(net.teacher_loss() - 0.5 * (ranks[0]['teacher_loss'] + ranks[1]['teacher_loss'])) <= 1e-5 * abs(net.teacher_loss())
        net.close()
        gmax = max(np.abs(g).max() for g in one.values())
        for n in names:   # (the tolerances of the sub-steps against the oracle; where all terms cancel, noise of the largest gradient's size)
            g = 0.5 * (shards[0][n] + shards[1][n])
            err = np.linalg.norm(one[n] - g) / (np.linalg.norm(g) + 1e-5 * gmax * np.sqrt(g.size))
            assert err <= (5e-2 if 'prelu' in n else 1e-2), (n, err)


def test_two_rank_iterations(shim, tmp_path):
    """Two iterations: both replicas identical, and the concurrent lanes give the bits of one stream."""
    lanes = run_ranks(shim, tmp_path, 'iterations', 'lanes')
    serial = run_ranks(shim, tmp_path, 'iterations', 'serial', EG_LANES='0')
    for n in lanes[0]:
        if _replicated(n) and n != 'teacher_loss':
            assert np.array_equal(lanes[0][n], lanes[1][n]), f'replicas differ in {n}'
        assert np.array_equal(lanes[0][n], serial[0][n]) and np.isfinite(lanes[0][n]).all(), n
    moved = [n for n, v in W.values().items() if 'LayerNorm' in n and not np.array_equal(lanes[0][n].reshape(-1), v.reshape(-1))]
    assert len(moved) > 30, len(moved)
