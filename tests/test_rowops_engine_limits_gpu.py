"""The row operators inside the engine where no other test takes them: 8-bit inference in every arithmetic mode, under every block norm and at other batch sizes; the command
lines with 'layernorm'."""
import os
import subprocess
import sys

import numpy as np
import pytest

import edgegan_amd as ea
from test_rowops_engine_gpu import moved_parameters

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize('flags', [dict(compute_dtype='f32x3'), dict(compute_dtype='f32x3', E_norm='layernorm', G_norm='layernorm'), dict(compute_dtype='bf16', E_norm='layernorm'),
                                   dict(compute_dtype='bf16', E_norm='batch', G_norm='batch'), dict(E_norm=None, G_norm='layernorm'), dict(compute_dtype='bf16', num_classes=0),
                                   dict(compute_dtype='bf16', E_norm=None), dict(height=128, width=256, compute_dtype='bf16')],
                         ids=lambda f: '-'.join(f'{k}={v}' for k, v in f.items()))
def test_8_bit_inference_in_every_mode(flags):
    """Near the unquantised graph for one image, a few and many; every slot gives the same bits; 0 gives the old ones back."""
    cfg = ea.Config(batch_size=2, **flags)
    net = ea.EdgeGAN(cfg, moved_parameters(cfg, 7))
    rng = np.random.RandomState(3)
    for nb in (1, 3, 40):
        imgs = rng.uniform(-1, 1, size=(nb, cfg.height, cfg.width, 3)).astype(np.float32)
        cls = (np.arange(nb) % 14).astype(np.int32) if cfg.num_classes else None
        net.infer_precision(0)
        full = net.infer(imgs, cls, eps2=[0.4, -1.1])
        net.infer_precision(8)
        q = net.infer(imgs, cls, eps2=[0.4, -1.1])
        for a, b in zip(q, full):
            # (the bound of test_inference_in_8_bits; a network without norms in its encoder hands on what the norms would take back)
            rms = np.sqrt(np.mean((a - b) ** 2)) / np.sqrt(np.mean(b ** 2))
            assert np.isfinite(a).all() and not np.array_equal(a, b) and rms < 0.05 + 1e-3, (nb, rms)
        net.infer_upload(imgs, cls, eps2=[0.4, -1.1])
        for runs in (1, 4, 7):
            for _ in range(runs):
                net.infer_run()
            e, i = net.infer_download()
            assert np.array_equal(e, q[0]) and np.array_equal(i, q[1]), (nb, runs)
        net.infer_precision(0)
        again = net.infer(imgs, cls, eps2=[0.4, -1.1])
        assert np.array_equal(again[0], full[0]) and np.array_equal(again[1], full[1]), nb
    net.close()


def test_command_lines_with_layer_norm(tmp_path):
    """python -m edgegan_amd.train with 'layernorm' in every network, and edgegan_amd.test on the checkpoint it wrote; without the flags the checkpoint's
    variables are not the graph's and the load fails."""
    from PIL import Image
    rng = np.random.RandomState(0)
    root = tmp_path / 'data'
    for part, n in (('train', 2), ('test', 1)):
        for c in (0, 5):
            os.makedirs(root / 'class14' / part / str(c))
            for i in range(n):
                Image.fromarray(rng.randint(0, 256, size=(64, 128, 3)).astype(np.uint8)).save(root / 'class14' / part / str(c) / f'{i}.png')
    norms = ['--E_norm=layernorm', '--G_norm=layernorm', '--D_norm=layernorm']

    def run(module, *args):
        return subprocess.run([sys.executable, '-m', f'edgegan_amd.{module}', '--name=ln', f'--dataroot={root}', '--batch_size=2', *args], cwd=tmp_path,
                              env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=100)
    p = run('train', *norms, '--epoch=1', '--save_checkpoint_frequency=3')
    assert p.returncode == 0 and sum(l.startswith('Epoch:') for l in p.stdout.splitlines()) == 2, p.stdout[-2000:] + p.stderr[-2000:]
    p = run('test', *norms)
    assert p.returncode == 0 and 'Load SUCCESS' in p.stdout, p.stdout[-2000:] + p.stderr[-2000:]
    assert len(list((tmp_path / 'outputs' / 'ln' / 'test_output').rglob('*.png'))) == 2
    p = run('test', '--E_norm=instance', '--G_norm=layernorm', '--D_norm=batch')
    assert p.returncode != 0
