"""One data-parallel rank of tests/test_rowops_dp_gpu.py (run as a subprocess): 'layernorm' in every network and a teacher of the classifier, its own shard of the batch and
of the teacher's logits; then one sub-step or two iterations.  Every variable and RMSProp slot goes to <out>/rank<r>.npz.

usage: dp_rowops_worker.py <rank> <world> <out_dir> <mode>      mode: substep1 | substep4 | iterations"""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

import numpy as np

import edgegan_amd as ea
from edgegan_amd import rendezvous

SHARD, TEMPERATURE, WEIGHT = 2, 2.0, 0.7


def config(batch=SHARD):
    return ea.Config(batch_size=batch, E_norm='layernorm', G_norm='layernorm', D_norm='layernorm')


def values():
    """Initial values with every norm's scale and shift moved off 1 and 0."""
    v = ea.init_variables(config(), 0)
    rng = np.random.RandomState(1)
    for n in v:
        if n.endswith('LayerNorm/gamma'):
            v[n] = (1.0 + 0.2 * rng.standard_normal(v[n].shape)).astype(np.float32)
        elif n.endswith('LayerNorm/beta'):
            v[n] = (0.1 * rng.standard_normal(v[n].shape)).astype(np.float32)
    return v


def shard(rank):
    return ea.synthetic_batch(config(), seed=4321, rank=rank)


def teacher(rank):
    """index, logits [SHARD, 5]; a padded entry in each shard."""
    u = (2 * np.random.RandomState(100 + rank).standard_normal((SHARD, 14))).astype(np.float32)
    index = np.argsort(-u, axis=1)[:, :5].astype(np.int32)
    logits = np.take_along_axis(u, index, 1)
    index[rank % SHARD, 4] = -1
    return index, logits


def main():
    rank, world, out, mode = int(sys.argv[1]), int(sys.argv[2]), sys.argv[3], sys.argv[4]
    net = ea.EdgeGAN(config(), values())
    rendezvous.init_data_parallel(net, rank, world)
    net.upload_batch(**shard(rank))
    net.set_teacher(*teacher(rank), temperature=TEMPERATURE, weight=WEIGHT)
    if mode == 'iterations':
        net.train_step()
        net.train_step()
    else:
        net.substep(int(mode[len('substep'):]), apply=True)
    net.sync()
    net.comm_barrier()
    result = net.get_variables(slots=True)
    if mode != 'substep1':
        result['teacher_loss'] = np.float32(net.teacher_loss())
        assert np.isfinite(result['teacher_loss'])
    np.savez(os.path.join(out, f'rank{rank}.npz'), **result)
    net.close()


if __name__ == '__main__':
    main()
