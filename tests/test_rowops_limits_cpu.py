"""Refusals and sizes of the row operators at the limits of what they take, on the host (the ordinary ones: test_rowops_cpu)."""
import numpy as np
import pytest

import test_rowops_cpu as R


def test_temperatures_whose_scale_is_infinite_are_refused(built_lib):
    """The kernels multiply by log2(e) / T: it has to be finite, not only 1 / T."""
    for t in (3e-39, 4.2e-39, 1e-45):
        assert R.distill(built_lib, t=t) == 1 and 'temperature' in built_lib.eg_last_error(None).decode(), t
    assert R.distill(built_lib, rows=0, t=5e-39) == 0 and R.distill(built_lib, rows=0, t=3e38) == 0


@pytest.mark.parametrize('dtype', [np.int32, np.int64, np.uint32, np.uint64, np.float32])
def test_teacher_indexes_of_any_width(dtype):
    """An index outside the classes is padding whatever integer type holds it: 2^32 + 3 is not class 3."""
    import edgegan_amd as ea

    class Lib:
        def eg_set_teacher(self, ctx, index, logits, top, temperature, weight):
            self.index = [index[i] for i in range(2 * top)]
            return 0
    net = ea.EdgeGAN.__new__(ea.EdgeGAN)
    net.config, net._ctx, net._lib = ea.Config(batch_size=2), None, Lib()
    rows = [[0, 13, 14, 2 ** 31 - 1], [3, 100, 5, 1]] if dtype in (np.int32, np.float32) else [[0, 13, 14, 2 ** 32 - 1], [3, 100, 5, 1]]
    index = np.array(rows, dtype=dtype)
    want = [0, 13, None, None, 3, None, 5, 1]
    if dtype in (np.int64, np.uint64):
        index[0, 2], index[1, 1] = 2 ** 32 + 3, 2 ** 40 + 13
    if dtype in (np.int32, np.int64):
        index[1, 3], want[7] = -2, None
    net.set_teacher(index, np.zeros((2, 4), np.float32))
    got = net._lib.index
    net._ctx = None
    assert [i if 0 <= i < 14 else None for i in got] == want


def test_numbers_past_every_float_are_refused():
    from edgegan_amd import EdgeGANLibError, ops
    assert ops._number(3, 'eps') == 3.0 and ops._number(np.float64(2.5), 'eps') == 2.5
    for bad in (10 ** 400, -10 ** 4400, '1', None, np.zeros(1)):
        with pytest.raises(EdgeGANLibError):
            ops._number(bad, 'eps')


def test_gradient_workspace_is_what_the_kernels_write(built_lib):
    """[blocks][2][cols] of f32: 512 blocks where a row has a block or four waves, 1,024 where a wave or less, 64 groups of rows where it is too long for registers; never more
    blocks than the rows give work to."""
    size = built_lib.eg_layer_norm_workspace
    for rows, cols, blocks in ((65536, 128, 1024), (16384, 4096, 512), (8192, 32768, 64), (100, 32768, 25), (300, 4096, 300), (129, 32, 5), (1 << 40, 1000, 1024), (5000, 8, 157)):
        assert size(rows, cols) == blocks * 2 * cols * 4, (rows, cols, size(rows, cols) / (8 * cols))
    for rows in (3, 17, 129, 700, 5000, 100000):
        for cols in (1, 7, 8, 33, 64, 65, 128, 200, 256, 500, 1000, 1024, 1025, 2048, 3000, 4096, 8192, 8193, 12000, 16384, 16385, 70000):
            assert 0 <= size(rows, cols) <= min(rows, 1024) * 8 * cols, (rows, cols)
