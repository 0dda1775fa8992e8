"""Refusals and sizes of the row operators at the limits of what they take, on the host (the ordinary ones: test_rowops_cpu)."""
import test_rowops_cpu as R


def test_temperatures_whose_scale_is_infinite_are_refused(built_lib):
    """The kernels multiply by log2(e) / T: it has to be finite, not only 1 / T."""
    for t in (3e-39, 4.2e-39, 1e-45):
        assert R.distill(built_lib, t=t) == 1 and 'temperature' in built_lib.eg_last_error(None).decode(), t
    assert R.distill(built_lib, rows=0, t=5e-39) == 0 and R.distill(built_lib, rows=0, t=3e38) == 0
