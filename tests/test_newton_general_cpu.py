"""Refusals of the Newton-Schulz entry that need no GPU."""

import ctypes

import pytest

from ozaki_triton_b200 import _lib


def call(schedule, m=512, n=512):
    flat = [v for row in schedule for v in row]
    p = ctypes.c_void_p(256)      # never dereferenced: validation fails first
    return _lib.load().oz_orthogonalize(p, _lib.OZ_F32, 1, m, n, m * n, n, 1, len(schedule),
                                        (ctypes.c_double * len(flat))(*flat), 1e-7, 2, p, p, 1 << 40, None)


@pytest.mark.parametrize("schedule,step", [
    ([(4.0, -6.0, 3.0)] * 5, 4),                      # singular values grow to 3300 in three steps
    ([(20.0, 0.0, 0.0)] * 2, 2),
    ([(1.0, 0.0, 1e300)] * 2, 1),                     # P = c S S past any scale
    ([(1e200, 1e200, 1e200)] * 3, 1),
])
def test_schedules_whose_matrices_leave_the_slices_are_refused(schedule, step):
    n0 = _lib.load().oz_launch_count()
    assert call(schedule) == _lib.OZ_ERR_UNSUPPORTED
    assert f"before step {step} of {len(schedule)}" in _lib.load().oz_last_error().decode()
    assert _lib.load().oz_launch_count() == n0
