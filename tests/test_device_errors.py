"""The device error words: each kernel file's is reported and cleared."""
import ctypes

import pytest

from capi_util import lib


def _flags(clear):
    f = ctypes.c_uint(77)
    assert lib().tpo_device_error_flags(ctypes.byref(f), clear) == 0
    return f.value


def test_units_are_checked():
    assert lib().tpo_device_error_raise(-1, 1) == 1 and lib().tpo_device_error_raise(1000, 1) == 1


@pytest.mark.gpu
def test_every_unit_is_reported_and_cleared():
    import torch

    torch.empty(1, device="cuda")
    assert _flags(1) == 0
    units = 0
    while lib().tpo_device_error_raise(units, 1 << units) == 0:
        units += 1
    # chamfer, fps, knn, and the three attention files
    assert units == 6 and _flags(0) == (1 << units) - 1 and _flags(1) == (1 << units) - 1 and _flags(0) == 0


@pytest.mark.gpu
def test_kernels_and_the_report_share_their_words():
    # a flag that a kernel raises joins one that the host raised in the same file's word
    import torch

    import torch_point_ops_b200 as tpo

    q = torch.randn(20, 2, 64, device="cuda", dtype=torch.bfloat16)
    tpo.packed_attention(q, q, q, torch.tensor([0, 40], device="cuda"))
    assert _flags(1) == 4
    assert _flags(0) == 0
