"""Addresses that the optimizer calls of the C ABI refuse: decided before anything is launched."""
import ctypes

import pytest

from sv3d import _lib as L
from test_train_ops_cpu import INVALID, SOME, tensor


@pytest.mark.parametrize("off", [1, 2, 3])
def test_step_counts_off_their_alignment(off):
    p = L.AdamWParams(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)
    arr = (L.AdamWTensor * 2)(tensor(), tensor(step=SOME + off))
    assert L.lib().sv3d_adamw_step(ctypes.byref(p), arr, 2, SOME, 1 << 16, None) == INVALID
    arr[1].numel = 0            # the count of an empty tensor is taken forward too
    assert L.lib().sv3d_adamw_step(ctypes.byref(p), arr, 2, SOME, 1 << 16, None) == INVALID


@pytest.mark.parametrize("name, off", [("lr_device", 2), ("grad_scale", 1), ("found_inf", 3), ("total_norm", 2), ("square_sums", 4)])
def test_scalars_off_their_alignment(name, off):
    p = L.AdamWParams(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, max_norm=1.0, square_sums=SOME, num_square_sums=4)
    setattr(p, name, SOME + off)
    assert L.lib().sv3d_adamw_step(ctypes.byref(p), (L.AdamWTensor * 1)(tensor()), 1, SOME, 1 << 16, None) == INVALID
