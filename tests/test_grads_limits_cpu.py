"""The limit of a clip is an f32 number on the device."""
import ctypes

import numpy as np
import pytest

import tikun_b200
from tikun_b200 import grads


@pytest.mark.parametrize("limit", [1e-50, 7e-46, np.float64(1e-300), 5e-324])
def test_a_limit_that_is_zero_as_f32_is_refused(limit):
    """Zero stands for no limit there, so nothing would be clipped."""
    assert limit > 0 and ctypes.c_float(limit).value == 0.0
    for call in (tikun_b200.clip_scale, tikun_b200.clip_grad_norm_):
        with pytest.raises(ValueError, match="max_norm is positive"):
            call([], limit)


def test_limits_in_range_are_rounded_to_f32():
    assert grads._positive(1e-45) == 2.0 ** -149
    assert grads._positive(0.1) == float(np.float32(0.1))
    assert grads._positive(np.float32(3.0)) == 3.0
    assert grads._positive(float("inf")) == float("inf")
    for bad in (0, -1.0, float("nan"), float("-inf")):
        with pytest.raises(ValueError, match="max_norm is positive"):
            grads._positive(bad)
