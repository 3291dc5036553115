"""Temperatures that float32 cannot divide by: 1 / temperature is infinite, and the largest logit's 0 * infinity NaN."""
import ctypes

import pytest


@pytest.mark.parametrize("temperature", [1e-45, 1e-39, 1.17e-38])
def test_a_temperature_below_the_normal_numbers_is_refused(temperature):
    from nnabla_b200 import build
    build.build()
    lib = ctypes.CDLL(build.LIB)
    lib.nb200_last_error.restype = ctypes.c_char_p
    p, i64, t = ctypes.c_void_p(4096), ctypes.c_int64, ctypes.c_float(temperature)  # (never read: refused before)
    assert t.value > 0.0
    assert lib.nb200_top_k_distillation(p, p, p, p, p, i64(2), i64(9), 3, t, 0, 4, None) == 1
    assert "temperature" in lib.nb200_last_error().decode()
    assert lib.nb200_top_k_distillation_backward(p, p, p, p, p, p, i64(2), i64(9), 3, t, 0, 4, 0, None) == 1
    assert "temperature" in lib.nb200_last_error().decode()
