"""Refusals of the normalization's and the losses' entry points that need no GPU: arguments are checked before any CUDA call."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from nnabla_b200 import build
    build.build()
    lib = ctypes.CDLL(build.LIB)
    lib.nb200_last_error.restype = ctypes.c_char_p
    return lib


def i64(v):
    return ctypes.c_int64(v)


P = ctypes.c_void_p(4096)  # never read: every call below is refused before


def refused(lib, rc, text, code=1):
    assert rc == code and text in lib.nb200_last_error().decode(), (rc, lib.nb200_last_error())


def test_layer_normalization(lib):
    f = lambda rows=2, size=8, type=0, param=0, x=P: lib.nb200_layer_normalization(
        x, None, None, P, None, None, i64(rows), i64(size), ctypes.c_float(1e-5), type, param, None)
    refused(lib, f(size=0), "empty row")
    refused(lib, f(size=1 << 31), "2^31")
    refused(lib, f(rows=-1), "rows")
    refused(lib, f(rows=1 << 30), "rows")
    refused(lib, f(type=3, param=3), "type code")
    refused(lib, f(type=0, param=1), "beta and gamma")
    refused(lib, f(type=1, param=2), "beta and gamma")
    refused(lib, f(x=None), "null")
    assert f(rows=0) == 0
    g = lambda dx=P, mean=P: lib.nb200_layer_normalization_backward(
        P, P, None, mean, P, dx, None, None, i64(2), i64(8), ctypes.c_float(1e-5), 0, 0, 0, 0, 0, None)
    refused(lib, g(mean=None), "null")
    assert g(dx=None) == 0


def test_affine_softmax_cross_entropy(lib):
    f = lambda rows=2, size=8, classes=4, type=0, label=8, x=P, stat=P: lib.nb200_affine_softmax_cross_entropy(
        x, P, None, P, P, stat, i64(rows), i64(size), i64(classes), type, label, None)
    refused(lib, f(size=0), "inputs")
    refused(lib, f(classes=0), "classes")
    refused(lib, f(classes=1 << 24), "classes")
    refused(lib, f(rows=1 << 22), "rows")
    refused(lib, f(label=2), "4 or 8")
    refused(lib, f(type=7), "type code")
    refused(lib, f(x=None), "null")
    refused(lib, f(stat=ctypes.c_void_p(4100)), "8-byte")
    assert f(rows=0) == 0
    g = lambda dx=P, dloss=P: lib.nb200_affine_softmax_cross_entropy_backward(
        P, P, None, P, P, dloss, dx, None, None, i64(2), i64(8), i64(4), 0, 8, 0, 0, 0, None)
    refused(lib, g(dloss=None), "null")
    assert g(dx=None) == 0


def test_top_k_distillation(lib):
    f = lambda rows=2, classes=9, best=3, t=1.0, type=0, index=4, x=P: lib.nb200_top_k_distillation(
        x, P, P, P, P, i64(rows), i64(classes), best, ctypes.c_float(t), type, index, None)
    refused(lib, f(classes=0), "classes")
    refused(lib, f(best=0), "entries")
    refused(lib, f(best=1025), "entries")
    for t in (0.0, -1.0, float("inf"), float("nan")):
        refused(lib, f(t=t), "temperature")
    refused(lib, f(index=1), "4 or 8")
    refused(lib, f(type=-1), "type code")
    refused(lib, f(x=None), "null")
    assert f(rows=0) == 0


def test_the_mirror_has_no_cpu_path():
    from nnabla_b200 import functions as F
    x, label = torch.zeros((2, 4)), torch.zeros((2, 1), dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        F.layer_normalization(x, None, None)
    with pytest.raises(RuntimeError, match="no CPU path"):
        F.affine_softmax_cross_entropy(x, torch.zeros((4, 3)), label)
    with pytest.raises(RuntimeError, match="no CPU path"):
        F.top_k_distillation(x, label, x[:, :1])
