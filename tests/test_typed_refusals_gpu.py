"""Refusals of the normalization and the losses in the Python mirror: types, shapes, devices, buffers that share memory."""
import pytest
import torch

from nnabla_b200 import functions as F

pytestmark = pytest.mark.gpu


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def test_layer_normalization():
    x, g = t(4, 6, 8), t(1, 6, 8)
    for bad, error, text in [((x.double(), None, None), TypeError, "float32 or bfloat16"), ((x, t(6, 7), None), RuntimeError, "shape"),
                             ((x, None, t(8)), RuntimeError, "shape"), ((x, g.cpu(), None), RuntimeError, "CPU"),
                             ((x, g.half(), None), TypeError, "float32"), ((x.bfloat16(), g, g.bfloat16()), TypeError, "one type"),
                             (([1.0], None, None), TypeError, "Tensor")]:
        with pytest.raises(error, match=text):
            F.layer_normalization(*bad)
    for axis, text in [([1], "leading"), ([0, 2], "leading"), ([0, 1, 2], "no axis"), (3, "fit"), ([0, 0], "fit")]:
        with pytest.raises(RuntimeError, match=text):
            F.layer_normalization(x, None, None, axis)
    with pytest.raises(RuntimeError, match="empty row"):
        F.layer_normalization(t(3, 0), None, None)
    for out in (t(4, 6, 7), t(4, 6, 8, dtype=torch.float16), t(4, 8, 6).transpose(1, 2)):
        with pytest.raises(RuntimeError, match="outputs"):
            F.layer_normalization(x, None, None, outputs=[out])
    base = t(4 * 48 + 1)
    with pytest.raises(RuntimeError, match="share memory"):
        F.layer_normalization(base[:-1].view(4, 48), None, None, outputs=[base[1:].view(4, 48)])
    y, mean, var = F.layer_normalization(x, None, g, output_stat=True)
    B = F.layer_normalization_backward
    for args, kw, text in [((x, t(4, 48), g, mean, var), {}, "dy must"), ((x, x, g, mean[:2], var), {}, "one a row"),
                           ((x, x, g, mean, var), dict(accum=(True, False, False)), "buffer"),
                           ((x, x, g, mean, var), dict(grads=(None, t(6, 8), None)), "grads"),
                           ((x, x, g, mean, var), dict(grads=(None, g, None)), "share memory"),
                           ((x, x, g, mean, var), dict(grads=(None, base[:48].view(1, 6, 8), base[1:49].view(1, 6, 8))), "share"),
                           ((x, x, g, mean.cpu(), var), {}, "CPU")]:
        with pytest.raises(RuntimeError, match=text):
            B(*args, **kw)
    with pytest.raises(TypeError, match="dy"):
        B(x, x.half(), g, mean, var)


def test_affine_softmax_cross_entropy():
    x, w, label, b = t(4, 6), t(6, 5), t(4, 1, dtype=torch.int64), t(5)
    L, B = F.affine_softmax_cross_entropy, F.affine_softmax_cross_entropy_backward
    for args, error, text in [((x, w.half(), label), TypeError, "weight"), ((x, w, label.float()), TypeError, "label"),
                              ((x, t(7, 5), label), RuntimeError, "mismatch"), ((x, w, label[:3]), RuntimeError, "label"),
                              ((x, w, label, t(4)), RuntimeError, "bias"), ((x, w, label.cpu()), RuntimeError, "CPU"),
                              ((x, t(6, 5, 2), label), RuntimeError, "matrix"), ((x.double(), w, label), TypeError, "x must"),
                              ((x, t(6, 0), label), RuntimeError, "empty"), ((x, w, label.to(torch.int16)), TypeError, "label")]:
        with pytest.raises(error, match=text):
            L(*args)
    with pytest.raises(RuntimeError, match="Base_axis"):
        L(x, w, label, base_axis=2)
    with pytest.raises(RuntimeError, match="outputs"):
        L(x, w, label, outputs=[t(4)])
    loss, stat = L(x, w, label, b, output_stat=True)
    dl = t(4, 1)
    for args, kw, text in [((x, w, label, stat[:3], dl), {}, "stat"), ((x, w, label, stat, t(3, 1)), {}, "dloss"),
                           ((x, w, label, stat, dl), dict(accum=(False, True, False)), "buffer"),
                           ((x, w, label, stat, dl), dict(grads=(x, None, None)), "share memory"),
                           ((x, w, label, stat, dl), dict(grads=(None, t(5, 6).t(), None)), "contiguous"),
                           ((x, w, label, stat, dl), dict(grads=(None, w, None)), "share memory")]:
        with pytest.raises(RuntimeError, match=text):
            B(*args, **kw)
    with pytest.raises(TypeError, match="dloss"):
        B(x, w, label, stat, dl.half())


def test_top_k_distillation():
    x, index, teacher = t(4, 9), t(4, 3, dtype=torch.int64), t(4, 3)
    D, B = F.top_k_distillation, F.top_k_distillation_backward
    for args, error, text in [((x, index.float(), teacher), TypeError, "index"), ((x, index, teacher.half()), TypeError, "teacher"),
                              ((x, index[:, :2], teacher), RuntimeError, "shape"), ((x, index[:3], teacher[:3]), RuntimeError, "shape"),
                              ((x, index.cpu(), teacher), RuntimeError, "CPU"), ((x.int(), index, teacher), TypeError, "x must"),
                              ((t(4, 0), index, teacher), RuntimeError, "no classes"), ((x, index, teacher, 0.0), RuntimeError, "temper"),
                              ((x, index, teacher, float("nan")), RuntimeError, "temper"),
                              ((x, t(4, 0, dtype=torch.int64), t(4, 0)), RuntimeError, "entries")]:
        with pytest.raises(error, match=text):
            D(*args)
    with pytest.raises(RuntimeError, match="entries"):
        D(t(1, 5000), t(1, 1025, dtype=torch.int64), t(1, 1025))
    loss, stat = D(x, index, teacher, output_stat=True)
    dl = t(4, 1)
    base = t(37)
    for args, kw, text in [((x, index, teacher, stat[:, :1].contiguous(), dl), {}, "stat"), ((x, index, teacher, stat, dl[:2]), {}, "stat"),
                           ((x, index, teacher, stat, dl), dict(accum=True), "buffer"),
                           ((x, index, teacher, stat, dl), dict(dx=t(4, 8)), "dx"),
                           ((base[:36].view(4, 9), index, teacher, stat, dl), dict(dx=base[1:].view(4, 9)), "share memory")]:
        with pytest.raises(RuntimeError, match=text):
            B(*args, **kw)


@pytest.mark.skipif("torch.cuda.device_count() < 2")
def test_another_device():
    x = torch.zeros((4, 6), device="cuda:1")
    with pytest.raises(RuntimeError, match="cuda:0"):
        F.layer_normalization(x, t(1, 6), None)
    y = F.layer_normalization(x + 1, None, None)  # of the tensors', not of the current one
    assert y.device == x.device
