"""affine_softmax_cross_entropy_backward where one row's gradient says nothing of the others'. Tolerances as in test_affine_loss_gpu."""
import math

import pytest
import torch

from nnabla_b200 import functions as F
from test_affine_loss_gpu import TYPES, check, data, reference, rms

pytestmark = pytest.mark.gpu


def rows_of_dx(x, w, label, bias, dloss, keep):
    """dx of the rows `keep` against the formula of these rows alone: a row of dx depends on nothing else."""
    loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, output_stat=True)
    dx = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias)[0][keep].double()
    logits, _, _, G = reference(x[keep], w, label[keep], bias, dloss[keep])
    half, dl = torch.finfo(x.dtype).eps / 2, dloss[keep].double()
    e = 1e-5 * rms(logits) + 1e-6
    relative = 2 * e + (half if x.dtype != torch.float32 else 2.0 ** -20)
    floor = float(dl.abs().max()) * 2.0 ** -38 if x.dtype == torch.float16 else 0.0
    dG = G.abs() * relative + floor + dl.abs() * 1e-6 * (label[keep] == torch.arange(w.shape[1], device="cuda"))
    want = G @ w.double().t()
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    bound = dG @ w.double().abs().t() + half * want.abs() * 1.01 + 1e-5 * rms(want) + tiny
    bad = ~((dx - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), float(((dx - want).abs() / bound).max()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 40, 300])
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
def test_a_gradient_that_is_not_finite_stays_in_its_row(dtype, rows, what):
    x, w, label, bias, dloss = data(rows, 96, 500, dtype, ignored=0.0)
    dloss = torch.sign(dloss) * 100.0
    dloss[3] = what
    rows_of_dx(x, w, label, bias, dloss, [i for i in range(rows) if i != 3])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [5, 40])
def test_a_row_whose_label_does_not_exist_sets_no_scale(dtype, rows):
    x, w, label, bias, dloss = data(rows, 96, 500, dtype, ignored=0.0)
    label[3], dloss[3] = 500, 1e30
    label[4], dloss[4] = -1, 1e30
    rows_of_dx(x, w, label, bias, dloss, [i for i in range(rows) if i not in (3, 4)])


def test_a_label_without_axes_is_refused():
    x, w, label, bias, dloss = data(1, 24, 50, torch.float32, ignored=0.0)
    loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, output_stat=True)
    with pytest.raises(RuntimeError, match="label must have the shape"):
        F.affine_softmax_cross_entropy(x, w, label[0, 0], bias)
    with pytest.raises(RuntimeError, match="label must have the shape"):
        F.affine_softmax_cross_entropy_backward(x, w, label[0, 0], stat, dloss, bias)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 3, 8])
@pytest.mark.parametrize("size,classes", [(1, 1), (5, 3), (16, 7), (17, 15), (33, 59), (200, 60), (31, 61), (130, 119), (40, 121),
                                          (300, 1001), (700, 16), (900, 33)])
def test_few_rows_with_rows_of_the_weights_that_begin_anywhere(dtype, rows, size, classes):
    """Every distance of W from a 16-byte boundary, with NaN around it, and every distance of its rows from one."""
    x, w, label, bias, dloss = data(rows, size, classes, dtype)
    for off in range(16 // w.element_size()):
        base = torch.full((16 + w.numel() + 16,), math.nan, dtype=dtype, device="cuda")
        at = base[8 + off:8 + off + w.numel()].view_as(w).copy_(w)
        check(x, at, label, bias, dloss)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 7])
@pytest.mark.parametrize("size,classes", [(5, 3), (40, 121), (130, 2048), (300, 4103)])
def test_few_rows_with_a_gradient_buffer_that_begins_anywhere(dtype, rows, size, classes):
    """dW beginning otherwise than W: the same bits, and what lies around it stays."""
    x, w, label, bias, dloss = data(rows, size, classes, dtype)
    loss, stat, want = check(x, w, label, bias, dloss)
    for off in range(16 // w.element_size()):
        base = torch.full((8 + off + w.numel() + 16,), 7.0, dtype=dtype, device="cuda")
        dw = base[8 + off:8 + off + w.numel()].view_as(w)
        for accum in (False, True):
            dw.fill_(1.0)
            got = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias, grads=(None, dw, None),
                                                          accum=(False, accum, False))
            assert got[1] is dw and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
            if accum:
                half = torch.finfo(dtype).eps / 2
                b = want[1].double()
                assert ((dw.double() - 1 - b).abs() <= half * (2 * b.abs() + 1.01) + 1e-6 * rms(b)).all()
            else:
                assert torch.equal(dw, want[1])
            assert (base[:8 + off] == 7).all() and (base[8 + off + w.numel():] == 7).all()
        alone = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias, grads=(None, dw.fill_(1.0), None),
                                                        propagate_down=(False, True, False))
        assert torch.equal(alone[1], want[1])


@pytest.mark.parametrize("rows,size,classes", [(9, 300, 28001), (17, 64, 131074), (64, 1024, 8209), (100, 4100, 2052), (127, 520, 16384),
                                               (128, 65, 140003), (33, 8200, 1025)])
@pytest.mark.parametrize("bias", [False, True])
def test_weights_of_a_large_float32_head_as_they_lie(rows, size, classes, bias):
    """Few rows and a large W, of which no pieces are laid out; the last: classes in two pieces."""
    x, w, label, b, dloss = data(rows, size, classes, torch.float32, bias)
    loss, stat, grads = check(x, w, label, b, dloss)
    again = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, b)
    assert all(g is None and a is None or torch.equal(g, a) for g, a in zip(grads, again))
    assert torch.equal(F.affine_softmax_cross_entropy(x, w, label, b), loss)
    held = [None if g is None else torch.ones_like(g) for g in grads]
    F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, b, accum=(True,) * 3, grads=held)
    for a, g in zip(held, grads):
        if g is not None:
            half, g = torch.finfo(torch.float32).eps / 2, g.double()
            assert ((a.double() - 1 - g).abs() <= half * (2 * g.abs() + 1.01) + 1e-6 * rms(g)).all()
    for flags in [(True, False, False), (False, True, False)]:
        part = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, b, propagate_down=flags)
        assert all((p is None) if not f else torch.equal(p, g) for f, p, g in zip(flags, part, grads))
    base = torch.full((16 + w.numel() + 16,), math.nan, device="cuda")  # off every boundary, with NaN around it
    check(x, base[9:9 + w.numel()].view_as(w).copy_(w), label, b, dloss)


def test_a_large_float32_head_on_a_stream_and_in_graphs():
    x, w, label, bias, dloss = data(40, 512, 16500, torch.float32)

    def step(x, dloss):
        loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, output_stat=True)
        grads = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias)
        return torch.cat([t.reshape(-1) for t in (loss,) + tuple(grads)])
    want = step(x, dloss)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, dloss)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    from nnabla_b200 import graphs
    a, b = graphs.Captured(step, x, dloss), graphs.Captured(step, x, dloss)
    other = (x * 0.5, dloss + 1)
    expected = step(*other)
    assert torch.equal(a(x, dloss), want) and torch.equal(b(*other), expected) and torch.equal(a(*other), expected)
    F.check_device_status()


def test_two_streams_at_once():
    """Heads in pieces, as they lie, and of few rows, each with its bias gradient, side by side: the bits of one after the other."""
    cases = [data(2048, 64, 20011, torch.bfloat16), data(40, 512, 16500, torch.float32), data(5, 300, 4103, torch.float16),
             data(1500, 64, 33000, torch.float32)]

    def step(x, w, label, bias, dloss):
        loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, output_stat=True)
        return (loss,) + tuple(F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias))
    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for turn in range(6):
        for i in range(len(cases)):
            with torch.cuda.stream(streams[(i + turn) % len(streams)]):
                got[i].append(step(*cases[i]))
    torch.cuda.synchronize()
    for i, results in enumerate(got):
        assert all(torch.equal(a, b) for r in results for a, b in zip(r, want[i])), i
    F.check_device_status()
