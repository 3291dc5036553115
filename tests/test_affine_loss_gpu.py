"""affine_softmax_cross_entropy, both directions, against the formula in 64 bits.

Tolerances. A logit is within 1e-5 of the logits' RMS (this library's tolerance for contractions) plus 1e-6; called e below.
  loss       three logits' errors (the largest, the label's, the sum's) and 2^-20 of itself
  G          2 e relative, and one rounding to 16 bits (fp16: relative to the largest dloss, 2^-38 of it at least)
  dx, dW     sum |G| |other operand| times G's relative error, 1e-5 of the result's RMS for the product, one rounding
  db         the same without an operand"""
import math

import pytest
import torch

from nnabla_b200 import functions as F

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def data(rows, size, classes, dtype, bias=True, seed=0, ignored=0.2, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    label = torch.randint(0, classes, (rows, 1), generator=g, device="cuda")
    label[torch.rand((rows, 1), generator=g, device="cuda") < ignored] = -1
    return (r(rows, size).to(dtype), (r(size, classes) * scale / math.sqrt(size)).to(dtype), label,
            (0.5 * r(classes)).to(dtype) if bias else None, r(rows, 1))


def reference(x, w, label, bias, dloss):
    x, w = x.double(), w.double()
    logits = x @ w + (bias.double() if bias is not None else 0.0)
    lse = torch.logsumexp(logits, 1, keepdim=True)
    counts, at = label >= 0, label.clamp(min=0)
    loss = torch.where(counts, lse - logits.gather(1, at), 0.0)
    G = (logits - lse).exp()
    G.scatter_add_(1, at, torch.full_like(lse, -1.0))
    G = torch.where(counts, G * dloss.double(), 0.0)
    return logits, lse, loss, G


def rms(t):
    return float(t.pow(2).mean().sqrt())


def check(x, w, label, bias, dloss, base_axis=1):
    dtype = x.dtype
    loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, base_axis, output_stat=True)
    grads = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias, base_axis)
    assert loss.shape == x.shape[:base_axis] + (1,) and stat.shape == x.shape[:base_axis] + (2,)
    assert loss.dtype == stat.dtype == torch.float32
    xf, lab, dl = x.reshape(-1, w.shape[0]), label.reshape(-1, 1).long(), dloss.reshape(-1, 1)
    logits, lse, want, G = reference(xf, w, lab, bias, dl)
    e = 1e-5 * rms(logits) + 1e-6
    err = (loss.double().reshape(-1, 1) - want).abs()
    assert (err <= 3 * e + 2.0 ** -20 * want.abs()).all(), float(err.max())
    s = stat.double().reshape(-1, 2)
    assert ((s[:, :1] + s[:, 1:] - lse).abs() <= 2 * e + 2.0 ** -20 * lse.abs()).all()
    half = torch.finfo(dtype).eps / 2
    relative = 2 * e + (half if dtype != torch.float32 else 2.0 ** -20)
    floor = float(dl.abs().max()) * 2.0 ** -38 if dtype == torch.float16 else 0.0
    dG = G.abs() * relative + floor + (lab >= 0) * dl.double().abs() * 1e-6 * (lab == torch.arange(w.shape[1], device="cuda"))
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    wants = (G @ w.double().t(), xf.double().t() @ G, G.sum(0))
    bounds = (dG @ w.double().abs().t(), xf.double().abs().t() @ dG, dG.sum(0))
    for name, got, ref, b in zip(("dx", "dw", "db"), grads, wants, bounds):
        if got is None:
            assert name == "db" and bias is None
            continue
        assert got.dtype == dtype
        got = got.double().reshape(ref.shape)
        bound = b + half * ref.abs() * 1.01 + 1e-5 * rms(ref) + tiny
        bad = ~((got - ref).abs() <= bound)
        assert not bad.any(), (name, int(bad.sum()), float(((got - ref).abs() / bound).max()))
    return loss, stat, grads


SIZES = [(1, 1, 1), (1, 3, 2), (2, 17, 5), (1, 64, 1000), (3, 100, 33), (8, 256, 4096), (9, 40, 129), (31, 31, 65), (64, 64, 64),
         (65, 128, 257), (128, 72, 999), (129, 520, 512), (200, 777, 1001), (256, 512, 1000), (300, 64, 6007), (7, 2048, 3001),
         (513, 136, 776), (1000, 48, 130)]


@pytest.mark.parametrize("rows,size,classes", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bias", [False, True])
def test_against_the_formula(rows, size, classes, dtype, bias):
    check(*data(rows, size, classes, dtype, bias))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,size,classes", [(2048, 320, 20011), (1500, 1024, 33000), (4, 1024, 70001)])
def test_many_classes(dtype, rows, size, classes):
    check(*data(rows, size, classes, dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_a_long_contraction_and_large_logits(dtype):
    check(*data(70, 8200, 300, dtype))
    check(*data(40, 200, 500, dtype, scale=40.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 6, 200])
def test_rows_that_do_not_count(dtype, rows):
    x, w, label, bias, dloss = data(rows, 128, 513, dtype)
    label[:] = -7
    dloss[0] = math.nan  # (nothing arrives from a row that does not count)
    loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, output_stat=True)
    assert (loss == 0).all()
    for g in F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias):
        assert (g == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 150])
def test_labels_outside_and_rows_that_are_not_finite(dtype, rows):
    x, w, label, bias, dloss = data(rows, 128, 500, dtype, ignored=0.0)
    label[1] = 500
    x[2, 3] = math.inf
    loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, output_stat=True)
    assert torch.isnan(loss[1]) and not torch.isfinite(loss[2])
    keep = [i for i in range(rows) if i not in (1, 2)]
    want = reference(x[keep], w, label[keep], bias, dloss[keep])[2]
    assert ((loss[keep].double() - want).abs() < 1e-4).all()
    dx, dw, db = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias)
    assert torch.isnan(dx[1]).all() and torch.isnan(dx[2]).all() and torch.isnan(dw).any() and torch.isnan(db).any()
    label[1:3] = -1  # the same rows, not counted
    loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, output_stat=True)
    dx, _, db = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias)
    assert torch.isfinite(loss).all() and (dx[1:3] == 0).all() and torch.isfinite(db).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [2, 200])
def test_a_class_ruled_out_by_its_bias(dtype, rows):
    x, w, label, bias, dloss = data(rows, 96, 300, dtype, ignored=0.0)
    bias[10] = -math.inf
    bias[20] = torch.finfo(dtype).min
    label[:] = 5
    _, _, grads = check_finite(x, w, label, bias, dloss)
    assert (grads[1][:, 10] == 0).all() and (grads[2][[10, 20]] == 0).all()
    label[0] = 10
    assert F.affine_softmax_cross_entropy(x, w, label, bias)[0] == math.inf


def check_finite(x, w, label, bias, dloss):
    loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, output_stat=True)
    grads = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias)
    logits, _, want, G = reference(x, w, label, bias, dloss)
    e = 1e-5 * rms(logits[:, 30:]) + 1e-6
    assert ((loss.double() - want).abs() <= 3 * e + 2.0 ** -20 * want.abs()).all()
    dx = G @ w.double().t()
    assert ((grads[0].double() - dx).abs() <= torch.finfo(dtype := x.dtype).eps * (G.abs() @ w.double().abs().t()) + 1e-4).all()
    return loss, stat, grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes", [(5, 700), (150, 3001), (300, 40000)])
def test_accumulation_repeatability_and_partial_propagation(dtype, rows, classes):
    x, w, label, bias, dloss = data(rows, 160, classes, dtype)
    loss, stat, grads = check(x, w, label, bias, dloss)
    again = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    assert torch.equal(F.affine_softmax_cross_entropy(x, w, label, bias), loss)
    held = [torch.ones_like(t) for t in grads]
    F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias, accum=(True,) * 3, grads=held)
    half = torch.finfo(dtype).eps / 2
    for a, b in zip(held, grads):
        assert ((a.double() - 1 - b.double()).abs() <= half * (2 * b.double().abs() + 1.01) + 1e-6 * rms(b.double())).all()
    for flags in [(True, False, False), (False, True, False), (False, False, True)]:
        part = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias, propagate_down=flags)
        for f, a, b in zip(flags, part, grads):
            assert (a is None) if not f else torch.equal(a, b)
    out = torch.empty_like(loss)
    assert F.affine_softmax_cross_entropy(x, w, label, bias, outputs=[out]) is out and torch.equal(out, loss)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [4, 96])
def test_axes_strides_offsets_and_label_types(dtype, rows):
    x, w, label, bias, dloss = data(rows, 120, 333, dtype)
    loss, stat, grads = check(x, w, label, bias, dloss)
    got = F.affine_softmax_cross_entropy(x, w, label.int(), bias, output_stat=True)
    assert torch.equal(got[0], loss) and torch.equal(got[1], stat)
    again = F.affine_softmax_cross_entropy_backward(x, w, label.int(), stat, dloss, bias)
    assert all(torch.equal(a, b) for a, b in zip(again, grads))
    assert torch.equal(F.affine_softmax_cross_entropy(x, w, label[:, 0], bias), loss)
    check(x.reshape(2, rows // 2, 120), w, label.reshape(2, rows // 2, 1), bias, dloss.reshape(2, rows // 2, 1), 2)
    check(x.reshape(rows, 4, 30), w, label, bias, dloss)
    check(x.t().contiguous().t(), w.t().contiguous().t(), label, bias, dloss)
    for t in (x, w, bias):  # off a 16-byte boundary
        base = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")
        off = base[1:].view_as(t).copy_(t)
        check(off if t is x else x, off if t is w else w, label, off if t is bias else bias, dloss)


@pytest.mark.parametrize("dtype", TYPES)
def test_gradients_that_differ_in_size(dtype):
    x, w, label, bias, dloss = data(200, 128, 500, dtype)
    dloss *= torch.logspace(-6, 6, 200, device="cuda")[:, None]
    if dtype == torch.float16:
        dloss *= 1e-3
    check(x, w, label, bias, dloss)
    dloss.zero_()
    loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, output_stat=True)
    for g in F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias):
        assert (g == 0).all()


@pytest.mark.parametrize("rows", [3, 140])
def test_stream_and_graph(rows):
    x, w, label, bias, dloss = data(rows, 256, 2000, torch.bfloat16)

    def step(x, dloss):
        loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, output_stat=True)
        grads = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias)
        return torch.cat([t.float().reshape(-1) for t in (loss,) + tuple(grads)])
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


def test_gradients_against_differences():
    x, w, label, bias, dloss = (t.double() if t.is_floating_point() else t for t in data(3, 6, 9, torch.float32))
    _, _, _, G = reference(x, w, label, bias, dloss)
    f = lambda x, w, b: float((reference(x, w, label, b, dloss)[2] * dloss).sum())
    h = 1e-6
    for i, j in [(0, 0), (1, 4), (2, 5)]:
        e, v = torch.zeros_like(x), torch.zeros_like(w)
        e[i, j], v[j, i] = h, h
        assert abs((f(x + e, w, bias) - f(x - e, w, bias)) / (2 * h) - float((G @ w.t())[i, j])) < 1e-6
        assert abs((f(x, w + v, bias) - f(x, w - v, bias)) / (2 * h) - float((x.t() @ G)[j, i])) < 1e-6


def test_no_rows():
    x, w, label, bias, dloss = data(4, 24, 50, torch.float32)
    x, label, dloss = x[:0], label[:0], dloss[:0]
    loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, output_stat=True)
    assert loss.shape == (0, 1)
    dx, dw, db = F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias)
    assert dx.shape == (0, 24) and (dw == 0).all() and (db == 0).all()
    held = [torch.empty_like(x), torch.ones_like(w), torch.ones_like(bias)]
    F.affine_softmax_cross_entropy_backward(x, w, label, stat, dloss, bias, accum=(True,) * 3, grads=held)
    assert (held[1] == 1).all() and (held[2] == 1).all()


def test_more_rows_than_one_pass_takes():
    """The forward pass takes the rows in slabs (here 16384 at a time: 512 pairs of a maximum and a sum a row)."""
    x, w, label, bias, dloss = data(20000, 16, 32700, torch.bfloat16)
    loss, stat = F.affine_softmax_cross_entropy(x, w, label, bias, output_stat=True)
    for at in (0, 8000, 16000, 19500):
        rows = slice(at, at + 500)
        logits, lse, want, _ = reference(x[rows], w, label[rows], bias, dloss[rows])
        e = 1e-5 * rms(logits) + 1e-6
        assert ((loss[rows].double() - want).abs() <= 3 * e + 2.0 ** -20 * want.abs()).all()
        s = stat[rows].double()
        assert ((s[:, :1] + s[:, 1:] - lse).abs() <= 2 * e + 2.0 ** -20 * lse.abs()).all()


@pytest.mark.parametrize("rows,size,classes", [(9, 200, 3000), (17, 64, 11008), (600, 96, 128), (3000, 40, 70), (2600, 320, 128)])
@pytest.mark.parametrize("dtype", TYPES)
def test_products_with_a_long_axis(rows, size, classes, dtype):
    """Shapes whose gradients have few tiles and a long K."""
    check(*data(rows, size, classes, dtype))
