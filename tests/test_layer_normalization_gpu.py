"""LayerNormalization, both directions, against the formula in 64 bits.

Tolerances. eps_t = torch.finfo(type).eps / 2 is the rounding of a result. In fp32 a sum of n values over the threads of a row
has at most log2-like depth plus the values a thread adds by itself, all in all fewer than 64 roundings a term for the sizes
here, so that mean, variance and the two backward means are within 64 * 2^-24 of the sum of the magnitudes; with u of unit
variance the normalized value then is within 128 * 2^-24 * (1 + |mean| / std) of its own size plus 1, and the parameters add
four roundings."""
import math

import pytest
import torch

from nnabla_b200 import functions as F

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    var = ((x - mean) ** 2).mean(1, keepdim=True)
    u = (x - mean) / (var + eps).sqrt()
    y = u * (gamma.double() if gamma is not None else 1.0) + (beta.double() if beta is not None else 0.0)
    return y, mean, var, u


def reference_backward(x, dy, gamma, eps):
    _, mean, var, u = reference(x, None, None, eps)
    dy = dy.double()
    g = dy * (gamma.double() if gamma is not None else 1.0)
    dx = (g - g.mean(1, keepdim=True) - u * (g * u).mean(1, keepdim=True)) / (var + eps).sqrt()
    return dx, dy.sum(0), (dy * u).sum(0), u


def close(got, want, magnitude, roundings):
    """|got - want| within one rounding of the result's type and `roundings` fp32 roundings of `magnitude`."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bound = half * want.abs() * (1 + 1e-6) + roundings * E32 * magnitude * (1 + half) + tiny
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (int(bad.sum()), float(((got.double() - want).abs() / bound).max()))


def data(rows, size, dtype, seed=0, shift=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    return ((r(rows, size) * 2 + shift).to(dtype), r(rows, size).to(dtype), 1 + 0.2 * r(1, size), 0.2 * r(1, size))


SIZES = [(1, 1), (3, 1), (1, 7), (5, 8), (4, 31), (300, 32), (2, 33), (7, 128), (9, 256), (600, 257), (3, 512), (700, 520),
         (2, 1000), (301, 1001), (1, 1024), (320, 1024), (33, 2048), (5, 4097), (310, 4096), (2, 16384), (3, 16400),
         (1, 33000), (2, 70001), (1, 140000), (400, 8200)]


@pytest.mark.parametrize("rows,size", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("param32", [False, True])
def test_forward_and_backward(rows, size, dtype, param32):
    x, dy, gamma, beta = data(rows, size, dtype)
    if not param32:
        gamma, beta = gamma.to(dtype), beta.to(dtype)
    y, mean, var = F.layer_normalization(x, beta, gamma, output_stat=True)
    wy, wm, wv, u = reference(x, gamma, beta, 1e-5)
    assert y.dtype == dtype and mean.shape == (rows, 1) and mean.dtype == torch.float32
    scale = x.double().abs().mean(1, keepdim=True)
    # a single value (or equal ones) has the variance 0 up to the squared rounding of its mean
    std = (wv + 1e-5).sqrt()
    close(mean, wm, scale, 64)
    close(var, wv, wv + 128 * E32 * scale ** 2, 128)
    unit = 1 + u.abs() + (scale + x.double().abs()) / std
    close(y, wy, unit * gamma.double().abs() + beta.double().abs(), 160)
    dx, db, dg = F.layer_normalization_backward(x, dy, gamma, mean, var)
    wdx, wdb, wdg, u = reference_backward(x, dy, gamma, 1e-5)
    g = (dy.double() * gamma.double()).abs()
    close(dx, wdx, (g + g.mean(1, keepdim=True) + unit * (g * unit).mean(1, keepdim=True)) / std, 400)
    assert dx.dtype == dtype and db.dtype == gamma.dtype and db.shape == gamma.shape
    close(db.reshape(-1), wdb, dy.double().abs().sum(0), 64)
    close(dg.reshape(-1), wdg, (dy.double().abs() * unit).sum(0), 256)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [48, 250, 2048, 20001])
def test_without_parameters_and_partial_propagation(dtype, size):
    x, dy, gamma, beta = data(37, size, dtype)
    y, mean, var = F.layer_normalization(x, None, None, output_stat=True)
    assert torch.equal(y, F.layer_normalization(x, torch.zeros_like(beta), torch.ones_like(gamma)))
    full = F.layer_normalization_backward(x, dy, gamma, mean, var)
    for flags in [(True, False, False), (False, True, True), (False, False, True), (True, True, False), (False,) * 3]:
        part = F.layer_normalization_backward(x, dy, gamma, mean, var, propagate_down=flags)
        for f, a, b in zip(flags, part, full):
            assert (a is None) if not f else torch.equal(a, b)
    dx, db, dg = F.layer_normalization_backward(x, dy, None, mean, var)
    assert dg.dtype == torch.float32 and dg.shape == (1, size) and torch.equal(db, full[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [64, 999, 17000])
def test_accumulation_in_place_and_repeatability(dtype, size):
    x, dy, gamma, beta = data(65, size, dtype)
    gamma, beta = gamma.to(dtype), beta.to(dtype)
    y, mean, var = F.layer_normalization(x, beta, gamma, output_stat=True)
    grads = F.layer_normalization_backward(x, dy, gamma, mean, var)
    again = F.layer_normalization_backward(x, dy, gamma, mean, var)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    held = [torch.ones_like(t) for t in grads]
    F.layer_normalization_backward(x, dy, gamma, mean, var, accum=(True,) * 3, grads=held)
    wdx, wdb, wdg, _ = reference_backward(x, dy, gamma, 1e-5)
    for got, want, m in zip(held, (wdx, wdb[None], wdg[None]), (8, 400, 400)):
        close(got, want + 1, torch.full_like(want, float(m)), 400)
    for target in ("dy", "x"):
        a, b = x.clone(), dy.clone()
        out = F.layer_normalization_backward(a, b, gamma, mean, var, grads=(b if target == "dy" else a, None, None))
        assert all(torch.equal(p, q) for p, q in zip(out, grads))
    z = x.clone()
    assert F.layer_normalization(z, beta, gamma, outputs=[z]) is z and torch.equal(z, y)


def test_axes_strides_and_offsets():
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((4, 6, 5, 3), generator=g, device="cuda")
    flat = F.layer_normalization(x.reshape(24, 15), None, None)
    y, mean, var = F.layer_normalization(x, None, None, batch_axis=[0, 1], output_stat=True)
    assert torch.equal(y.reshape(24, 15), flat) and mean.shape == (4, 6, 1, 1)
    assert torch.equal(F.layer_normalization(x, None, None, batch_axis=(1, 0)), y)
    assert torch.equal(F.layer_normalization(x, None, None, batch_axis=[-3, -4]), y)
    # strides of another order, and rows that begin off a 16-byte boundary
    t = torch.randn((64, 40), generator=g, device="cuda").to(torch.bfloat16)
    assert torch.equal(F.layer_normalization(t.t(), None, None), F.layer_normalization(t.t().contiguous(), None, None))
    base = torch.randn(1 + 40 * 64, generator=g, device="cuda")
    off = base[1:].view(40, 64)
    w, m, v, _ = reference(off, None, None, 1e-5)
    close(F.layer_normalization(off, None, None), w, 4 + w.abs(), 200)


def test_rows_of_none_and_values_that_are_not_finite():
    x = torch.empty((0, 16), device="cuda")
    y, mean, var = F.layer_normalization(x, None, None, output_stat=True)
    assert y.shape == (0, 16)
    gamma = torch.ones((1, 16), device="cuda")
    dx, db, dg = F.layer_normalization_backward(x, x, gamma, mean, var)
    assert torch.equal(db, torch.zeros_like(gamma)) and torch.equal(dg, torch.zeros_like(gamma))
    held = torch.full_like(gamma, 3.0)
    F.layer_normalization_backward(x, x, gamma, mean, var, accum=(False, True, False), grads=(None, held, None))
    assert torch.equal(held, torch.full_like(gamma, 3.0))
    x = torch.randn((3, 100), device="cuda")
    x[1, 5] = math.nan
    x[2, 7] = math.inf
    y = F.layer_normalization(x, None, None)
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()
    # values far from zero: the variance is taken from centred values
    x = torch.randn((5, 4096), device="cuda") + 1000.0
    want, _, _, _ = reference(x, None, None, 1e-5)
    close(F.layer_normalization(x, None, None), want, 1 + 1002.0 + want.abs(), 8)


def test_gradients_against_differences():
    torch.manual_seed(0)
    x = torch.randn((3, 50), device="cuda").double()
    dy, gamma = torch.randn((3, 50), device="cuda").double(), torch.randn((1, 50), device="cuda").double()
    dx, _, dg, _ = reference_backward(x, dy, gamma, 1e-5)
    f = lambda a, b: float((reference(a, b, None, 1e-5)[0] * dy).sum())
    for i, j in [(0, 0), (1, 20), (2, 49)]:
        e = torch.zeros_like(x)
        e[i, j] = 1e-6
        assert abs((f(x + e, gamma) - f(x - e, gamma)) / 2e-6 - float(dx[i, j])) < 1e-6
        assert abs((f(x, gamma + e[i]) - f(x, gamma - e[i])) / 2e-6 - float(dg[j])) < 1e-6


def test_stream_and_graph():
    x, dy, gamma, beta = data(200, 777, torch.bfloat16)

    def step(x, dy):
        y, mean, var = F.layer_normalization(x, beta, gamma, output_stat=True)
        return torch.cat([t.float().reshape(-1) for t in (y,) + F.layer_normalization_backward(x, dy, gamma, mean, var)])
    want = step(x, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    from nnabla_b200 import graphs
    captured = graphs.Captured(step, x, dy)
    assert torch.equal(captured(x, dy), want)
    assert torch.equal(captured(dy, x), step(dy, x))
