"""The end of a network as it is trained: normalization of the features, the head's loss against labels and a teacher, and all
gradients, in one chain; against torch's own differentiation of the formulas in 64 bits.

Tolerances: 1e-4 of the largest gradient for fp32 (this library's contractions are within 1e-5 of their RMS, and the chain has
three of them in a row), and for 16 bits eight roundings of the type along the chain (features, G, dx of the head, dx of the
normalization, each once and relative to the largest value)."""
import math

import pytest
import torch

from nnabla_b200 import functions as F
from nnabla_b200 import parametric_functions as PF
from nnabla_b200 import resnet18

pytestmark = pytest.mark.gpu


def near(got, want, tolerance):
    scale = float(want.abs().max())
    assert float((got.double() - want).abs().max()) <= tolerance * scale, (float((got.double() - want).abs().max()), scale)


def data(rows, size, classes, dtype, best=5):
    g = torch.Generator(device="cuda").manual_seed(rows + size)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    label = torch.randint(0, classes, (rows, 1), generator=g, device="cuda")
    label[::7] = -1
    index = torch.rand((rows, classes), generator=g, device="cuda").argsort(1)[:, :best].contiguous()
    index[::5, best - 2:] = -1
    return (r(rows, size).to(dtype), 1 + 0.1 * r(1, size), 0.1 * r(1, size), (r(size, classes) / math.sqrt(size)).to(dtype),
            (0.1 * r(classes)).to(dtype), label, index, (2 * r(rows, best)).to(dtype))


@pytest.mark.parametrize("rows,size,classes", [(3, 64, 50), (130, 200, 1000), (64, 512, 1003)])
@pytest.mark.parametrize("dtype,teacher", [(torch.float32, False), (torch.float32, True), (torch.bfloat16, False),
                                           (torch.float16, False)])
def test_chain(rows, size, classes, dtype, teacher):
    x, gamma, beta, w, b, label, index, best = data(rows, size, classes, dtype)
    h, mean, var = F.layer_normalization(x, beta, gamma, output_stat=True)
    loss, (dh, dw, db) = resnet18.head_loss(h, w, b, label, (index, best) if teacher else None, temperature=2.0, share=0.3)
    dx, dbeta, dgamma = F.layer_normalization_backward(x, dh, gamma, mean, var)

    leaves = [t.double().requires_grad_() for t in (x, gamma, beta, w, b)]
    X, Gm, Bt, W, B = leaves
    H = (X - X.mean(1, keepdim=True)) / (X.var(1, correction=0, keepdim=True) + 1e-5).sqrt() * Gm + Bt
    logits = H @ W + B
    counts = label >= 0
    each = counts.double() / counts.sum().clamp(min=1)
    ce = torch.where(counts, torch.logsumexp(logits, 1, keepdim=True) - logits.gather(1, label.clamp(min=0)), 0.0)
    total = (ce * each).sum() * (0.7 if teacher else 1.0)
    if teacher:
        t = (best.double() / 2.0).masked_fill(index < 0, -math.inf)
        p = torch.softmax(t, 1)
        log_q = torch.log_softmax(logits / 2.0, 1).gather(1, index.clamp(min=0))
        kl = 4.0 * torch.where(p > 0, p * (torch.log_softmax(t, 1).masked_fill(index < 0, 0.0) - log_q), 0.0)
        total = total + 0.3 * (kl.sum(1, keepdim=True) * each).sum()
    total.backward()
    tolerance = 1e-4 if dtype == torch.float32 else 8 * torch.finfo(dtype).eps / 2
    assert abs(float(loss) - float(total)) <= tolerance * abs(float(total))
    for got, leaf in zip((dx, dgamma, dbeta, dw, db), leaves):
        near(got, leaf.grad, tolerance)
    F.check_device_status()


def test_chain_in_a_graph():
    from nnabla_b200 import graphs
    x, gamma, beta, w, b, label, index, best = data(96, 128, 700, torch.float32)

    def step(x):
        h, mean, var = F.layer_normalization(x, beta, gamma, output_stat=True)
        loss, (dh, dw, db) = resnet18.head_loss(h, w, b, label, (index, best))
        return torch.cat([loss.reshape(1)] + [t.reshape(-1) for t in
                                              (dw, db) + F.layer_normalization_backward(x, dh, gamma, mean, var)])
    want, other = step(x), step(x * 2 + 1)
    captured = graphs.Captured(step, x)
    assert torch.equal(captured(x), want) and torch.equal(captured(x * 2 + 1), other)
    assert torch.equal(step(x), want)


def test_parametric_functions():
    PF.clear_parameters()
    x = torch.randn((12, 4, 10), device="cuda")
    label = torch.randint(0, 33, (12, 1), device="cuda")
    with PF.parameter_scope("net"):
        h = PF.layer_normalization(x)
        loss = PF.affine_softmax_cross_entropy(h, label, 33)
        y = PF.affine(h, 33)
    assert PF.get_parameters()["net/layer_normalization/gamma"].shape == (1, 4, 10)
    want = torch.logsumexp(y.double(), 1, keepdim=True) - y.double().gather(1, label)
    assert ((loss.double() - want).abs() < 1e-5).all()
    y = PF.layer_normalization(x, batch_axis=[0, 1], no_scale=True, no_bias=True)
    assert torch.equal(y, F.layer_normalization(x, None, None, [0, 1]))
    PF.clear_parameters()
