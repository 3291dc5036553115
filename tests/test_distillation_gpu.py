"""top_k_distillation, both directions, against the formula in 64 bits.

Tolerances. An exponent (v - maximum) / tau - log sum is within eight fp32 roundings of its terms' magnitudes, which is the
relative error of its exponential; the sum of the exponentials has at most 600 roundings in a thread (a row of 128000 on 512 threads is 250). The
exponential itself is 2^-22.5 relative, the logarithm's result 2^-22 of itself plus 2^-22."""
import math

import pytest
import torch

from nnabla_b200 import functions as F

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def reference(x, index, teacher, tau, dloss):
    x, t = x.double() / tau, teacher.double() / tau
    lse = torch.logsumexp(x, -1, keepdim=True)
    t = t.masked_fill(index < 0, -math.inf)
    some = (t > -math.inf).any(-1, keepdim=True)
    p = torch.where(some, torch.softmax(torch.where(some, t, 0.0), -1), 0.0)
    log_p = torch.where(some, torch.log_softmax(torch.where(some, t, 0.0), -1), 0.0)
    at = index.clamp(min=0)
    terms = torch.where(p > 0, p * (log_p - (x.gather(-1, at) - lse)), 0.0)
    loss = tau * tau * terms.sum(-1, keepdim=True)
    dx = torch.where(some, (x - lse).exp(), 0.0)
    dx = dx.scatter_add(-1, at, -p) * tau * dloss.double()
    dx = torch.where(some, dx, 0.0)
    return loss, lse, dx, p, log_p, x - lse


def check(x, index, teacher, tau, dloss):
    loss, lse = F.top_k_distillation(x, index, teacher, tau, output_stat=True)
    dx = F.top_k_distillation_backward(x, index, teacher, lse, dloss, tau)
    wl, ws, wd, p, log_p, log_q = reference(x, index, teacher, tau, dloss)
    # (terms of the exponents: the student's and the teacher's largest magnitudes)
    big = x.double().abs().nan_to_num(posinf=0).amax(-1, keepdim=True) / tau + ws.abs()
    bt = teacher.double().abs().nan_to_num(posinf=0).amax(-1, keepdim=True) / tau + 8
    relative = E32 * (16 * big + 620)  # of a probability q, and (absolute) of log_sum
    rp = E32 * (16 * bt + 64)
    assert loss.dtype == torch.float32 and loss.shape == x.shape[:-1] + (1,)
    assert lse.shape == x.shape[:-1] + (2,) and (lse[..., :1] == x.float().amax(-1, keepdim=True)).all()
    # (the sum of the pair: the first one's division by tau is the reader's)
    assert ((lse[..., :1].double() / tau + lse[..., 1:] - ws).abs() <= relative).all()
    at = index.clamp(min=0)
    spread = torch.where(p > 0, p * (log_p.abs() + log_q.gather(-1, at).abs()), 0.0).sum(-1, keepdim=True)
    bound = tau * tau * (relative + rp * (1 + 3 * spread))
    assert ((loss.double() - wl).abs() <= bound).all(), float(((loss.double() - wl).abs() / bound).max())
    half, tiny = torch.finfo(x.dtype).eps / 2, torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    psum = torch.zeros_like(wd).scatter_add(-1, at, p)
    bound = half * wd.abs() + ((log_q.exp() * relative + psum * rp) * tau * dloss.double().abs()) * 1.01 + tiny
    assert dx.dtype == x.dtype and dx.shape == x.shape
    assert ((dx.double() - wd).abs() <= bound).all(), float(((dx.double() - wd).abs() / bound).max())
    return loss, lse, dx


def data(rows, classes, best, dtype, seed=0, index_type=torch.int64, kept=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (3 * torch.randn((rows, classes), generator=g, device="cuda")).to(dtype)
    index = torch.rand((rows, classes), generator=g, device="cuda").argsort(-1)[:, :best].contiguous().to(index_type)
    teacher = (3 * torch.randn((rows, best), generator=g, device="cuda")).to(dtype)
    if kept is not None:
        index[torch.arange(best, device="cuda") >= torch.tensor(kept, device="cuda")[:, None]] = -1
    return x, index, teacher, torch.randn((rows, 1), generator=g, device="cuda")


SIZES = [(1, 1, 1), (2, 3, 2), (3, 17, 17), (5, 100, 10), (256, 1000, 10), (7, 1001, 33), (1, 32000, 32), (3, 50257, 64),
         (2, 8192, 1024), (300, 2049, 5), (1, 200001, 300), (9, 8193, 4), (160, 20000, 40)]


@pytest.mark.parametrize("rows,classes,best", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tau", [1.0, 3.0])
def test_against_the_formula(rows, classes, best, dtype, tau):
    check(*data(rows, classes, best, dtype)[:3], tau, data(rows, classes, best, dtype)[3])


@pytest.mark.parametrize("dtype", TYPES)
def test_missing_entries_rows_of_none_and_int32(dtype):
    x, index, teacher, dloss = data(6, 333, 8, dtype, index_type=torch.int32, kept=[8, 1, 0, 3, 0, 7])
    index[3, 0] = -5  # an entry missing at the front
    loss, _, dx = check(x, index.long(), teacher, 2.0, dloss)
    got, lse = F.top_k_distillation(x, index, teacher, 2.0, output_stat=True)
    assert torch.equal(got, loss)
    assert torch.equal(F.top_k_distillation_backward(x, index, teacher, lse, dloss, 2.0), dx)
    for row in (2, 4):
        assert loss[row] == 0 and (dx[row] == 0).all()


@pytest.mark.parametrize("classes", [50, 9001])
def test_a_class_named_more_than_once(classes):
    x, index, teacher, dloss = data(4, classes, 12, torch.float32)
    index[:, 5] = index[:, 0]
    index[:, 11] = index[:, 0]
    index[1, :] = 7
    _, _, dx = check(x, index, teacher, 1.0, dloss)
    lse = F.top_k_distillation(x, index, teacher, output_stat=True)[1]
    assert torch.equal(F.top_k_distillation_backward(x, index, teacher, lse, dloss), dx)


def test_infinities_and_classes_that_do_not_exist():
    x, index, teacher, dloss = data(8, 100, 4, torch.float32)
    dloss.fill_(1.0)
    x[0, index[0, 0]] = -math.inf           # the student rules out what the teacher wants
    teacher[0, 0] = 1.0
    teacher[1, 2] = -math.inf               # the teacher rules out an entry, and so does the student
    x[1, index[1, 2]] = -math.inf
    teacher[2, :] = -math.inf               # a row whose entries are all ruled out: as one without entries
    index[3, 1] = 100                       # no such class
    teacher[4, 1] = math.nan
    x[5, 3] = math.nan
    x[6, :] = -math.inf                     # nothing left: no softmax
    x[7, ::2] = torch.finfo(torch.float32).min
    loss, lse = F.top_k_distillation(x, index, teacher, output_stat=True)
    dx = F.top_k_distillation_backward(x, index, teacher, lse, dloss)
    assert loss[0] == math.inf and torch.isfinite(dx[0]).all() and dx[0, index[0, 0]] < 0
    assert torch.isfinite(loss[1]) and torch.isfinite(dx[1]).all() and dx[1, index[1, 2]] == 0
    assert loss[2] == 0 and (dx[2] == 0).all()
    assert torch.isnan(loss[3]) and torch.isnan(dx[3]).all()
    assert torch.isnan(loss[4]) and torch.isnan(dx[4, index[4]]).all()
    assert torch.isnan(loss[5])
    assert torch.isnan(loss[6])
    check(x[[1, 7]], index[[1, 7]], teacher[[1, 7]], 1.0, dloss[[1, 7]])
    # the type's lowest value everywhere leaves a uniform softmax
    for dtype in TYPES:
        x = torch.full((1, 100), torch.finfo(dtype).min, dtype=dtype, device="cuda")
        loss, stat = F.top_k_distillation(x, index[:1], torch.zeros((1, 4), dtype=dtype, device="cuda"), output_stat=True)
        dx = F.top_k_distillation_backward(x, index[:1], torch.zeros((1, 4), dtype=dtype, device="cuda"), stat, dloss[:1])
        assert abs(float(loss) - math.log(25.0)) < 1e-5
        want = torch.full((100,), 0.01, dtype=torch.float64, device="cuda")
        want[index[0]] -= 0.25
        assert ((dx[0].double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 1e-6).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [1000, 10007])
def test_accumulation_in_place_and_offsets(dtype, classes):
    x, index, teacher, dloss = data(5, classes, 9, dtype)
    loss, lse, dx = check(x, index, teacher, 1.0, dloss)
    held = torch.ones_like(x)
    F.top_k_distillation_backward(x, index, teacher, lse, dloss, accum=True, dx=held)
    want = reference(x, index, teacher, 1.0, dloss)[2] + 1
    assert ((held.double() - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + 1e-4 * (want - 1).abs() + 1e-6).all()
    same = x.clone()
    assert F.top_k_distillation_backward(same, index, teacher, lse, dloss, dx=same) is same and torch.equal(same, dx)
    # x, or dx, off a 16-byte boundary
    base = torch.empty(1 + x.numel(), dtype=dtype, device="cuda")
    off = base[1:].view_as(x)
    F.top_k_distillation_backward(x, index, teacher, lse, dloss, dx=off)
    assert torch.equal(off, dx)
    off.copy_(x)
    check(off, index, teacher, 1.0, dloss)
    assert torch.equal(F.top_k_distillation_backward(off, index, teacher, lse, dloss), dx)


def test_batch_axes_stream_and_graph():
    x, index, teacher, dloss = data(24, 3000, 20, torch.bfloat16)

    def step(x, dloss):
        loss, lse = F.top_k_distillation(x, index.view(4, 6, 20), teacher.view(4, 6, 20), 2.0, output_stat=True)
        return torch.cat([loss.reshape(-1), F.top_k_distillation_backward(
            x, index.view(4, 6, 20), teacher.view(4, 6, 20), lse, dloss, 2.0).float().reshape(-1)])
    x, dloss = x.view(4, 6, 3000), dloss.view(4, 6, 1)
    want = step(x, dloss)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, dloss)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    from nnabla_b200 import graphs
    captured = graphs.Captured(step, x, dloss)
    assert torch.equal(captured(x, dloss), want)
    other = (x * 0.5, dloss + 1)
    assert torch.equal(captured(*other), step(*other))


def test_gradient_against_differences():
    x, index, teacher, dloss = data(2, 40, 5, torch.float32, kept=[5, 3])
    x, teacher = x.double(), teacher.double()
    wd = reference(x, index, teacher, 2.0, dloss)[2]
    f = lambda a: float((reference(a, index, teacher, 2.0, dloss)[0] * dloss).sum())
    for i, j in [(0, int(index[0, 0])), (1, int(index[1, 2])), (1, 39), (0, 0)]:
        e = torch.zeros_like(x)
        e[i, j] = 1e-6
        assert abs((f(x + e) - f(x - e)) / 2e-6 - float(wd[i, j])) < 1e-6


def test_no_rows():
    x = torch.empty((0, 10), device="cuda")
    index = torch.empty((0, 2), dtype=torch.int64, device="cuda")
    loss, lse = F.top_k_distillation(x, index, torch.empty((0, 2), device="cuda"), output_stat=True)
    assert loss.shape == (0, 1)
    assert F.top_k_distillation_backward(x, index, torch.empty((0, 2), device="cuda"), lse, loss).shape == (0, 10)
