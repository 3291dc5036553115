"""Operators at the end of a network that is trained, and the work that their users have them do.

Three operators, alone (forward) or with their gradients (train):

  layer_normalization  y = (x - mean) / sqrt(variance + eps) * gamma + beta over the features of each row
  cross_entropy        the loss of an affine layer's classes, -log softmax(x . weight + bias)[label], without its logits
  distillation         temperature^2 * KL(teacher || student), where of the teacher its best K classes are known

`run` computes them from elementary torch operations in 32 bits, rounded once at the end, or, where `own` is true, calls
nnabla_b200.functions. All data is synthetic and made from the seed.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # serving: the features of one token
        dict(name="norm_1x1024_f32", op="layer_normalization", train=False, type="f32", params="f32", rows=1, size=1024),
        # inference on a batch of long sequences
        dict(name="norm_16384x4096_bf16", op="layer_normalization", train=False, type="bf16", params="bf16", rows=16384,
             size=4096),
        # training in bf16 with the parameters kept in fp32
        dict(name="norm_train_8192x2048_bf16", op="layer_normalization", train=True, type="bf16", params="f32", rows=8192,
             size=2048),
        # training in fp32; rows and features of no round size
        dict(name="norm_train_3001x1001_f32", op="layer_normalization", train=True, type="f32", params="f32", rows=3001,
             size=1001),
        # scoring one token: a single row against all classes
        dict(name="loss_1x2048x32000_bf16", op="cross_entropy", train=False, type="bf16", rows=1, size=2048, classes=32000,
             bias=False, ignored=False),
        # perplexity of a long text
        dict(name="loss_4096x1024x50257_f16", op="cross_entropy", train=False, type="f16", rows=4096, size=1024,
             classes=50257, bias=False, ignored=False),
        # the head of the ResNet-18 at its training batch
        dict(name="loss_train_256x512x1000_f32", op="cross_entropy", train=True, type="f32", rows=256, size=512, classes=1000,
             bias=True, ignored=False),
        # a mid-sized head in fp32 with padded rows; no size is round
        dict(name="loss_train_1000x777x10007_f32", op="cross_entropy", train=True, type="f32", rows=1000, size=777,
             classes=10007, bias=True, ignored=True),
        # a large head in bf16, a batch of sequences with padding
        dict(name="loss_train_8192x2048x128000_bf16", op="cross_entropy", train=True, type="bf16", rows=8192, size=2048,
             classes=128000, bias=False, ignored=True),
        # one token against its teacher
        dict(name="distill_1x32000_k32_f16", op="distillation", train=False, type="f16", rows=1, classes=32000, best=32,
             padded=False, temperature=1.0),
        # the ResNet-18's classes against a teacher's ten best
        dict(name="distill_train_256x1000_k10_f32", op="distillation", train=True, type="f32", rows=256, classes=1000, best=10,
             padded=False, temperature=4.0),
        # a long batch over a large vocabulary; some rows have fewer entries, some none
        dict(name="distill_train_4096x128000_k64_bf16", op="distillation", train=True, type="bf16", rows=4096, classes=128000,
             best=64, padded=True, temperature=2.0),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["layer_normalization", "cross_entropy", "distillation"])
    train, kind = rng.random() < 0.6, rng.choice(["f32", "bf16", "f16"])
    if op == "layer_normalization":
        size = _spread(rng, 16, 16384)
        rows = _spread(rng, 1, min(32768, (1 << 26) // size))
        return dict(op=op, train=train, type=kind, params=rng.choice([kind, "f32"]), rows=rows, size=size)
    classes = _spread(rng, 100, 131072)
    if rng.random() < 0.5:
        classes = max(128, classes // 128 * 128)
    if op == "distillation":
        return dict(op=op, train=train, type=kind, rows=_spread(rng, 1, min(16384, (1 << 29) // classes)), classes=classes,
                    best=_spread(rng, 1, min(256, classes)), padded=rng.random() < 0.5,
                    temperature=rng.choice([0.5, 1.0, 2.0, 4.0]))
    size = _spread(rng, 16, 4096)
    if rng.random() < 0.5:
        size = max(64, size // 64 * 64)
    # no more work, and no larger logits of the plain form, than the largest listed case has
    rows = _spread(rng, 1, min(8192, (8192 * 2048 * 128000) // (6 * size * classes) + 1, (1 << 30) // classes))
    return dict(op=op, train=train, type=kind, rows=rows, size=size, classes=classes, bias=rng.random() < 0.5,
                ignored=rng.random() < 0.5)


def _loss_scale(case):
    """Training in f16 scales its loss, so that small gradients stay in the type's range."""
    return 1024.0 if case["type"] == "f16" else 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, rows = TYPES[case["type"]], case["rows"]

    def normal(*shape, scale=1.0, shift=0.0, type=kind):
        return torch.randn(shape, generator=g, device="cuda").mul_(scale).add_(shift).to(type)

    if case["op"] == "layer_normalization":
        size, params = case["size"], TYPES[case["params"]]
        # activations of a residual stream: a mean of their own per feature
        x = (torch.randn((rows, size), generator=g, device="cuda").mul_(2.0).add_(normal(1, size, type=torch.float32))).to(kind)
        state = dict(case=case, x=x, gamma=normal(1, size, scale=0.1, shift=1.0, type=params),
                     beta=normal(1, size, scale=0.1, type=params))
        if case["train"]:
            state["dy"] = normal(rows, size)
        return state
    if case["op"] == "cross_entropy":
        size, classes = case["size"], case["classes"]
        state = dict(case=case, x=normal(rows, size), weight=normal(size, classes, scale=2.0 / math.sqrt(size)),
                     bias=normal(classes, scale=0.5) if case["bias"] else None)
        label = torch.randint(0, classes, (rows, 1), generator=g, device="cuda")
        if case["ignored"]:  # padding behind the sequences
            label[torch.rand((rows, 1), generator=g, device="cuda") < 0.1] = -1
        state["label"] = label
        if case["train"]:  # of the mean over the rows that count
            count = (label >= 0).sum().clamp(min=1)
            state["dloss"] = torch.full((rows, 1), _loss_scale(case), device="cuda") / count
        return state
    classes, best = case["classes"], case["best"]
    state = dict(case=case, x=normal(rows, classes, scale=3.0))
    # distinct classes, best first; the teacher's logits fall off from the first to the last
    steps = torch.rand((rows, best), generator=g, device="cuda", dtype=torch.float64)
    index = ((torch.arange(best, device="cuda") + steps) * (classes / best)).long().clamp_(max=classes - 1)
    order = torch.rand((rows, best), generator=g, device="cuda").argsort(1)
    index = index.gather(1, order)
    teacher = 8.0 - 8.0 * torch.rand((rows, best), generator=g, device="cuda").sort(1)[0]
    if case["padded"]:
        kept = torch.randint(0, best + 1, (rows, 1), generator=g, device="cuda")
        index = torch.where(torch.arange(best, device="cuda") < kept, index, -1)
    state["index"], state["teacher"] = index, teacher.to(kind)
    if case["train"]:
        state["dloss"] = torch.full((rows, 1), _loss_scale(case) / rows, device="cuda")
    return state


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _layer_normalization(s):
    x, gamma = s["x"].float(), s["gamma"].float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    variance = (centred * centred).mean(1, keepdim=True)
    r = 1.0 / torch.sqrt(variance + EPS)
    unit = centred * r
    y = (unit * gamma + s["beta"].float()).to(s["x"].dtype)
    if not s["case"]["train"]:
        return y
    dy = s["dy"].float()
    g = dy * gamma
    dx = r * (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True))
    return (y, dx.to(s["x"].dtype), dy.sum(0, keepdim=True).to(s["beta"].dtype),
            (dy * unit).sum(0, keepdim=True).to(s["gamma"].dtype))


def _cross_entropy(s):
    x, w, label = s["x"].float(), s["weight"].float(), s["label"]
    logits = x @ w
    if s["bias"] is not None:
        logits += s["bias"].float()
    top = logits.amax(1, keepdim=True)
    log_sum = top + torch.log(torch.exp(logits - top).sum(1, keepdim=True))
    counts = label >= 0
    at = label.clamp(min=0)
    loss = torch.where(counts, log_sum - logits.gather(1, at), 0.0)
    if not s["case"]["train"]:
        return loss
    factor = torch.where(counts, s["dloss"], 0.0)
    grad = logits.sub_(log_sum).exp_().mul_(factor)
    grad.scatter_add_(1, at, -factor)
    kind = s["x"].dtype
    db = grad.sum(0).to(kind) if s["bias"] is not None else None
    return loss, (grad @ w.t()).to(kind), (x.t() @ grad).to(kind), db


def _distillation(s):
    x, t = s["x"].float(), s["case"]["temperature"]
    known = s["index"] >= 0
    at = s["index"].clamp(min=0)
    x = x / t
    top = x.amax(1, keepdim=True)
    log_sum = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    teacher = torch.where(known, s["teacher"].float() / t, -math.inf)
    best = teacher.amax(1, keepdim=True)
    some = best > -math.inf  # rows with an entry
    shifted = torch.where(some, teacher - torch.where(some, best, 0.0), -math.inf)
    p = torch.exp(shifted)
    total = p.sum(1, keepdim=True)
    log_p = shifted - torch.log(torch.where(some, total, 1.0))
    p = torch.where(some, p / torch.where(some, total, 1.0), 0.0)
    log_q = x.gather(1, at) - log_sum
    loss = t * t * torch.where(p > 0, p * (log_p - log_q), 0.0).sum(1, keepdim=True)
    if not s["case"]["train"]:
        return loss
    factor = t * s["dloss"]
    grad = x.sub_(log_sum).exp_().mul_(torch.where(some, factor, 0.0))
    grad.scatter_add_(1, at, -p * factor)
    return loss, grad.to(s["x"].dtype)


# ---- the framework's calls ---------------------------------------------------------------------------------------------

def _own(s):
    from nnabla_b200 import functions as F
    case = s["case"]
    if case["op"] == "layer_normalization":
        if not case["train"]:
            return F.layer_normalization(s["x"], s["beta"], s["gamma"], eps=EPS)
        y, mean, variance = F.layer_normalization(s["x"], s["beta"], s["gamma"], eps=EPS, output_stat=True)
        return (y,) + tuple(F.layer_normalization_backward(s["x"], s["dy"], s["gamma"], mean, variance, eps=EPS))
    if case["op"] == "cross_entropy":
        if not case["train"]:
            return F.affine_softmax_cross_entropy(s["x"], s["weight"], s["label"], s["bias"])
        loss, stat = F.affine_softmax_cross_entropy(s["x"], s["weight"], s["label"], s["bias"], output_stat=True)
        return (loss,) + tuple(F.affine_softmax_cross_entropy_backward(s["x"], s["weight"], s["label"], stat, s["dloss"],
                                                                       s["bias"]))
    if not case["train"]:
        return F.top_k_distillation(s["x"], s["index"], s["teacher"], case["temperature"])
    loss, stat = F.top_k_distillation(s["x"], s["index"], s["teacher"], case["temperature"], output_stat=True)
    return loss, F.top_k_distillation_backward(s["x"], s["index"], s["teacher"], stat, s["dloss"], case["temperature"])


def run(state):
    if own:
        return _own(state)
    return {"layer_normalization": _layer_normalization, "cross_entropy": _cross_entropy,
            "distillation": _distillation}[state["case"]["op"]](state)


def work(case):
    size_of = {"f32": 4, "bf16": 2, "f16": 2}
    e, rows = size_of[case["type"]], case["rows"]
    if case["op"] == "layer_normalization":
        n, params = rows * case["size"], case["size"] * size_of[case["params"]]
        # x, y (and dy, dx); gamma, beta (and their gradients)
        return dict(bytes=(4 if case["train"] else 2) * (n * e + params), flops=(24 if case["train"] else 8) * n)
    if case["op"] == "cross_entropy":
        size, classes = case["size"], case["classes"]
        operands = (rows * size + size * classes + (classes if case["bias"] else 0)) * e
        # the products: the logits, and for training dx and dW
        return dict(bytes=(2 if case["train"] else 1) * operands + rows * (20 if case["train"] else 12),
                    flops=(6 if case["train"] else 2) * rows * size * classes)
    n, best = rows * case["classes"], case["best"]
    return dict(bytes=(2 if case["train"] else 1) * n * e + rows * (best * (8 + e) + 8), flops=(8 if case["train"] else 4) * n)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    double = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    x = double["x"]
    if case["op"] == "layer_normalization":
        n = case["size"]
        variance, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        std = (variance + EPS).sqrt()
        unit = (x - mean) / std
        y = double["beta"] + double["gamma"] * unit
        if not case["train"]:
            return y
        dy = double["dy"]
        u = double["gamma"] * dy
        dx = (u - (u.sum(1, keepdim=True) + unit * (u * unit).sum(1, keepdim=True)) / n) / std
        return y, dx, dy.sum(0, keepdim=True), torch.einsum("rc,rc->c", dy, unit)[None]
    if case["op"] == "cross_entropy":
        w, label, rows = double["weight"], s["label"], case["rows"]
        bias = double.get("bias")
        losses, dx = [], []
        dw = torch.zeros_like(w) if case["train"] else None
        db = torch.zeros(case["classes"], dtype=torch.float64, device="cuda")
        for a in range(0, rows, 2048):  # (some rows at a time: the logits in 64 bits are large)
            part, at = x[a:a + 2048], label[a:a + 2048, 0]
            logits = torch.mm(part, w) if bias is None else torch.addmm(bias, part, w)
            log_sum = torch.logsumexp(logits, 1)
            valid = at >= 0
            row = torch.arange(part.shape[0], device="cuda")[valid]
            loss = torch.zeros_like(log_sum)
            loss[valid] = log_sum[valid] - logits[row, at[valid]]
            losses.append(loss)
            if case["train"]:
                probability = torch.softmax(logits, 1)
                probability[row, at[valid]] -= 1.0
                probability *= (double["dloss"][a:a + 2048, 0] * valid)[:, None]
                dx.append(probability @ w.T)
                dw.addmm_(part.T, probability)
                db += probability.sum(0)
        loss = torch.cat(losses)[:, None]
        if not case["train"]:
            return loss
        return loss, torch.cat(dx), dw, (db if bias is not None else None)
    t = case["temperature"]
    index, rows = s["index"], case["rows"]
    losses, grads = [], []
    for a in range(0, rows, 1024):
        part, at, teacher = x[a:a + 1024] / t, index[a:a + 1024], double["teacher"][a:a + 1024] / t
        log_sum = torch.logsumexp(part, 1, keepdim=True)
        teacher = teacher.masked_fill(at < 0, -math.inf)
        p = torch.softmax(teacher, 1).nan_to_num(0.0)  # (a row without entries)
        entropy = torch.special.entr(p).sum(1, keepdim=True)
        cross = (p * (part.gather(1, at.clamp(min=0)) - log_sum)).sum(1, keepdim=True)
        losses.append(-t * t * (entropy + cross))
        if case["train"]:
            q = torch.softmax(part, 1) * p.sum(1, keepdim=True)
            grads.append((q.scatter_add(1, at.clamp(min=0), -p) * (t * double["dloss"][a:a + 1024])))
    if not case["train"]:
        return torch.cat(losses)
    return torch.cat(losses), torch.cat(grads)
