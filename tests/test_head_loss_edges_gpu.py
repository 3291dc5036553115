"""resnet18.head_loss: rows that do not count, whatever the teacher says of them."""
import math

import pytest
import torch

from nnabla_b200 import resnet18
from test_training_head_gpu import data

pytestmark = pytest.mark.gpu


def same(a, b):
    return torch.equal(a[0], b[0]) and all(torch.equal(p, q) for p, q in zip(a[1], b[1]))


@pytest.mark.parametrize("rows", [5, 60])
def test_the_teacher_of_a_row_that_does_not_count(rows):
    _, _, _, w, b, label, index, best = data(rows, 48, 100, torch.float32)
    x = torch.randn((rows, 48), device="cuda")
    assert label[0] == -1
    b[17] = -math.inf  # ruled out by the student; no row that counts names it
    index[index == 17] = -1
    clean = index.clone()
    clean[0] = -1
    want = resnet18.head_loss(x, w, b, label, (clean, best), temperature=2.0, share=0.3)
    assert torch.isfinite(want[0]) and all(torch.isfinite(g).all() for g in want[1])
    for entry, logit in [(100, 1.0), (1 << 20, 1.0), (17, 1.0), (3, math.nan), (3, math.inf)]:
        row, kept = index.clone(), best.clone()
        row[0, 0], kept[0, 0] = entry, logit
        given = row.clone()
        assert same(resnet18.head_loss(x, w, b, label, (row, kept), temperature=2.0, share=0.3), want), (entry, logit)
        assert torch.equal(row, given)  # the caller's tensor stays


def test_no_row_counts():
    _, _, _, w, b, label, index, best = data(12, 48, 100, torch.float32)
    x = torch.randn((12, 48), device="cuda")
    label.fill_(-1)
    index[3, 0] = 100
    loss, grads = resnet18.head_loss(x, w, b, label, (index, best))
    assert loss == 0 and all((g == 0).all() for g in grads)


@pytest.mark.parametrize("teacher", [False, True])
def test_labels_as_a_vector(teacher):
    _, _, _, w, b, label, index, best = data(30, 48, 100, torch.float32)
    x = torch.randn((30, 48), device="cuda")
    given = (index, best) if teacher else None
    want = resnet18.head_loss(x, w, b, label, given)
    assert same(resnet18.head_loss(x, w, b, label[:, 0], given), want)
    with pytest.raises(RuntimeError, match="label"):
        resnet18.head_loss(x, w, b, label[:29, 0], given)


@pytest.mark.parametrize("teacher", [False, True])
def test_a_head_without_bias(teacher):
    _, _, _, w, b, label, index, best = data(30, 48, 100, torch.float32)
    x = torch.randn((30, 48), device="cuda")
    given = (index, best) if teacher else None
    loss, (dx, dw, db) = resnet18.head_loss(x, w, None, label, given)
    want = resnet18.head_loss(x, w, torch.zeros_like(b), label, given)
    assert db is None and same((loss, (dx, dw)), (want[0], want[1][:2]))


def test_a_parametric_head_is_trained():
    from nnabla_b200 import functions as F
    from nnabla_b200 import parametric_functions as PF
    PF.clear_parameters()
    x, label = torch.randn((24, 10), device="cuda"), torch.randint(0, 33, (24, 1), device="cuda")
    loss, stat = PF.affine_softmax_cross_entropy(x, label, 33, output_stat=True)
    assert torch.equal(loss, PF.affine_softmax_cross_entropy(x, label, 33))
    p = PF.get_parameters()
    w, b = p["affine/W"], p["affine/b"]
    grads = F.affine_softmax_cross_entropy_backward(x, w, label, stat, torch.full((24, 1), 1 / 24, device="cuda"), b)
    want = resnet18.head_loss(x, w, b, label)
    assert all(torch.equal(g, v) for g, v in zip(grads, want[1]))
    PF.clear_parameters()
