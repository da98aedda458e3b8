"""Distillation from a teacher's top logits: the definition in 64 bits, its gradient, and what is refused."""
import math

import pytest
import torch

from chronicals_b200 import ops

NEG = -math.inf


def definition(z, idx, lg, tau=1.0, labels=None, ignore=-100):
    """``(rows, valid)`` in 64 bits with a dense teacher: the cross-entropy of the two distributions less the teacher's entropy."""
    z, V = z.double(), z.shape[1]
    rows, valid = [], []
    for r in range(z.shape[0]):
        t = {}
        for i, l in zip(idx[r].tolist(), lg[r].double().tolist()):
            if 0 <= i < V and l != NEG:
                t.setdefault(i, []).append(l / tau)
        on = bool(t) and (labels is None or int(labels[r]) != ignore)
        valid.append(on)
        if not on:
            rows.append(z[r].sum() * 0.0)
            continue
        every = [l for ls in t.values() for l in ls]
        top = max(every)
        total = sum(math.exp(l - top) for l in every)
        logp = torch.log_softmax(z[r] / tau, 0)
        row = 0.0
        for i, ls in t.items():
            q = sum(math.exp(l - top) for l in ls) / total
            if q > 0:
                row = row + q * (math.log(q) - logp[i])
        rows.append(tau * tau * row)
    return torch.stack([torch.as_tensor(r, dtype=torch.float64, device=z.device) for r in rows]), torch.tensor(valid, device=z.device)


def entries(T, V, K, seed=0, device="cpu"):
    """Distinct entries, with an absent one, a -inf, a far one, an index past the vocabulary, and a row of none."""
    g = torch.Generator().manual_seed(seed + K)
    idx = torch.stack([torch.randperm(max(V, K), generator=g)[:K] for _ in range(T)])
    lg = torch.randn(T, K, generator=g) * 3
    if K > 4:
        idx[0, 1], lg[0, 2], lg[0, 3], idx[0, 4] = -1, NEG, -300.0, V
    if T > 2:
        idx[2] = -7
    return idx.to(device), lg.to(device)


@pytest.mark.parametrize("T,V,K,tau", [(1, 5, 1, 1.0), (4, 50, 7, 1.0), (6, 33, 40, 2.5), (5, 300, 5, 0.5)])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("linear", [False, True])
def test_definition_and_gradient(T, V, K, tau, reduction, masked, linear):
    idx, lg = entries(T, V, K)
    labels = torch.arange(T).masked_fill(torch.arange(T) % 3 == 1, -100) if masked else None
    H = 8
    h = torch.randn(T, H, dtype=torch.float64, requires_grad=True)
    w = torch.randn(V, H, dtype=torch.float64, requires_grad=True)
    z = (h @ w.t()).detach().requires_grad_()
    args = (idx, lg, tau, labels, -100, reduction)
    loss = ops.linear_distillation(h, w, *args) if linear else ops.distillation_logits(z, *args)
    z64 = h @ w.t() if linear else z
    rows, valid = definition(z64, idx, lg, tau, labels)
    want = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / max(1, int(valid.sum()))}[reduction]
    assert loss.shape == want.shape and torch.allclose(loss, want, atol=1e-12)
    up = torch.randn(loss.shape, dtype=torch.float64)
    leaves = (h, w) if linear else (z,)
    got, ref = (torch.autograd.grad(x, leaves, up) for x in (loss, want))
    assert all(torch.allclose(a, b, atol=1e-12) for a, b in zip(got, ref))


def test_gradient_against_differences():
    z = torch.randn(3, 9, dtype=torch.float64, requires_grad=True)
    idx, lg = torch.tensor([[1, 4, 8], [0, 0, 3], [-1, 2, 9]]), torch.randn(3, 3)
    assert torch.autograd.gradcheck(lambda x: ops.distillation_logits(x, idx, lg, 1.7), (z,))


def test_entries_of_one_index_add_up():
    z = torch.randn(1, 6, dtype=torch.float64)
    one = ops.distillation_logits(z, torch.tensor([[2, 5]]), torch.tensor([[math.log(3.0), 0.0]]).double())
    three = ops.distillation_logits(z, torch.tensor([[2, 2, 5, 2]]), torch.zeros(1, 4).double())
    # log 3 is given in 32 bits, at most half a step (2^-24 of a number below 2) off; the loss moves by q (log q - log p - loss) of
    # that, here below 1
    assert abs(float(three - one)) < 2.0 ** -23


def test_a_teacher_that_is_the_student_over_the_whole_vocabulary_loses_nothing():
    z = torch.randn(4, 20, dtype=torch.float64, requires_grad=True)
    loss = ops.distillation_logits(z, torch.arange(20).expand(4, 20), z, 2.0)
    assert abs(loss.item()) < 1e-12
    assert torch.autograd.grad(loss, z)[0].abs().max() < 1e-12


def test_nothing_takes_part():
    z = torch.randn(3, 7, requires_grad=True)
    for idx, labels in ((torch.full((3, 2), -1), None), (torch.zeros(3, 2, dtype=torch.int32), torch.full((3,), -100))):
        loss = ops.distillation_logits(z, idx, torch.zeros(3, 2), 1.0, labels)
        assert loss.item() == 0 and torch.autograd.grad(loss, z)[0].abs().max() == 0
    assert ops.distillation_logits(z[:0], torch.zeros(0, 2, dtype=torch.int64), torch.zeros(0, 2)).item() == 0


def test_student_logits_of_minus_infinity():
    """At an absent word they carry no weight; at a word of the teacher's the loss is infinite, as the formula says."""
    z = torch.randn(1, 6)
    z[0, 3] = NEG
    z.requires_grad_()
    loss = ops.distillation_logits(z, torch.tensor([[0, 1]]), torch.zeros(1, 2))
    assert math.isfinite(loss.item()) and torch.isfinite(torch.autograd.grad(loss, z)[0]).all()
    assert ops.distillation_logits(z, torch.tensor([[0, 3]]), torch.zeros(1, 2)).item() == math.inf


def test_leading_dimensions():
    z, idx, lg = torch.randn(2, 3, 11), torch.randint(0, 11, (2, 3, 4)), torch.randn(2, 3, 4)
    rows = ops.distillation_logits(z, idx, lg, reduction="none")
    assert rows.shape == (2, 3)
    flat = ops.distillation_logits(z.view(6, 11), idx.view(6, 4), lg.view(6, 4), reduction="none")
    assert torch.equal(rows.reshape(6), flat)
    assert torch.allclose(ops.distillation_logits(z, idx, lg, labels=torch.zeros(2, 3, dtype=torch.int64)), flat.mean())


@pytest.mark.parametrize("change,what", [
    (dict(idx=torch.zeros(3, 2, dtype=torch.int64)), "teacher_indices"), (dict(idx=torch.zeros(4, 0, dtype=torch.int64), lg=torch.zeros(4, 0)), "K >= 1"),
    (dict(lg=torch.zeros(4, 3)), "teacher_logits"), (dict(idx=torch.zeros(4, 2)), "whole numbers"), (dict(lg=torch.zeros(4, 2, dtype=torch.int64)), "floating"),
    (dict(idx=torch.zeros(4, 2, dtype=torch.bool)), "whole numbers"), (dict(tau=0.0), "temperature"), (dict(tau=-1.0), "temperature"),
    (dict(tau=math.inf), "temperature"), (dict(tau=math.nan), "temperature"), (dict(labels=torch.zeros(3, dtype=torch.int64)), "labels"),
    (dict(labels=torch.zeros(4)), "labels"), (dict(reduction="batchmean"), "reduction")])
@pytest.mark.parametrize("linear", [False, True])
def test_refusals(change, what, linear):
    idx, lg = change.get("idx", torch.zeros(4, 2, dtype=torch.int64)), change.get("lg", torch.zeros(4, 2))
    args = (idx, lg, change.get("tau", 1.0), change.get("labels"), -100, change.get("reduction", "mean"))
    with pytest.raises(ValueError, match=what):
        ops.linear_distillation(torch.zeros(4, 8), torch.zeros(9, 8), *args) if linear else ops.distillation_logits(torch.zeros(4, 9), *args)


def test_weight_that_does_not_fit():
    with pytest.raises(ValueError, match="weight"):
        ops.linear_distillation(torch.zeros(4, 8), torch.zeros(9, 7), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2))
