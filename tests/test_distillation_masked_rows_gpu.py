"""Rows that take no part in a distillation loss get a gradient of exactly zero, whatever comes from upstream."""
import math

import pytest
import torch

from chronicals_b200 import ops
from chronicals_b200.ops import _ext
from test_distillation_cpu import definition, entries
from test_distillation_gpu import form  # noqa: F401  (both forms of the loss from hidden states)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def _case(T, linear):
    H, V, K = 64, 3000, 6
    g = torch.Generator(device=DEV).manual_seed(T)
    idx, lg = entries(T, V, K, device=DEV)                            # row 2 has no entry
    labels = torch.arange(T, device=DEV).masked_fill(torch.arange(T, device=DEV) % 4 == 1, -100)
    if linear:
        x = (torch.randn(T, H, device=DEV, generator=g).to(BF), (torch.randn(V, H, device=DEV, generator=g) / 8).to(BF))
    else:
        x = (torch.randn(T, V, device=DEV, generator=g),)
    return tuple(t.requires_grad_() for t in x), idx, lg, labels, g


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("linear", [False, True])
@pytest.mark.parametrize("T", [40, 300])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_rows_of_losses(linear, T, bad):
    """A loss of zero sends an infinity through a root or a quotient."""
    x, idx, lg, labels, g = _case(T, linear)
    x64 = tuple(t.detach().double().requires_grad_() for t in x)
    rows, valid = definition(x64[0] @ x64[1].t() if linear else x64[0], idx, lg, 1.5, labels)
    up = torch.randn(T, device=DEV, generator=g)
    want = torch.autograd.grad(rows.to(DEV), x64, torch.where(valid, up, 0.0).double())
    op = ops.linear_distillation if linear else ops.distillation_logits
    loss = op(*x, idx, lg, 1.5, labels, reduction="none")
    got = torch.autograd.grad(loss, x, torch.where(valid, up, bad))
    _ext.check_status()
    assert 0 < int(valid.sum()) < T and (got[0][~valid] == 0).all()
    # d(logits) is rounded to bf16 (half a step, 2^-8) before the products and their results once more; held logits to fp32
    for a, b in zip(got, want):
        assert (a.double() - b).norm() <= (2.0 ** -7 if linear else 1e-5) * b.norm()


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("linear", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_reduced_loss(linear, reduction):
    """An overflowed loss scale: rows that take part are not finite, the others are zero."""
    x, idx, lg, labels, _ = _case(300, linear)
    op = ops.linear_distillation if linear else ops.distillation_logits
    loss = op(*x, idx, lg, 1.5, labels, reduction=reduction)
    (got,) = torch.autograd.grad(loss, x[:1], torch.full_like(loss, math.inf))
    _ext.check_status()
    off = (labels == -100) | (torch.arange(300, device=DEV) == 2)
    assert (got[off] == 0).all() and not torch.isfinite(got[~off]).any()
