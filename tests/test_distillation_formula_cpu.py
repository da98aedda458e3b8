"""The formula's path of the distillation losses: rows that take no part are not read, and logits not all held at once."""
import math

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from chronicals_b200 import ops
from chronicals_b200.ops import ref
from test_distillation_cpu import definition


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.float64])
def test_rows_that_take_no_part(value, reduction, dtype):
    z = torch.randn(4, 50).to(dtype)
    z[1:3] = value
    z.requires_grad_()
    idx, lg = torch.tensor([[1, 4], [0, 3], [-1, 50], [7, 7]]), torch.zeros(4, 2)
    labels = torch.tensor([0, -100, 0, 0])                            # row 1 is masked, row 2 has no entry
    loss = ops.distillation_logits(z, idx, lg, 1.0, labels, reduction=reduction)
    (grad,) = torch.autograd.grad(loss.sum(), z)
    z64 = z.detach().double()
    z64[1:3] = 0.0                                                    # the definition multiplies them by zero
    z64.requires_grad_()
    rows, valid = definition(z64, idx, lg, 1.0, labels)
    want = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / valid.sum()}[reduction]
    assert torch.allclose(loss.double(), want, rtol=1e-5)
    assert (grad[1:3] == 0).all()
    (exact,) = torch.autograd.grad(rows[[0, 3]].sum() / (valid.sum() if reduction == "mean" else 1), z64)
    eps = torch.finfo(dtype).eps
    assert (grad[[0, 3]].double() - exact[[0, 3]]).abs().max() <= eps / 2 * exact.abs().max() + 1e-6


class _Largest(TorchDispatchMode):
    values = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        for t in out if isinstance(out, (tuple, list)) else (out,):
            if isinstance(t, torch.Tensor):
                self.values = max(self.values, t.numel())
        return out


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("masked", [False, True])
def test_logits_are_formed_a_stretch_of_rows_at_a_time(monkeypatch, reduction, masked):
    T, V, H, K = 37, 300, 8, 4
    h, w = (torch.randn(n, H, dtype=torch.float64, requires_grad=True) for n in (T, V))
    idx, lg = torch.randint(0, V, (T, K)), torch.randn(T, K)
    labels = torch.arange(T).masked_fill(torch.arange(T) % 3 == 0, -100) if masked else None
    up = torch.randn(T if reduction == "none" else ())
    want = ops.linear_distillation(h, w, idx, lg, 1.5, labels, reduction=reduction)
    dense = torch.autograd.grad(want, (h, w), up)
    monkeypatch.setattr(ref, "LINEAR_DISTILL_VALUES", 5 * V)
    with _Largest() as largest:
        got = ops.linear_distillation(h, w, idx, lg, 1.5, labels, reduction=reduction)
        grads = torch.autograd.grad(got, (h, w), up)
    assert largest.values <= max(5 * V, V * H) < T * V
    assert torch.allclose(got, want) and all(torch.allclose(a, b) for a, b in zip(grads, dense))
    with torch.no_grad():
        assert torch.equal(ops.linear_distillation(h, w, idx, lg, 1.5, labels, reduction=reduction), got)
