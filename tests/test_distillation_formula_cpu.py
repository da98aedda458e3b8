"""The formula's path of the distillation losses: rows that take no part are not read."""
import math

import pytest
import torch

from chronicals_b200 import ops
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
    (ref,) = torch.autograd.grad(rows[[0, 3]].sum() / (valid.sum() if reduction == "mean" else 1), z64)
    eps = torch.finfo(dtype).eps
    assert (grad[[0, 3]].double() - ref[[0, 3]]).abs().max() <= eps / 2 * ref.abs().max() + 1e-6
