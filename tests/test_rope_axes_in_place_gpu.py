"""Rotating in place is seen by what keeps the buffer for a backward pass."""
import pytest
import torch

from chronicals_b200 import ops
from test_rope_axes_gpu import _inputs

pytestmark = pytest.mark.gpu


def test_a_buffer_kept_for_a_backward_pass():
    x, cos, sin, pos = _inputs(20, 2, 1, 64, 3)
    w = torch.ones_like(x, requires_grad=True)
    y = x * w                                                         # keeps x: its value is the gradient of w
    ops.qk_rope_axes_(x, cos, sin, pos, 2, 1, 64, (8, 12, 12))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_without_autograd():
    x, cos, sin, pos = _inputs(20, 2, 1, 64, 3)
    want = ops.qk_rope_axes_(x.clone(), cos, sin, pos, 2, 1, 64, (8, 12, 12))
    with torch.inference_mode():
        assert torch.equal(ops.qk_rope_axes_(x.clone(), cos, sin, pos, 2, 1, 64, (8, 12, 12)), want)
    with torch.no_grad():
        leaf = x.clone().requires_grad_()
        assert torch.equal(ops.qk_rope_axes_(leaf, cos, sin, pos, 2, 1, 64, (8, 12, 12)), want)
