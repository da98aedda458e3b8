"""Labels, indices and positions of types that are not whole numbers are refused, not read as such."""
import pytest
import torch

from chronicals_b200 import ops

TYPES = [torch.bool, torch.float32, torch.bfloat16, torch.complex64]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("linear", [False, True])
def test_distillation(dtype, linear):
    h, w = torch.randn(3, 8), torch.randn(11, 8)
    x, op = ((h, w), ops.linear_distillation) if linear else ((h @ w.t(),), ops.distillation_logits)
    idx, lg, ones = torch.tensor([[0, 1]] * 3), torch.zeros(3, 2), torch.ones(3, dtype=torch.int32)
    assert op(*x, idx, lg, labels=ones).isfinite()
    with pytest.raises(ValueError, match="whole numbers"):
        op(*x, idx, lg, labels=ones.to(dtype))
    with pytest.raises(ValueError, match="whole numbers"):
        op(*x, idx.to(dtype), lg)


@pytest.mark.parametrize("dtype", TYPES)
def test_positions(dtype):
    qkv, cos, sin = torch.randn(3, 48), torch.ones(4, 8), torch.zeros(4, 8)
    pos = torch.zeros(2, 3, dtype=torch.int16)
    ops.qk_rope_axes_(qkv, cos, sin, pos, 1, 1, 16, (4, 4))
    with pytest.raises(ValueError, match="whole numbers"):
        ops.qk_rope_axes_(qkv, cos, sin, pos.to(dtype), 1, 1, 16, (4, 4))
