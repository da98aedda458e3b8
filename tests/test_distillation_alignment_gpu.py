"""Logits that start off a 16-byte boundary, or whose rows do: the gradient's rows lie as theirs do and no value is read or written alone
that need not be."""
import pytest
import torch

from chronicals_b200 import ops
from chronicals_b200.ops import _ext
from test_distillation_cpu import definition, entries
from test_distillation_gpu import _over

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


# an odd vocabulary from the second row on, columns out of wider rows (twice as wide and more too), rows on top of each other
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("T,V,ld,skip", [(40, 1001, 1001, 1001), (40, 1000, 1011, 3), (700, 257, 600, 5), (3, 9001, 30001, 7), (1, 501, 501, 1),
                                         (6, 1003, 0, 2), (5, 3, 3, 1)])
def test_any_alignment(dtype, T, V, ld, skip):
    g = torch.Generator(device=DEV).manual_seed(V)
    buf = (torch.randn(skip + (T - 1) * ld + V, device=DEV, generator=g) * 3).to(dtype)
    z = buf.as_strided((T, V), (ld, 1), skip).detach().requires_grad_()
    idx, lg = entries(T, V, 9, device=DEV)
    z64 = z.detach().double().requires_grad_()
    rows, valid = definition(z64, idx, lg, 1.5)
    loss = ops.distillation_logits(z, idx, lg, 1.5, reduction="sum")
    (want,) = torch.autograd.grad(rows.sum(), z64)
    # the node's own result, as its kernel wrote it
    grads = []
    hook = loss.grad_fn.register_hook(lambda into, _: grads.append(into[0]))
    torch.autograd.grad(loss, z)
    hook.remove()
    (got,) = grads
    _ext.check_status()
    size = z.element_size()
    assert got.shape == z.shape and (got.data_ptr() - z.data_ptr()) % 16 == 0 and (T == 1 or (got.stride(0) - ld) * size % 16 == 0)
    assert got.stride(0) < V + 16 or got.stride(0) == ld < 2 * V      # no more memory than the logits' own rows, or a vector a row
    # half a step of the type, and p and q 2^-19 off each (22 bits of the exponential, logits of up to 15)
    p = torch.softmax(z64.detach() / 1.5, 1) * 1.5
    assert _over(got.double() - want, torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -18 * (p + (p - want).abs()) + 2.0 ** -126) == 0


def test_entry_point_refuses_rows_at_another_distance():
    z, idx = torch.zeros(4, 16, device=DEV), torch.zeros(2, 2, dtype=torch.int64, device=DEV)
    f = torch.zeros(64, device=DEV)

    def call(shift, ldd):
        return _ext.lib().cb_kd_logits_grad(z.data_ptr(), z.data_ptr() + shift, 2, 16, ldd, 8, 0, idx.data_ptr(), 2, 1, f.data_ptr(), 2, 0, 2,
                                            None, -100, 1.0, f.data_ptr(), f.data_ptr(), f.data_ptr(), None, None, _ext.stream_ptr())
    assert call(4, 16) == call(0, 17) == -1
