"""Boundaries filled up with empty documents, with the lengths of the others beside them."""
import pytest
import torch

from chronicals_b200 import ops
from chronicals_b200.ops import _ext
from test_attention_window_gpu import _check, _inputs, _truth

pytestmark = pytest.mark.gpu


# head size 80 has no kernel: the library's path, with and without a window
@pytest.mark.parametrize("hq,hk,d", [(16, 4, 64), (2, 1, 128), (2, 1, 80)])
@pytest.mark.parametrize("lens", [[2500], [700, 40, 0, 1300]])
@pytest.mark.parametrize("window,sinks", [(1100, 3), (None, 0)])
def test_lengths_of_the_documents_that_are_not_empty(hq, hk, d, lens, window, sinks):
    qkv, do, cu = _inputs(hq, hk, d, lens, 0)
    more = torch.cat((cu, cu[-1:].expand(60)))
    x = qkv.detach().requires_grad_()
    o = ops.attention_qkv_packed(x, more, hq, hk, d, None, [n for n in lens if n], window, sinks)
    (g,) = torch.autograd.grad(o, x, do)
    _ext.check_status()
    _check((o.detach(), g), _truth(qkv, do, hq, hk, d, lens, window or 10 ** 6, sinks), hq, hk, d, sum(lens))
