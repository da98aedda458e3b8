"""Rows of no document on the kernels: zeros in the output and in the gradient, whatever was in memory before."""
import math

import pytest
import torch

from chronicals_b200 import ops
from chronicals_b200.ops import _ext
from test_attention_rows_outside_cpu import definition
from test_attention_window_cpu import cu_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


# rows in front and behind that together take a block or several; tiles that leave the fewest CTAs for them
@pytest.mark.parametrize("lens,lead,pad", [([200], 1, 1), ([127], 1, 0), ([128, 1, 300], 130, 61), ([1], 700, 0), ([129] * 3, 127, 129), ([0, 77], 300, 5)])
@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (2, 1, 128)])
@pytest.mark.parametrize("window,sinks", [(70, 2), (None, 0)])
def test_rows_before_the_first_document(lens, lead, pad, hq, hk, d, window, sinks):
    T = lead + sum(lens) + pad
    g = torch.Generator(device=DEV).manual_seed(T)
    qkv = torch.randn(T, (hq + 2 * hk) * d, device=DEV, generator=g).to(BF)
    do = torch.randn(T, hq * d, device=DEV, generator=g).to(BF)
    x64 = qkv.double().requires_grad_()
    want = definition(x64, lens, lead, hq, hk, d, window or T, sinks)
    (ref,) = torch.autograd.grad(want, x64, do.double())
    qkv.requires_grad_()
    for n in (1, 2, 4):                                               # what the allocator hands out next is not zero
        torch.full((n * qkv.numel(),), math.nan, dtype=BF, device=DEV)
    o = ops.attention_qkv_packed(qkv, cu_of(lens, DEV) + lead, hq, hk, d, window=window, sinks=sinks)
    (dx,) = torch.autograd.grad(o, qkv, do)
    _ext.check_status()
    inside = slice(lead, lead + sum(lens))
    for a, b in ((o, want), (dx, ref)):
        assert (a[:lead] == 0).all() and (a[inside.stop:] == 0).all()
        # as in the tests of documents that begin with the first row: two roundings to bf16
        assert (a[inside].double() - b[inside]).norm() <= 2.0 ** -7 * b[inside].norm() + 1e-3
