"""Tokens before the first boundary belong to no document, like those behind the last one: zeros, and no gradient."""
import pytest
import torch

from chronicals_b200 import ops
from chronicals_b200.ops.attention import _sdpa_docs
from test_attention_window_cpu import cu_of, dense


def definition(qkv, lens, lead, hq, hk, d, window, sinks):
    T = qkv.shape[0]
    q, k, v = (t.reshape(T, -1, d)[lead:] for t in qkv.split((hq * d, hk * d, hk * d), 1))
    return torch.cat((qkv.new_zeros(lead, hq, d), dense(q, k, v, lens, window, sinks))).reshape(T, hq * d)


@pytest.mark.parametrize("lens,lead,pad", [([7], 3, 2), ([7], 3, 0), ([4, 0, 5], 1, 0), ([], 5, 3)])
@pytest.mark.parametrize("window", [4, None])
def test_rows_before_the_first_document(lens, lead, pad, window):
    hq, hk, d, T = 4, 2, 8, lead + sum(lens) + pad
    qkv = torch.randn(T, (hq + 2 * hk) * d, requires_grad=True)
    up = torch.randn(T, hq * d)
    cu = lead + cu_of(lens)
    want = definition(qkv, lens, lead, hq, hk, d, window or 100, 0)
    ref = torch.autograd.grad(want, qkv, up)[0] if lens else torch.zeros_like(qkv)
    q, k, v = (t.reshape(T, -1, d) for t in qkv.split((hq * d, hk * d, hk * d), 1))
    for got in (ops.attention_qkv_packed(qkv, cu, hq, hk, d, window=window), ops.attention_varlen(q, k, v, cu, window=window).reshape(T, -1)):
        assert torch.allclose(got, want, atol=1e-5)
        if got.requires_grad:
            assert torch.allclose(torch.autograd.grad(got, qkv, up, retain_graph=True)[0], ref, atol=1e-5)


@pytest.mark.parametrize("lens,lead,pad", [([7], 3, 2), ([4, 0, 5], 1, 0), ([6, 6], 2, 1), ([6, 6], 0, 0)])
def test_the_librarys_path(lens, lead, pad):
    """Head sizes without a kernel, on the GPU."""
    hq, hk, d, T = 4, 2, 8, lead + sum(lens) + pad
    qkv = torch.randn(T, (hq + 2 * hk) * d, requires_grad=True)
    q, k, v = (t.reshape(T, -1, d) for t in qkv.split((hq * d, hk * d, hk * d), 1))
    got = _sdpa_docs(q, k, v, (lead + cu_of(lens)).tolist(), True, d ** -0.5).reshape(T, -1)
    want = definition(qkv, lens, lead, hq, hk, d, T, 0)
    up = torch.randn_like(want)
    assert torch.allclose(got, want, atol=1e-5)
    assert torch.allclose(torch.autograd.grad(got, qkv, up, retain_graph=True)[0], torch.autograd.grad(want, qkv, up)[0], atol=1e-5)
