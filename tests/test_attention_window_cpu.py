"""Attention with a window and sinks: the definition, its gradient, and what is refused."""
import math

import pytest
import torch

from chronicals_b200 import ops


def dense(q, k, v, lens, window, sinks, scale=None):
    """Document by document with the full mask; differentiable, in the inputs' type.  ``q [T, hq, d]``, ``k / v [T, hk, d]``."""
    out, at, rep = [], 0, q.shape[1] // k.shape[1]
    for n in lens:
        i = torch.arange(n, device=q.device)
        see = (i[None] <= i[:, None]) & ((i[:, None] - i[None] < window) | (i[None] < sinks))
        s = torch.einsum("ihd,jhd->hij", q[at:at + n], k[at:at + n].repeat_interleave(rep, 1)) * (scale or q.shape[2] ** -0.5)
        p = torch.softmax(s.masked_fill(~see, -math.inf), -1)
        out.append(torch.einsum("hij,jhd->ihd", p, v[at:at + n].repeat_interleave(rep, 1)))
        at += n
    out.append(q.new_zeros(q.shape[0] - at, *q.shape[1:]))
    return torch.cat(out)


def cu_of(lens, device="cpu"):
    return torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=device)


@pytest.mark.parametrize("lens,pad", [([1], 0), ([7, 1, 30], 2), ([0, 5, 0], 0), ([600], 3)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 0), (3, 2), (1, 1), (1000, 0), (4, 50), (513, 4)])
def test_definition_and_gradient(lens, pad, window, sinks):
    hq, hk, d = 4, 2, 8
    T = sum(lens) + pad
    qkv = torch.randn(T, (hq + 2 * hk) * d, dtype=torch.float64, requires_grad=True)
    q, k, v = (t.reshape(T, -1, d) for t in qkv.split((hq * d, hk * d, hk * d), 1))
    want = dense(q, k, v, lens, window, sinks)
    up = torch.randn_like(want)
    (ref,) = torch.autograd.grad(want, qkv, up, retain_graph=True)
    cu = cu_of(lens)
    for got in (ops.attention_qkv_packed(qkv, cu, hq, hk, d, window=window, sinks=sinks).view(T, hq, d),
                ops.attention_varlen(q, k, v, cu, window=window, sinks=sinks)):
        assert torch.allclose(got, want, atol=1e-12)
        assert torch.allclose(torch.autograd.grad(got, qkv, up, retain_graph=True)[0], ref, atol=1e-12)


def test_gradient_against_differences():
    qkv = torch.randn(6, 12, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda x: ops.attention_qkv_packed(x, cu_of([4, 2]), 1, 1, 4, window=2, sinks=1), (qkv,))


def test_a_window_over_the_whole_document_is_plain_attention():
    x, cu = torch.randn(20, 32), cu_of([12, 8])
    assert torch.allclose(ops.attention_qkv_packed(x, cu, 2, 1, 8, window=12), ops.attention_qkv_packed(x, cu, 2, 1, 8), atol=1e-6)


def test_scale():
    q = torch.randn(9, 2, 8, dtype=torch.float64)
    got = ops.attention_varlen(q, q, q, cu_of([9]), softmax_scale=0.7, window=4, sinks=1)
    assert torch.allclose(got, dense(q, q, q, [9], 4, 1, 0.7), atol=1e-12)


def test_no_documents():
    x = torch.randn(3, 32)
    assert (ops.attention_qkv_packed(x, torch.zeros(1, dtype=torch.int32), 2, 1, 8, window=2) == 0).all()
    assert ops.attention_qkv_packed(x[:0], torch.zeros(2, dtype=torch.int32), 2, 1, 8, window=2).shape == (0, 16)


@pytest.mark.parametrize("kw,what", [
    (dict(window=0), "window 0"), (dict(window=-3), "window -3"), (dict(window=2.0), "whole"), (dict(window=True), "whole"),
    (dict(window=4, sinks=-1), "negative"), (dict(window=4, sinks=1.0), "whole"), (dict(sinks=2), "without a window")])
@pytest.mark.parametrize("packed", [False, True])
def test_refusals(kw, what, packed):
    x = torch.randn(5, 32)
    with pytest.raises(ValueError, match=what):
        if packed:
            ops.attention_qkv_packed(x, cu_of([5]), 2, 1, 8, **kw)
        else:
            q, k, v = (t.reshape(5, -1, 8) for t in x.split((16, 8, 8), 1))
            ops.attention_varlen(q, k, v, cu_of([5]), **kw)


def test_refusals_of_shapes_and_options():
    x, cu = torch.randn(5, 32), cu_of([5])
    for heads in ((2, 2, 8), (3, 2, 8), (2, 0, 16), (2, 1, 16)):
        with pytest.raises(ValueError, match="qkv"):
            ops.attention_qkv_packed(x, cu, *heads, window=2)
    q, k = torch.randn(5, 4, 8), torch.randn(5, 2, 8)
    for bad in ((q, k, k[:4]), (q, k[:4], k[:4]), (q, torch.randn(5, 3, 8), torch.randn(5, 3, 8)), (q, k[..., :4], k[..., :4])):
        with pytest.raises(ValueError, match="do not fit"):
            ops.attention_varlen(*bad, cu, window=2)
    with pytest.raises(ValueError, match="causal"):
        ops.attention_varlen(q, k, k, cu, causal=False, window=2)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="softmax_scale"):
            ops.attention_varlen(q, k, k, cu, softmax_scale=scale, window=2)
