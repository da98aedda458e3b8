"""The windowed attention kernels against the definition in 64 bits."""
import math

import pytest
import torch

from chronicals_b200 import ops
from chronicals_b200.ops import _ext
from test_attention_window_cpu import cu_of, dense

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16


def _inputs(hq, hk, d, lens, pad, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(sum(lens) + hq + d)
    T = sum(lens) + pad
    qkv = (torch.randn(T, (hq + 2 * hk) * d, device=DEV, generator=g) * scale).to(BF)
    return qkv, torch.randn(T, hq * d, device=DEV, generator=g).to(BF), cu_of(lens, DEV)


def _truth(qkv, do, hq, hk, d, lens, window, sinks):
    x = qkv.detach().double().requires_grad_()
    q, k, v = (t.reshape(x.shape[0], -1, d) for t in x.split((hq * d, hk * d, hk * d), 1))
    o = dense(q, k, v, lens, window, sinks).reshape(x.shape[0], -1)
    return o.detach(), torch.autograd.grad(o, x, do.double())[0]


def _run(qkv, do, cu, hq, hk, d, window, sinks):
    x = qkv.detach().requires_grad_()
    o = ops.attention_qkv_packed(x, cu, hq, hk, d, window=window, sinks=sinks)
    (g,) = torch.autograd.grad(o, x, do)
    _ext.check_status()
    return o.detach(), g


def _check(got, want, hq, hk, d, valid, bound=2.0 ** -7):
    # P is rounded to bf16 (relative 2^-9 on average) before the product with V, the result once more; the gradient's P and dS
    # likewise, and delta comes from the rounded output: below 2^-7 of the norm together, of the whole and of the worst row
    (o, g), (o64, g64) = got, want
    assert (o[valid:] == 0).all() and (g[valid:] == 0).all()
    parts = [(o, o64)] + [(g[:, a:b], g64[:, a:b]) for a, b in ((0, hq * d), (hq * d, (hq + hk) * d), ((hq + hk) * d, (hq + 2 * hk) * d))]
    for x, y in parts:
        off = (x[:valid].double() - y[:valid]).norm().item()
        assert off <= bound * y[:valid].norm().item() + 1e-3, (off, y[:valid].norm().item())
    rows = (o[:valid].double() - o64[:valid]).norm(dim=1) - 2.0 ** -6 * o64[:valid].norm(dim=1)
    assert rows.max().item() <= 0


# windows of one token, one short of, at and past a key block (64 forward, 128 backward) and a tile; sinks likewise, merging with
# the window or apart from it
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 5), (63, 0), (64, 1), (65, 64), (127, 65), (128, 0), (129, 4), (200, 128),
                                          (300, 129), (511, 0), (700, 300), (5000, 0), (5000, 7)])
def test_windows_and_sinks(d, window, sinks):
    hq, hk, lens, pad = 4, 2, [650, 1, 129, 64, 300], 37
    qkv, do, cu = _inputs(hq, hk, d, lens, pad)
    _check(_run(qkv, do, cu, hq, hk, d, window, sinks), _truth(qkv, do, hq, hk, d, lens, window, sinks), hq, hk, d, sum(lens))


# lengths from one token, around the tile sizes; more documents than lanes of a warp; empty documents; every head layout
@pytest.mark.parametrize("hq,hk,d,lens,pad", [
    (1, 1, 64, [1], 0), (1, 1, 128, [1], 0), (3, 3, 128, [127, 128, 129], 0), (3, 1, 64, [63, 65, 255, 257], 1), (2, 1, 64, [3] * 70 + [130], 200),
    (4, 2, 128, [0, 31, 0, 0, 257, 600, 2, 0], 5), (7, 1, 128, [385, 512], 0), (14, 2, 64, [511, 512], 0), (24, 24, 64, [200], 0),
    (28, 4, 128, [333], 3), (8, 8, 64, [640, 511], 130)])
@pytest.mark.parametrize("window,sinks", [(100, 0), (100, 4), (33, 70)])
def test_lengths_and_heads(hq, hk, d, lens, pad, window, sinks):
    qkv, do, cu = _inputs(hq, hk, d, lens, pad)
    _check(_run(qkv, do, cu, hq, hk, d, window, sinks), _truth(qkv, do, hq, hk, d, lens, window, sinks), hq, hk, d, sum(lens))


# long documents: sinks are met by every later block, in several runs; both backward kernels of head size 64 (one CTA an SM where
# the grid is small or the loops are long, two where it is large and they are short)
@pytest.mark.parametrize("hq,hk,d,lens,window,sinks", [
    (2, 1, 64, [4100], 130, 4), (2, 1, 128, [4100], 130, 4), (2, 2, 64, [3000], 900, 200), (2, 2, 128, [2500], 600, 129), (1, 1, 64, [5000], 2500, 1),
    (16, 4, 64, [2600, 300], 200, 3), (16, 2, 64, [2700], 64, 150), (16, 16, 64, [2400], 1100, 0), (4, 1, 128, [2100, 2000], 1, 1)])
def test_long_documents(hq, hk, d, lens, window, sinks):
    qkv, do, cu = _inputs(hq, hk, d, lens, 0)
    _check(_run(qkv, do, cu, hq, hk, d, window, sinks), _truth(qkv, do, hq, hk, d, lens, window, sinks), hq, hk, d, sum(lens))


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("lens,window,sinks", [([57, 59, 30, 84] * 10, 2000, 1), ([120] * 18, 33, 4), ([2300], 20, 0), ([900], 300, 2)])
def test_gradients_of_few_visible_keys(hq, hk, d, lens, window, sinks):
    """The gradient's own rounding, and that of P or dS before the products, as large and independent of it: the square root of two
    roundings together.  That of O, which the row sums would take in, is kept out where few keys are visible."""
    qkv, do, cu = _inputs(hq, hk, d, lens, 0)
    g64 = _truth(qkv, do, hq, hk, d, lens, window, sinks)[1]
    g = _run(qkv, do, cu, hq, hk, d, window, sinks)[1]
    assert (g.double() - g64).norm() <= 1.5 * (g64.to(BF).double() - g64).norm()


@pytest.mark.parametrize("d", [64, 128])
def test_many_sinks_in_many_short_documents(d):
    """Every document's whole length is sinks: no more tiles than its own blocks ask for."""
    hq, hk, lens = 2, 1, [7] * 1100 + [300]
    qkv, do, cu = _inputs(hq, hk, d, lens, 0)
    _check(_run(qkv, do, cu, hq, hk, d, 2, 8000), _truth(qkv, do, hq, hk, d, lens, 2, 8000), hq, hk, d, sum(lens))


@pytest.mark.parametrize("d", [64, 128])
def test_large_scores(d):
    """Scores of several hundreds: the running maximum moves, and most probabilities vanish."""
    hq, hk, lens = 4, 2, [700, 130]
    qkv, do, cu = _inputs(hq, hk, d, lens, 0, scale=6.0)
    o, g = _run(qkv, do, cu, hq, hk, d, 150, 3)
    o64, g64 = _truth(qkv, do, hq, hk, d, lens, 150, 3)
    assert torch.isfinite(o).all() and torch.isfinite(g).all()
    assert (o.double() - o64).norm() <= 2.0 ** -6 * o64.norm()       # the exponent of a score of 300 is 300 * 2^-24 * log2(e) off


@pytest.mark.parametrize("d", [64, 128])
def test_a_window_over_the_whole_document_is_plain_attention(d):
    hq, hk, lens = 4, 2, [300, 515]
    qkv, do, cu = _inputs(hq, hk, d, lens, 9)
    x = qkv.detach().requires_grad_()
    o = ops.attention_qkv_packed(x, cu, hq, hk, d)
    (g,) = torch.autograd.grad(o, x, do)
    a, b = _run(qkv, do, cu, hq, hk, d, 515, 0)
    assert (a.double() - o.double()).norm() <= 2.0 ** -8 * o.double().norm()
    assert (b.double() - g.double()).norm() <= 2.0 ** -7 * g.double().norm()


def test_strided_rows_and_separate_tensors():
    hq, hk, d, lens = 4, 2, 64, [130, 200]
    qkv, do, cu = _inputs(hq, hk, d, lens, 0)
    want = _run(qkv, do, cu, hq, hk, d, 90, 4)
    for gap in (8, 24, 3):                                            # the last: rows that TMA cannot address
        buf = torch.full((qkv.shape[0], qkv.shape[1] + gap), math.nan, dtype=BF, device=DEV)
        buf[:, : qkv.shape[1]] = qkv
        got = _run(buf[:, : qkv.shape[1]], do, cu.long(), hq, hk, d, 90, 4)
        assert torch.equal(got[0], want[0]) and (got[1].double() - want[1].double()).norm() <= 2.0 ** -8 * want[1].double().norm()
    q, k, v = (t.reshape(qkv.shape[0], -1, d) for t in qkv.split((hq * d, hk * d, hk * d), 1))
    assert torch.equal(ops.attention_varlen(q, k, v, cu, window=90, sinks=4).reshape(-1, hq * d), want[0])
    wide = torch.empty(do.numel() + 1, dtype=BF, device=DEV)[1:].view_as(do).copy_(do)      # a gradient off the 16-byte boundary
    assert (_run(qkv, wide, cu, hq, hk, d, 90, 4)[1].double() - want[1].double()).norm() <= 2.0 ** -8 * want[1].double().norm()


@pytest.mark.parametrize("dtype,d", [(torch.float32, 64), (BF, 80), (torch.float16, 64)])
def test_what_the_kernels_do_not_take_follows_the_formula(dtype, d):
    hq, hk, lens = 2, 1, [70, 600]
    qkv, do, cu = _inputs(hq, hk, d, lens, 3)
    qkv, do = qkv.to(dtype), do.to(dtype)
    _check(_run(qkv, do, cu, hq, hk, d, 50, 4), _truth(qkv, do, hq, hk, d, lens, 50, 4), hq, hk, d, sum(lens))


def test_other_stream_and_graph():
    hq, hk, d, lens = 4, 2, 64, [300, 77]
    qkv, do, cu = _inputs(hq, hk, d, lens, 3)
    want = _run(qkv, do, cu, hq, hk, d, 64, 4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = _run(qkv, do, cu, hq, hk, d, 64, 4)
    torch.cuda.current_stream().wait_stream(s)
    buf = torch.zeros_like(qkv).requires_grad_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = ops.attention_qkv_packed(buf, cu, hq, hk, d, window=64, sinks=4)
        (dx,) = torch.autograd.grad(o, buf, do)
    with torch.no_grad():
        buf.copy_(qkv)
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    for a, b in ((side[0], side[1]), (o.detach(), dx)):
        assert torch.equal(a, want[0])
        # the additions into dQ, dK and dV come in any order: last bits of 32, then a rounding that may fall the other way
        assert (b.double() - want[1].double()).norm() <= 2.0 ** -8 * want[1].double().norm()


def test_entry_points_refuse_bad_arguments():
    x = torch.zeros(128, 256, dtype=BF, device=DEV)
    f = torch.zeros(4096, device=DEV)
    cu = cu_of([128], DEV)
    st = _ext.status_buffer(x.device).data_ptr()
    p = x.data_ptr()

    def fwd(T=128, docs=1, hq=2, hk=1, d=64, window=4, sinks=0):
        return _ext.lib().cb_attn_window_fwd(p, p, p, p, f.data_ptr(), cu.data_ptr(), docs, T, hq, hk, d, 256, 256, 256, 256, 0.125, window,
                                             sinks, None, st, _ext.stream_ptr())
    assert fwd(T=0) == fwd(docs=0) == fwd(hk=0) == fwd(hq=3, hk=2) == fwd(d=80) == fwd(window=0) == fwd(sinks=-1) == -1
    assert fwd(docs=70000) == -1                                      # more tiles than a grid has rows
    assert _ext.lib().cb_attn_window_bwd(p, p, p, p, p, f.data_ptr(), cu.data_ptr(), 1, 128, 2, 1, 64, 256, 256, 256, 256, 256, 0.125, 0, 0, None,
                                         f.data_ptr(), f.data_ptr(), f.data_ptr(), f.data_ptr(), p, 256, st, _ext.stream_ptr()) == -1


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 64), (32, 8, 64), (4, 2, 128)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -1e30])
def test_documents_keep_to_themselves(hq, hk, d, value):
    """Whatever the document in the middle and the padding behind the last one hold, the others' results are the same."""
    lens, pad, window, sinks = [600, 70, 650], 50, 200, 3
    qkv, do, cu = _inputs(hq, hk, d, lens, pad)
    want = _truth(qkv, do, hq, hk, d, lens, window, sinks)
    a, b, T = 600, 670, 1320
    for t in (qkv, do):
        t[a:b] = value
        t[T:] = value
    o, g = _run(qkv, do, cu, hq, hk, d, window, sinks)
    assert (o[T:] == 0).all() and (g[T:] == 0).all()
    for rows in (slice(0, a), slice(b, T)):
        for x, y in ((o, want[0]), (g, want[1])):
            assert torch.isfinite(x[rows]).all() and (x[rows].double() - y[rows]).norm() <= 2.0 ** -7 * y[rows].norm()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bounds", [[0, 100, 5000], [0, 100, 60, 300], [-40, 100, 300], [0, 300, -7], [290, 10, 1 << 30]])
def test_bad_boundaries_reach_no_other_memory(d, bounds):
    """What such a batch gives is not defined; guards around every buffer stay as they are, and the next call is right."""
    T, hq, hk, pad = 300, 2, 1, 256
    qkv, do, cu = _inputs(hq, hk, d, [T], 0)
    want = _run(qkv, do, cu, hq, hk, d, 40, 3)
    nq, n = hq * d, (hq + 2 * hk) * d
    buf = torch.full((pad + T * nq + pad,), 7.0, dtype=BF, device=DEV)
    o = buf[pad:pad + T * nq].view(T, nq)
    lse = torch.full((hq * T + 2 * pad,), 7.0, device=DEV)
    bad = torch.tensor(bounds, dtype=torch.int32, device=DEV)
    st = _ext.status_buffer(qkv.device).data_ptr()
    at = qkv.data_ptr()
    args = (len(bounds) - 1, T, hq, hk, d, n, n, n, nq)
    assert _ext.lib().cb_attn_window_fwd(at, at + 2 * nq, at + 2 * (nq + hk * d), o.data_ptr(), lse.data_ptr() + 4 * pad, bad.data_ptr(), *args,
                                         d ** -0.5, 40, 3, None, st, _ext.stream_ptr()) == 0
    acc = torch.full((pad + hq * T // 4 * 4 + 64 + T * n + pad,), 7.0, device=DEV)
    delta = acc.data_ptr() + 4 * pad
    dq = delta + 4 * (-(-hq * T // 64) * 64)
    g = torch.full((pad + T * n + pad,), 7.0, dtype=BF, device=DEV)
    assert _ext.lib().cb_attn_window_bwd(at, at + 2 * nq, at + 2 * (nq + hk * d), o.data_ptr(), do.data_ptr(), lse.data_ptr() + 4 * pad,
                                         bad.data_ptr(), *args, nq, d ** -0.5, 40, 3, None, delta, dq, dq + 4 * T * nq,
                                         dq + 4 * T * (nq + hk * d), g.data_ptr() + 2 * pad, n, st, _ext.stream_ptr()) == 0
    _ext.check_status()
    for t, m in ((buf, T * nq), (lse, hq * T), (g, T * n)):
        assert (t[:pad] == 7).all() and (t[pad + m:] == 7).all()
    assert (acc[:pad] == 7).all() and (acc[-pad + 64:] == 7).all()
    assert torch.equal(_run(qkv, do, cu, hq, hk, d, 40, 3)[0], want[0])
