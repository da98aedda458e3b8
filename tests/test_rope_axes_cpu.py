"""Rotary positions with several axes: the formula in 64 bits, its gradient, and what is refused."""
import pytest
import torch

from chronicals_b200 import ops
from chronicals_b200.ops import ref


def turned(x, cos, sin, pos, axes, heads, d, pairs, inverse=False):
    """Each pair of each of the first ``heads`` heads as a complex number times the unit number of its axis's position."""
    T = x.shape[0]
    rows = pos.clamp(0, cos.shape[0] - 1)
    turn = torch.stack([torch.complex(cos[rows[a], f].double(), sin[rows[a], f].double()) for f, a in enumerate(axes)], 1)[:, None]
    turn = turn.conj() if inverse else turn
    y = x.double().reshape(T, -1, d)
    h = y[:, :heads]
    z = torch.complex(h[..., 0::2], h[..., 1::2]) if pairs else torch.complex(h[..., : d // 2], h[..., d // 2:])
    z = z * turn
    h = torch.stack((z.real, z.imag), -1).flatten(-2) if pairs else torch.cat((z.real, z.imag), -1)
    return torch.cat((h, y[:, heads:]), 1).reshape(T, -1)


AXES = {((2, 3, 3), False): (0, 0, 1, 1, 1, 2, 2, 2), ((4, 2, 2), True): (0, 1, 2, 0, 1, 2, 0, 0), ((8,), False): (0,) * 8,
        ((4, 4), True): (0, 1) * 4, ((0, 8), False): (1,) * 8, ((2, 2, 2, 2), True): (0, 1, 2, 3) * 2}


@pytest.mark.parametrize("sections,cyclic", list(AXES))
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_formula(sections, cyclic, pairs, inverse):
    T, hq, hk, d = 7, 3, 1, 16
    g = torch.Generator().manual_seed(len(sections))
    x = torch.randn(T, (hq + 2 * hk) * d, generator=g, dtype=torch.float32)
    cos, sin = ref.rope_cache(40, d, 1e4)
    pos = torch.randint(0, 40, (len(sections), T), generator=g)
    got = ops.qk_rope_axes_(x.clone(), cos, sin, pos, hq, hk, d, sections, cyclic=cyclic, interleaved=pairs, inverse=inverse)
    want = turned(x, cos, sin, pos, AXES[sections, cyclic], hq + hk, d, pairs, inverse)
    # two products and a sum in 32 bits, each off by at most 2^-24 of a magnitude below |x1| + |x2|
    assert (got.double() - want).abs().max() <= 4 * 2.0 ** -24 * 2 * x.abs().max()
    assert torch.equal(got[:, (hq + hk) * d:], x[:, (hq + hk) * d:])


def test_equal_axes_are_the_rotation_of_one_axis():
    T, hq, hk, d = 9, 2, 2, 32
    x = torch.randn(T, (hq + 2 * hk) * d)
    cos, sin = ref.rope_cache(64, d, 1e6)
    pos = torch.randint(0, 64, (T,))
    got = ops.qk_rope_axes_(x.clone(), cos, sin, pos.expand(3, T), hq, hk, d, (4, 6, 6))
    assert torch.equal(got, ops.qk_rope_(x.clone(), cos, sin, pos, hq, hk, d))


def test_gradient_against_differences():
    T, hq, hk, d = 3, 1, 1, 16
    cos, sin = (t.double() for t in ref.rope_cache(16, d, 1e2))
    pos = torch.tensor([[0, 3, 15], [1, 1, 1], [7, 0, 2]])
    x = torch.randn(T, 3 * d, dtype=torch.float32, requires_grad=True)
    w = torch.randn(T, 3 * d)
    (ops.qk_rope_axes_(x, cos, sin, pos, hq, hk, d, (2, 3, 3)) * w).sum().backward()
    back = turned(w, cos, sin, pos, AXES[(2, 3, 3), False], hq + hk, d, False, inverse=True)
    assert torch.allclose(x.grad.double(), back, atol=1e-5)
    f = lambda v: (turned(v, cos, sin, pos, AXES[(2, 3, 3), False], hq + hk, d, False) * w).sum()  # noqa: E731
    for at in [(0, 0), (1, 9), (2, 17), (2, 30), (1, 40)]:
        e = torch.zeros(T, 3 * d, dtype=torch.float64)
        e[at] = 1e-4                                                  # the function is linear: the difference is exact
        diff = (f(x.detach().double() + e) - f(x.detach().double() - e)) / 2e-4
        assert abs(diff - x.grad[at].double()) < 1e-5


@pytest.mark.parametrize("kw,what", [
    (dict(sections=(2, 3)), "sections"), (dict(sections=()), "sections"), (dict(sections=(-1, 9)), "sections"),
    (dict(sections=(2, 2, 2, 1, 1)), "sections"), (dict(sections=(2, 3, 3), cyclic=True), "in turn"), (dict(axes=2), "position_ids"),
    (dict(tokens=6), "position_ids"), (dict(pos_dtype=torch.float32), "position_ids"), (dict(pos_dtype=torch.bool), "position_ids"),
    (dict(half=7), "tables"), (dict(rows=0), "tables"), (dict(heads=4), "qkv"), (dict(three=True), "qkv")])
def test_refusals(kw, what):
    T, hq, hk, d = 5, 2, 1, 16
    x = torch.randn(T, (hq + 2 * hk) * d)
    cos = torch.ones(kw.get("rows", 8), kw.get("half", 8))
    sections = kw.get("sections", (2, 3, 3))
    pos = torch.zeros(kw.get("axes", len(sections)), kw.get("tokens", T), dtype=kw.get("pos_dtype", torch.int64))
    x = x[None] if kw.get("three") else x
    with pytest.raises(ValueError, match=what):
        ops.qk_rope_axes_(x, cos, cos, pos, kw.get("heads", hq), hk, d, sections, cyclic=kw.get("cyclic", False))
