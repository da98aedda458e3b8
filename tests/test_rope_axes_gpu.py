"""The rotary kernel for several axes against the formula in 64 bits."""
import pytest
import torch

from chronicals_b200 import ops
from chronicals_b200.ops import _ext, ref
from test_rope_axes_cpu import turned

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF_STEP = torch.finfo(torch.bfloat16).eps / 2


def _inputs(T, hq, hk, d, axes, seed=0, gap=0, span=500):
    g = torch.Generator(device=DEV).manual_seed(seed + T)
    x = torch.randn(T, (hq + 2 * hk) * d + gap, device=DEV, generator=g).to(torch.bfloat16)[:, : (hq + 2 * hk) * d]
    cos, sin = ref.rope_cache(span, d, 1e6, device=DEV)
    return x, cos, sin, torch.randint(0, span, (axes, T), device=DEV, generator=g)


def _check(got, want):
    # one rounding to bf16, half a step of the value; the 32-bit products before it add far less: 2^-22 of the pair's size
    off = (got.double() - want).abs()
    assert (off <= HALF_STEP * want.abs() + 2.0 ** -20 * want.abs().max()).all(), off.max().item()


# one token, more than a block's, an odd number; heads that leave lanes idle (d = 48: 3 lanes a head), several passes a token
@pytest.mark.parametrize("T,hq,hk,d,sections,cyclic", [
    (1, 1, 1, 64, (8, 12, 12), False), (9, 14, 2, 64, (12, 10, 10), True), (1000, 28, 4, 128, (16, 24, 24), False),
    (257, 28, 4, 128, (24, 20, 20), True), (33, 5, 5, 48, (8, 8, 8), False), (33, 3, 1, 48, (12, 12), True), (17, 1, 1, 16, (2, 3, 3), False),
    (40, 2, 1, 512, (64, 64, 64, 64), True), (40, 2, 1, 512, (1, 200, 55), False), (70, 40, 8, 128, (64,), False), (6, 4, 0, 64, (0, 32), False)])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
def test_kernel(T, hq, hk, d, sections, cyclic, pairs, inverse):
    x, cos, sin, pos = _inputs(T, hq, hk, d, len(sections), gap=8)
    axes = ref.rope_axis_map(sections, cyclic)
    want = turned(x, cos, sin, pos, axes, hq + hk, d, pairs, inverse)
    rest = x[:, (hq + hk) * d:].clone()
    got = ops.qk_rope_axes_(x, cos, sin, pos, hq, hk, d, sections, cyclic=cyclic, interleaved=pairs, inverse=inverse)
    assert got.data_ptr() == x.data_ptr()
    _check(got, want)
    assert torch.equal(got[:, (hq + hk) * d:], rest)


def test_gap_between_rows_is_left_alone():
    T, hq, hk, d = 21, 3, 1, 64
    buf = torch.full((T, (hq + 2 * hk) * d + 40), 7.0, dtype=torch.bfloat16, device=DEV)
    _, cos, sin, pos = _inputs(T, hq, hk, d, 3)
    ops.qk_rope_axes_(buf[:, : (hq + 2 * hk) * d], cos, sin, pos, hq, hk, d, (8, 12, 12))
    assert (buf[:, (hq + hk) * d:] == 7).all() and not (buf[:, : (hq + hk) * d] == 7).all()


def test_positions_outside_the_tables_use_the_first_or_last_row():
    x, cos, sin, pos = _inputs(50, 2, 1, 64, 3, span=20)
    pos = pos * 3 - 20
    want = turned(x, cos, sin, pos, ref.rope_axis_map((8, 12, 12)), 3, 64, False)
    _check(ops.qk_rope_axes_(x, cos, sin, pos, 2, 1, 64, (8, 12, 12)), want)


@pytest.mark.parametrize("kind", ["int32", "expanded", "transposed"])
def test_position_layouts(kind):
    T = 100
    x, cos, sin, pos = _inputs(T, 2, 1, 64, 3)
    if kind == "expanded":
        pos = pos[:1].expand(3, T)
    want = turned(x, cos, sin, pos, ref.rope_axis_map((8, 12, 12)), 3, 64, False)
    given = {"int32": pos.int(), "expanded": pos, "transposed": pos.t().contiguous().t()}[kind]
    _check(ops.qk_rope_axes_(x, cos, sin, given, 2, 1, 64, (8, 12, 12)), want)


@pytest.mark.parametrize("shape", ["unaligned rows", "float32"])
def test_what_the_kernel_does_not_take_follows_the_formula(shape):
    T, hq, hk, d = 13, 2, 1, 64
    x, cos, sin, pos = _inputs(T, hq, hk, d, 3)
    if shape == "float32":
        x = x.float()
    else:
        x = torch.empty(T, x.shape[1] + 3, dtype=x.dtype, device=DEV)[:, : x.shape[1]].copy_(x)
    want = turned(x, cos, sin, pos, ref.rope_axis_map((8, 12, 12)), hq + hk, d, False)
    _check(ops.qk_rope_axes_(x, cos, sin, pos, hq, hk, d, (8, 12, 12)), want)


@pytest.mark.parametrize("pairs", [False, True])
def test_gradient_leaves_the_incoming_one_as_it_is(pairs):
    T, hq, hk, d, sec = 130, 14, 2, 64, (8, 12, 12)
    x, cos, sin, pos = _inputs(T, hq, hk, d, 3)
    x = x.contiguous().requires_grad_()
    w = torch.randn(T, x.shape[1], device=DEV).to(torch.bfloat16)
    keep = w.clone()
    other = torch.zeros_like(x, requires_grad=True)
    y = ops.qk_rope_axes_(x * 1.0, cos, sin, pos, hq, hk, d, sec, interleaved=pairs)
    (y + other).backward(w)                                           # the same gradient goes to both branches
    assert torch.equal(w, keep) and torch.equal(other.grad, keep)
    _check(x.grad, turned(w, cos, sin, pos, ref.rope_axis_map(sec), hq + hk, d, pairs, inverse=True))


def test_gradient_and_tables_off_the_16_byte_boundary():
    T, hq, hk, d, sections = 13, 2, 1, 64, (8, 12, 12)
    x, cos, sin, pos = _inputs(T, hq, hk, d, 3)
    axes = ref.rope_axis_map(sections)
    up = torch.randn(x.numel() + 3, device=DEV).to(torch.bfloat16)
    wide = torch.empty(2, cos.numel() + 1, device=DEV)[:, 1:]
    c, s = (w.copy_(t.flatten()).view_as(t) for w, t in zip(wide, (cos, sin)))
    assert c.data_ptr() % 16 and up[3:].data_ptr() % 16
    leaf = x.clone().requires_grad_()
    y = ops.qk_rope_axes_(leaf * 1, c, s, pos, hq, hk, d, sections)
    _check(y.detach(), turned(x, cos, sin, pos, axes, hq + hk, d, False))
    # the gradient that reaches the node starts six bytes into that of the larger buffer
    (g,) = torch.autograd.grad(torch.cat((x.new_zeros(3), y.flatten())), leaf, up)
    want = turned(up[3:].view_as(x), cos, sin, pos, axes, hq + hk, d, False, True)
    _check(g, want)


def test_leaf_in_place_is_refused():
    x, cos, sin, pos = _inputs(4, 1, 1, 64, 1)
    with pytest.raises(RuntimeError):
        ops.qk_rope_axes_(x.contiguous().requires_grad_(), cos, sin, pos, 1, 1, 64, (32,))


def test_no_tokens():
    x, cos, sin, pos = _inputs(0, 2, 1, 64, 3)
    assert ops.qk_rope_axes_(x, cos, sin, pos, 2, 1, 64, (8, 12, 12)).shape == (0, 256)


def test_rows_beyond_32_bits_of_offset():
    """The last rows of a buffer of more than 2^31 values."""
    T, hq, hk, d = (1 << 31) // 4096 + 3, 28, 2, 128
    buf = torch.zeros(T, 4096, dtype=torch.bfloat16, device=DEV)
    x, cos, sin, pos = _inputs(T, 1, 1, 16, 1, span=300)
    _, cos, sin, _ = _inputs(1, 1, 1, d, 1, span=300)
    buf[-2:] = torch.randn(2, 4096, device=DEV).to(torch.bfloat16)
    want = turned(buf[-2:], cos, sin, pos[:, -2:], (0,) * 64, hq + hk, d, False)
    _check(ops.qk_rope_axes_(buf, cos, sin, pos, hq, hk, d, (64,))[-2:], want)


def test_captured_and_replayed_on_a_side_stream():
    x, cos, sin, pos = _inputs(300, 14, 2, 64, 3)
    want = turned(x, cos, sin, pos, ref.rope_axis_map((8, 12, 12)), 16, 64, False)
    buf = x.clone()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=s):
        ops.qk_rope_axes_(buf, cos, sin, pos, 14, 2, 64, (8, 12, 12))
    for _ in range(2):
        buf.copy_(x)
        g.replay()
        torch.cuda.synchronize()
        _check(buf, want)


def test_entry_point_refuses_what_the_kernel_cannot_address():
    x, cos, sin, pos = _inputs(4, 2, 1, 64, 3)
    words = ops._rope_axis_words((8, 12, 12), False)
    import ctypes

    def call(d=64, n=3, ld=x.stride(0), shift=0, rows=cos.shape[0]):
        return _ext.lib().cb_qk_rope_axes(x.data_ptr() + shift, x.data_ptr() + shift, cos.data_ptr(), sin.data_ptr(), pos.data_ptr(),
                                          pos.stride(0), n, 2, 3, 0, d, ld, ld, ctypes.addressof(words), 0, 0, rows, _ext.stream_ptr())
    assert call(d=40) == call(n=0) == call(n=5) == call(ld=x.stride(0) + 1) == call(shift=2) == call(rows=0) == -1
