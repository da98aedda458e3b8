"""The distillation kernels against the definition in 64 bits."""
import math

import pytest
import torch

from chronicals_b200 import ops
from chronicals_b200.ops import _ext
from test_distillation_cpu import definition, entries

pytestmark = pytest.mark.gpu
DEV = "cuda"
NEG = -math.inf
BF = torch.bfloat16


@pytest.fixture(params=["logits held", "logits formed twice"])
def form(request, monkeypatch):
    """The two forms of the loss from hidden states, whatever the size."""
    if request.param == "logits formed twice":
        monkeypatch.setattr(ops, "_HELD_LOGITS_BYTES", 0)


def _truth(z, idx, lg, tau, labels, up=None):
    z = z.detach().double().requires_grad_()
    rows, valid = definition(z, idx, lg, tau, labels)
    rows = rows.to(DEV)
    return z, rows, valid.to(DEV), max(1, int(valid.sum()))


def _over(off, tol):
    """How many values are further off than they may be."""
    return int((~(off.abs() <= tol)).sum())


def _loss_tolerance(z, tau, extra=0.0):
    # log2 p is z log2(e) / tau less the reference less log2 of the sum: three roundings of numbers of up to |z| log2(e) / tau, and
    # terms of the sum that are 2^-21 off (22 bits of the approximation, the rounded reference)
    return tau * tau * (2.0 ** -20 + (3 * 2.0 ** -24 + extra) * 2 * z.abs().max().item() / tau)


# rows that share a block or take several; odd vocabularies and pitches; more entries than words
@pytest.mark.parametrize("T,V,K,tau", [(1, 7, 1, 1.0), (3, 1000, 9, 2.0), (5, 33, 40, 0.5), (37, 32000, 8, 1.0), (2, 151936, 64, 1.3),
                                       (1200, 257, 33, 3.0), (700, 4099, 5, 1.0)])
@pytest.mark.parametrize("dtype", [torch.float32, BF])
@pytest.mark.parametrize("gap", [0, 5])
def test_held_logits(T, V, K, tau, dtype, gap):
    g = torch.Generator(device=DEV).manual_seed(T + V)
    buf = (torch.randn(T, V + gap, device=DEV, generator=g) * 3).to(dtype)
    z = buf[:, :V].requires_grad_()
    idx, lg = entries(T, V, K, device=DEV)
    labels = torch.arange(T, device=DEV).masked_fill(torch.arange(T, device=DEV) % 4 == 1, -100)
    z64, rows, valid, n = _truth(z, idx, lg, tau, labels)
    loss = ops.distillation_logits(z, idx, lg, tau, labels)
    got = ops.distillation_logits(z, idx, lg, tau, labels, reduction="none")
    assert _over(got - rows, _loss_tolerance(z64, tau) + 2.0 ** -22 * rows.abs()) == 0
    assert abs(loss.item() - rows.sum().item() / n) <= _loss_tolerance(z64, tau) + 2.0 ** -20 * abs(rows.sum().item()) / n
    assert (got[~valid] == 0).all()
    (want,) = torch.autograd.grad(rows.sum() / n, z64)
    (grad,) = torch.autograd.grad(loss, z)
    p = torch.softmax(z64.detach() / tau, 1) * tau / n
    # p from 22 bits and a rounded exponent, then one rounding to the type (and, below its normal range, to zero).  At a word of
    # the teacher's the value is a difference p - q, so that q's own error counts, however small the difference: its exponent
    # t / tau is rounded three times (half a step, 2^-24 of up to |t| / tau, each), its exponential and its sum are 2^-21 off.
    q, t = (p - want).abs(), lg[lg > -50].abs().max().item()
    tol = p * (2.0 ** -20 + 2.0 ** -22 * z64.abs().max().item() / tau) + 2.0 ** -22 * want.abs() + 2.0 ** -126
    tol = tol + q * (2.0 ** -20 + 3 * 2.0 ** -24 * t / tau) + (torch.finfo(dtype).eps / 2 * want.abs() if dtype == BF else 0)
    assert _over(grad.double() - want, tol) == 0
    assert (grad[~valid] == 0).all()
    if gap:
        assert not buf[:, V:].isnan().any()


@pytest.mark.parametrize("T,H,V,K,tau", [(1, 64, 520, 3, 1.0), (130, 256, 4096, 16, 1.0), (300, 896, 5001, 33, 2.0), (257, 128, 32000, 64, 0.7),
                                         (77, 2048, 9000, 5, 1.5), (64, 72, 100, 130, 1.0)])
@pytest.mark.usefixtures("form")
def test_from_hidden_states(T, H, V, K, tau):
    g = torch.Generator(device=DEV).manual_seed(T + H)
    h = torch.randn(T, H, device=DEV, generator=g).to(BF).requires_grad_()
    w = (torch.randn(V, H, device=DEV, generator=g) * 2 / math.sqrt(H)).to(BF).requires_grad_()
    idx, lg = entries(T, V, K, device=DEV)
    labels = torch.arange(T, device=DEV).masked_fill(torch.arange(T, device=DEV) % 4 == 1, -100)
    h64, w64 = h.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    z64 = h64 @ w64.t()
    rows, valid = definition(z64, idx, lg, tau, labels)
    n = max(1, int(valid.sum()))
    loss = ops.linear_distillation(h, w, idx, lg, tau, labels)
    with torch.no_grad():
        got = ops.linear_distillation(h, w, idx, lg, tau, labels, reduction="none")
    # a logit is a sum of H products in 32 bits: 2^-24 of the sum of their sizes, a few times over
    size = (h64.detach().abs() @ w64.detach().abs().t()).max().item()
    tol = _loss_tolerance(z64, tau) + tau * 2.0 ** -20 * size
    assert _over(got - rows.to(DEV), tol) == 0
    assert abs(loss.item() - rows.sum().item() / n) <= tol
    want = torch.autograd.grad(rows.sum().to(DEV) / n, (h64, w64))
    _ext.check_status()
    # d(logits) is rounded to bf16 (half a step, 2^-8) before the products and their results once more: 2^-7 of the norm
    for a, b in zip(torch.autograd.grad(loss, (h, w)), want):
        assert a.dtype == BF and ((a.double() - b).norm() <= 2.0 ** -7 * b.norm() + 1e-12).item(), ((a.double() - b).norm() / b.norm()).item()
    _ext.check_status()


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("linear", [False, True])
@pytest.mark.parametrize("reduction", ["sum", "none", "mean"])
def test_reductions_and_upstream_gradient(linear, reduction):
    T, H, V, K, tau = 40, 64, 600, 6, 1.5
    g = torch.Generator(device=DEV).manual_seed(3)
    h = torch.randn(T, H, device=DEV, generator=g).to(BF).requires_grad_()
    w = (torch.randn(V, H, device=DEV, generator=g) / 8).to(BF).requires_grad_()
    z = torch.randn(T, V, device=DEV, generator=g).requires_grad_()
    idx, lg = entries(T, V, K, device=DEV)
    x = (h, w) if linear else (z,)
    x64 = tuple(t.detach().double().requires_grad_() for t in x)
    rows, valid = definition(x64[0] @ x64[1].t() if linear else x64[0], idx, lg, tau)
    want = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / int(valid.sum())}[reduction].to(DEV)
    op = ops.linear_distillation if linear else ops.distillation_logits
    loss = op(*x, idx, lg, tau, reduction=reduction)
    up = torch.randn(loss.shape, device=DEV, generator=g)
    assert torch.allclose(loss.double(), want, rtol=1e-5, atol=1e-4)
    for a, b in zip(torch.autograd.grad(loss, x, up), torch.autograd.grad(want, x64, up.double())):
        assert (a.double() - b).norm() <= (2.0 ** -7 if linear else 1e-5) * b.norm()


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("linear", [False, True])
@pytest.mark.parametrize("idx_type,lg_type", [(torch.int32, BF), (torch.int16, torch.float16), (torch.int64, torch.float64), (torch.int32, torch.float32)])
def test_types_and_layouts_of_the_teacher(linear, idx_type, lg_type):
    T, H, V, K = 20, 64, 500, 7
    x = ((torch.randn(T, H, device=DEV).to(BF), torch.randn(V, H, device=DEV).to(BF)) if linear else (torch.randn(T, V, device=DEV).to(BF),))
    idx, lg = entries(T, V, K, device=DEV)
    lg = lg.to(lg_type)
    op = ops.linear_distillation if linear else ops.distillation_logits
    want = op(*x, idx, lg.float(), reduction="none")
    assert torch.equal(op(*x, idx.to(idx_type), lg, reduction="none"), want)
    wide = torch.full((T, 3 * K), -5, dtype=idx_type, device=DEV)
    wide[:, K:2 * K] = idx.to(idx_type)
    assert torch.equal(op(*x, wide[:, K:2 * K], lg.t().contiguous().t(), reduction="none"), want)


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("linear", [False, True])
def test_one_index_several_times(linear):
    T, H, V = 9, 64, 300
    g = torch.Generator(device=DEV).manual_seed(5)
    x = (torch.randn(T, H, device=DEV, generator=g).to(BF).requires_grad_(), torch.randn(V, H, device=DEV, generator=g).mul(0.2).to(BF).requires_grad_())
    x = x if linear else (torch.randn(T, V, device=DEV, generator=g).requires_grad_(),)
    op = ops.linear_distillation if linear else ops.distillation_logits
    idx = torch.tensor([[4, 9, 4, 4, 299, 9]], device=DEV).expand(T, 6)
    lg = torch.randn(T, 6, device=DEV, generator=g)
    merged = torch.stack((lg[:, [0, 2, 3]].logsumexp(1), lg[:, [1, 5]].logsumexp(1), lg[:, 4]), 1)
    a, b = op(*x, idx, lg), op(*x, torch.tensor([[4, 9, 299]], device=DEV).expand(T, 3), merged)
    assert abs(a.item() - b.item()) <= 1e-5
    for p, q in zip(torch.autograd.grad(a, x), torch.autograd.grad(b, x)):
        assert (p.double() - q.double()).norm() <= (2.0 ** -8 if linear else 1e-6) * q.double().norm()


# absent by the type's lowest value over a small temperature, by -inf, by an index outside; a row of the lowest values alone
@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("linear", [False, True])
def test_masked_entries(linear):
    T, H, V, K, tau = 6, 64, 400, 5, 0.5
    low = torch.finfo(torch.float32).min
    g = torch.Generator(device=DEV).manual_seed(8)
    x = (torch.randn(T, H, device=DEV, generator=g).to(BF).requires_grad_(), torch.randn(V, H, device=DEV, generator=g).mul(0.2).to(BF).requires_grad_())
    x = x if linear else (torch.randn(T, V, device=DEV, generator=g).requires_grad_(),)
    op = ops.linear_distillation if linear else ops.distillation_logits
    idx = torch.randint(0, V, (T, K), device=DEV, generator=g)
    idx[:, 0] = torch.arange(T, device=DEV)
    lg = torch.randn(T, K, device=DEV, generator=g)
    lg[0, 1], lg[1, 1], idx[2, 1], lg[2, 1], idx[3, 1], lg[3, 1] = low, NEG, -1, math.nan, V, math.inf
    lg[4] = low                                                       # over the temperature: -inf, the row takes no part
    keep = torch.ones(T, K, dtype=torch.bool, device=DEV)
    keep[torch.arange(4), 1] = False
    loss = op(*x, idx, lg, tau)
    rows = op(*x, idx, lg, tau, reduction="none")
    clean = op(*x, torch.where(keep, idx, -1), torch.where(keep, lg, 0.0), tau, torch.where(torch.arange(T, device=DEV) == 4, -100, 0))
    assert rows[4].item() == 0 and math.isfinite(loss.item()) and abs(loss.item() - clean.item()) <= 1e-6
    for p, q in zip(torch.autograd.grad(loss, x), torch.autograd.grad(clean, x)):
        assert torch.equal(p, q)
    same = op(*x, idx, torch.full_like(lg, low), 1.0, reduction="none")     # at a temperature of 1 they are equal entries
    assert torch.allclose(same, op(*x, idx, torch.zeros_like(lg), 1.0, reduction="none"))


@pytest.mark.usefixtures("form")
def test_rows_that_take_no_part_are_not_read():
    z = torch.full((4, 1000), math.nan, device=DEV)
    z[0] = 1.0
    z.requires_grad_()
    loss = ops.distillation_logits(z, torch.zeros(4, 2, dtype=torch.int64, device=DEV), torch.zeros(4, 2, device=DEV), 1.0,
                                   torch.tensor([0, -100, -100, -100], device=DEV))
    assert abs(loss.item() - math.log(1000.0)) < 1e-5
    grad = torch.autograd.grad(loss, z)[0]
    assert torch.isfinite(grad).all() and (grad[1:] == 0).all()


@pytest.mark.usefixtures("form")
def test_nothing_takes_part():
    z = torch.randn(3, 700, device=DEV, requires_grad=True)
    h, w = torch.randn(3, 64, device=DEV).to(BF).requires_grad_(), torch.randn(700, 64, device=DEV).to(BF).requires_grad_()
    idx, lg = torch.full((3, 2), -1, device=DEV), torch.zeros(3, 2, device=DEV)
    for loss, x in ((ops.distillation_logits(z, idx, lg), (z,)), (ops.linear_distillation(h, w, idx, lg), (h, w))):
        assert loss.item() == 0 and all(t.abs().max() == 0 for t in torch.autograd.grad(loss, x))
    assert ops.distillation_logits(z[:0], idx[:0], lg[:0]).item() == 0
    assert ops.linear_distillation(h[:0], w, idx[:0], lg[:0]).item() == 0


def test_student_logits_of_minus_infinity():
    z = torch.randn(2, 5000, device=DEV)
    z[:, 7:4000] = NEG
    z.requires_grad_()
    idx = torch.tensor([[0, 1], [2, 7]], device=DEV)
    rows = ops.distillation_logits(z, idx, torch.zeros(2, 2, device=DEV), reduction="none")
    want, _ = definition(z.detach().cpu(), idx.cpu(), torch.zeros(2, 2))
    assert abs(rows[0].item() - want[0].item()) < 1e-5 and rows[1].item() == math.inf
    assert torch.isfinite(torch.autograd.grad(rows[0], z)[0]).all()


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("linear", [False, True])
def test_the_same_bits_every_time(linear):
    T, H, V, K = 500, 256, 20000, 32
    x = (torch.randn(T, H, device=DEV).to(BF).requires_grad_(), torch.randn(V, H, device=DEV).mul(0.1).to(BF).requires_grad_())
    x = x if linear else (torch.randn(T, V, device=DEV).to(BF).requires_grad_(),)
    op = ops.linear_distillation if linear else ops.distillation_logits
    idx, lg = entries(T, V, K, device=DEV)
    first = None
    for _ in range(3):
        loss = op(*x, idx, lg, 2.0)
        now = (loss, *torch.autograd.grad(loss, x))
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("linear", [False, True])
def test_captured_and_replayed(linear):
    T, H, V, K = 90, 64, 3000, 8
    x = (torch.randn(T, H, device=DEV).to(BF).requires_grad_(), torch.randn(V, H, device=DEV).mul(0.2).to(BF).requires_grad_())
    x = x if linear else (torch.randn(T, V, device=DEV).to(BF).requires_grad_(),)
    op = ops.linear_distillation if linear else ops.distillation_logits
    idx, lg = entries(T, V, K, device=DEV)

    def step():
        loss = op(*x, idx, lg, 2.0)
        return (loss.detach(), *torch.autograd.grad(loss, x))
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    lg.copy_(torch.randn_like(lg))
    g.replay()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_logits_beyond_32_bits_of_offset():
    V, T = 151936, 14200                                              # 2^31 values lie before row 14135
    z = torch.zeros(T, V, dtype=BF, device=DEV)
    z[-2:] = torch.randn(2, V, device=DEV).to(BF)
    z.requires_grad_()
    idx = torch.full((T, 3), -1, device=DEV)
    idx[-2:] = torch.tensor([[5, 151935, 70000], [0, 1, 2]], device=DEV)
    lg = torch.randn(T, 3, device=DEV)
    loss = ops.distillation_logits(z, idx, lg)
    grad = torch.autograd.grad(loss, z)[0][-2:].double()
    z64 = z[-2:].detach().double().requires_grad_()
    rows, _ = definition(z64, idx[-2:], lg[-2:])
    (want,) = torch.autograd.grad(rows.mean(), z64)
    assert abs(loss.item() - rows.mean().item()) < 1e-5
    assert (grad - want).norm() <= torch.finfo(BF).eps / 2 * want.norm()


def test_entry_points_refuse_bad_sizes():
    L, z = _ext.lib(), torch.zeros(2, 16, device=DEV)
    idx = torch.zeros(2, 2, dtype=torch.int64, device=DEV)
    f = torch.zeros(64, device=DEV)

    def call(rows=2, V=16, K=2, tau=1.0):
        return L.cb_kd_logits(z.data_ptr(), rows, 16, V, 0, idx.data_ptr(), 2, 1, f.data_ptr(), 2, 0, K, None, -100, tau, 1, f.data_ptr(),
                              f.data_ptr(), f.data_ptr(), f.data_ptr(), f.data_ptr(), _ext.stream_ptr())
    assert call(rows=0) == call(V=0) == call(K=0) == call(K=L.cb_kd_max_entries() + 1) == call(tau=0.0) == call(tau=math.nan) == -1


def test_more_entries_than_the_kernels_take_follow_the_formula():
    K = _ext.lib().cb_kd_max_entries() + 1
    z = torch.randn(2, 6000, device=DEV, requires_grad=True)
    idx, lg = torch.arange(K, device=DEV).expand(2, K), torch.randn(2, K, device=DEV)
    loss = ops.distillation_logits(z, idx, lg)
    short = ops.distillation_logits(z, idx[:, :-1], lg[:, :-1].masked_fill(idx[:, :-1] == 0, NEG))
    assert math.isfinite(loss.item()) and math.isfinite(short.item()) and abs(loss.item() - short.item()) < 0.1


@pytest.mark.parametrize("M,N,K,n", [(1, 64, 4096, 7), (120, 256, 5000, 13), (129, 72, 640, 3), (300, 896, 1000, 16), (5, 8, 64, 1)])
def test_product_in_slabs(M, N, K, n):
    """Ranges of the inner dimension in slabs of their own, a second product over a shorter one added, summed in order."""
    g = torch.Generator(device=DEV).manual_seed(M + K)
    L, S = _ext.lib(), _ext.status_buffer(torch.device("cuda", torch.cuda.current_device())).data_ptr()
    slabs = torch.full((n, -(-M // 128) * 128, N), math.nan, device=DEV)
    out = torch.full((M, N), math.nan, dtype=BF, device=DEV)
    want = torch.zeros(M, N, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(want)
    for add, k in ((0, K), (1, K), (1, max(8, K // 3 // 8 * 8))):
        a, b = (torch.randn(*s, device=DEV, generator=g).to(BF) for s in ((M, -(-k // 8) * 8), (k, N)))
        code = L.cb_gemm_bf16_slabs(a.data_ptr(), b.data_ptr(), slabs.data_ptr(), M, N, k, a.stride(0), N, 0, 1, n, add, S, _ext.stream_ptr())
        per = -(-(-(-k // 64)) // n)
        if not add and -(-(-(-k // 64)) // per) != n:                 # blocks of 64 that leave a slab without any are refused
            assert code == -1
            return
        assert code == 0
        want += a[:, :k].double() @ b.double()
        size += a[:, :k].double().abs() @ b.double().abs()
    assert L.cb_slab_sum(slabs.data_ptr(), out.data_ptr(), M, N, n, 0, None, _ext.stream_ptr()) == 0
    _ext.check_status()
    # the sums in 32 bits, a few roundings of the sum of sizes (n slabs of at least 64 products in one accumulator); then half a step
    assert _over(out.double() - want, torch.finfo(BF).eps / 2 * want.abs() + 2.0 ** -20 * size + 1e-12) == 0


def test_slabs_only_where_tiles_are_few():
    L = _ext.lib()
    assert L.cb_gemm_slabs(120, 256, 32000, 0, 1, 148) > 8 and L.cb_gemm_slabs(8192, 896, 8192, 0, 1, 148) == 1
    for M in (1, 100, 500, 1021, 3000):
        for K in (64, 1000, 32000, 151936):
            n = L.cb_gemm_slabs(M, 896, K, 0, 1, 148)
            per = -(-(-(-K // 64)) // n)
            assert 1 <= n <= 96 and -(-(-(-K // 64)) // per) == n    # every slab of the first product is written
    assert L.cb_gemm_bf16_slabs(None, None, None, 0, 8, 8, 8, 8, 0, 1, 1, 0, None, None) == -1
    assert L.cb_gemm_bf16_slabs(None, None, None, 8, 6, 8, 8, 8, 0, 1, 1, 0, None, None) == -1
    assert L.cb_slab_sum(None, None, 8, 6, 1, 0, None, None) == -1


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("linear", [False, True])
def test_loss_may_be_changed_in_place_before_the_backward_pass(linear):
    T, H, V, K = 30, 64, 500, 4
    x = (torch.randn(T, H, device=DEV).to(BF).requires_grad_(), torch.randn(V, H, device=DEV).mul(0.2).to(BF).requires_grad_())
    x = x if linear else (torch.randn(T, V, device=DEV).requires_grad_(),)
    op = ops.linear_distillation if linear else ops.distillation_logits
    idx, lg = entries(T, V, K, device=DEV)
    want = torch.autograd.grad(op(*x, idx, lg) * 0.5, x)
    loss = op(*x, idx, lg)
    loss.mul_(0.5)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(loss, x), want))


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("T,masked", [(700, [(0, 300)]), (700, [(128, 384), (600, 700)]), (513, [(0, 512)]), (256, [(0, 256)]), (384, [(5, 380)])])
def test_blocks_of_rows_that_take_no_part(T, masked):
    """Whole blocks of 128 masked rows are left out of the products, mixed ones are not; large logits in masked rows do no harm."""
    H, V, K, tau = 128, 3000, 6, 1.5
    g = torch.Generator(device=DEV).manual_seed(T)
    h = torch.randn(T, H, device=DEV, generator=g).to(BF)
    labels = torch.zeros(T, dtype=torch.int64, device=DEV)
    for a, b in masked:
        labels[a:b] = -100
        h[a:b] *= 100
    h.requires_grad_()
    w = (torch.randn(V, H, device=DEV, generator=g) / 8).to(BF).requires_grad_()
    idx, lg = entries(T, V, K, device=DEV)
    h64, w64 = h.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    rows, valid = definition(h64 @ w64.t(), idx, lg, tau, labels)
    want = torch.autograd.grad(rows.sum() / max(1, int(valid.sum())), (h64, w64))
    loss = ops.linear_distillation(h, w, idx, lg, tau, labels)
    assert abs(loss.item() - rows.sum().item() / max(1, int(valid.sum()))) <= 1e-4
    got = torch.autograd.grad(loss, (h, w))
    _ext.check_status()
    for a, b in zip(got, want):
        assert ((a.double() - b).norm() <= 2.0 ** -7 * b.norm()).item()
    assert (got[0][labels == -100] == 0).all()


@pytest.mark.parametrize("T,V", [(1, 4096), (7, 5001), (64, 3000), (65, 3000)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_gradients_of_few_tokens_are_rounded_once(T, V, reduction):
    """Up to 64 tokens d(logits) keeps what its rounding left out: the gradients are half a step of bf16 off, value by value."""
    H, K, tau = 512, 9, 1.3
    g = torch.Generator(device=DEV).manual_seed(T)
    h = torch.randn(T, H, device=DEV, generator=g).to(BF).requires_grad_()
    w = (torch.randn(V, H, device=DEV, generator=g) / 12).to(BF).requires_grad_()
    idx, lg = entries(T, V, K, device=DEV)
    h64, w64 = h.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    rows, valid = definition(h64 @ w64.t(), idx, lg, tau)
    up = torch.rand(T, device=DEV, generator=g) if reduction == "none" else torch.tensor(0.7, device=DEV)
    want = torch.autograd.grad(rows.to(DEV) if reduction == "none" else rows.sum().to(DEV) / int(valid.sum()), (h64, w64), up.double())
    got = torch.autograd.grad(ops.linear_distillation(h, w, idx, lg, tau, reduction=reduction), (h, w), up)
    _ext.check_status()
    with torch.no_grad():
        # sizes that cancel in the sums: |d(logits)| |W| and |d(logits)|^T |H|, at most the softmax's and the teacher's part apart
        p = torch.softmax(h64 @ w64.t() / tau, 1)
        q = torch.zeros_like(p).scatter_add_(1, idx.clamp(0, V - 1), torch.softmax(lg.double().masked_fill((idx < 0) | (idx >= V), -1e9) / tau, 1))
        scale = tau * (up.double()[:, None] if reduction == "none" else up.double() / int(valid.sum()))
        size = ((p + q) * scale) @ w64.abs(), ((p + q) * scale).t() @ h64.abs()
    for a, b, c in zip(got, want, size):
        if T <= 64:                                    # two bf16 numbers leave 2^-16 of d(logits), p and q are 2^-19 off
            assert _over(a.double() - b, torch.finfo(BF).eps / 2 * b.abs() + 2.0 ** -15 * c) == 0
        assert (a.double() - b).norm() <= 2.0 ** -7 * b.norm()


@pytest.mark.usefixtures("form")
@pytest.mark.parametrize("T,V,H", [(151, 20000, 64), (302, 5000, 256), (605, 20000, 128)])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_the_factor_of_the_gradient_is_not_rounded(T, V, H, reduction):
    """One word a row: d(logits) is close to the same number in every row, and its rounding would scale the whole gradient.  121 rows
    (or 242, 484) take part: 1 / 121 is 2^-8.4 of itself off in bf16."""
    g = torch.Generator(device=DEV).manual_seed(V)
    h = torch.randn(T, H, device=DEV, generator=g).to(BF).requires_grad_()
    w = (torch.randn(V, H, device=DEV, generator=g) / (8 * math.sqrt(H))).to(BF).requires_grad_()
    idx, lg = torch.randint(0, V, (T, 1), device=DEV, generator=g), torch.zeros(T, 1, device=DEV)
    labels = torch.where(torch.arange(T, device=DEV) < T // 5, -100, 0)
    n = int((labels != -100).sum())
    assert n % 121 == 0
    h64, w64 = h.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    rows, _ = definition(h64 @ w64.t(), idx, lg, 1.0, labels)
    want = torch.autograd.grad(rows.sum() / n, (h64, w64))
    loss = ops.linear_distillation(h, w, idx, lg, 1.0, labels, reduction=reduction)
    got = torch.autograd.grad(loss if reduction == "mean" else loss * (1.0 / n), (h, w))
    _ext.check_status()
    p = torch.softmax(h64 @ w64.t(), 1).max().item()
    for a, b in zip(got, want):
        # 1 - p is rounded to 1 or to the number below it: p off, or half a step of 2^-8.  The results' roundings, d at most 2^-8 each, are
        # as often up as down: the sum of b^2 d over that of b^2 has a deviation of at most 2^-8 sqrt(sum b^4) / sum b^2.  (Few values
        # carry the weight's gradient: the rows of the words.)
        off = abs(((a.double() * b).sum() / (b * b).sum()).item() - 1)
        assert off <= min(p, 2.0 ** -9) + 6 * 2.0 ** -8 * (b ** 4).sum().sqrt().item() / (b * b).sum().item(), off
        assert (a.double() - b).norm() <= 2.0 ** -8 * b.norm()
