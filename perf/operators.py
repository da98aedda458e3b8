"""Windowed attention, rotary positions with several axes and distillation losses as cases that can be timed and compared.

Each case is one pass through one operator of ``chronicals_b200.ops``:

* ``attention``: causal attention of packed documents in which a query sees the last ``window`` tokens of its document, its own
  among them, and the document's first ``sinks`` tokens; forward and backward, or the forward pass alone;
* ``rope``: rotary positions with several axes on the Q and K heads of a packed QKV buffer, in place, or their inverse (which is
  what the backward pass does to the gradient);
* ``kd_logits``: the distillation loss against a teacher's top logits on student logits that a program holds, and their gradient;
* ``kd_linear``: the same loss from hidden states and the output weight, and the gradients of both.

Head layouts, hidden sizes and vocabularies are those of the package's architecture presets.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
BF = torch.bfloat16
IGNORE = -100
HEADS = ((4, 2, 64), (14, 2, 64), (32, 8, 64), (24, 24, 64), (12, 2, 128), (28, 4, 128))
SECTIONS = {(64, False): (8, 12, 12), (128, False): (16, 24, 24), (64, True): (12, 10, 10), (128, True): (24, 20, 20)}


def listed():
    return [
        # the smallest call: one short prompt through a tiny model's heads; launches and latency
        {"name": "attn_tiny", "kind": "attention", "hq": 4, "hk": 2, "d": 64, "T": 77, "pad": 0, "docs": 1, "mix": 0, "window": 32,
         "sinks": 4, "grad": True},
        # a micro-batch of ragged packed documents with padding behind them, heads of the 0.5B model
        {"name": "attn_docs_0.5b", "kind": "attention", "hq": 14, "hk": 2, "d": 64, "T": 8192, "pad": 61, "docs": 9, "mix": 1,
         "window": 1024, "sinks": 4, "grad": True},
        # one long document, 28 / 4 heads of 128: long-context fine-tuning of a 7B model
        {"name": "attn_long_7b", "kind": "attention", "hq": 28, "hk": 4, "d": 128, "T": 8192, "pad": 0, "docs": 1, "mix": 2,
         "window": 2048, "sinks": 8, "grad": True},
        # scoring a very long document without gradients
        {"name": "attn_eval_32k", "kind": "attention", "hq": 14, "hk": 2, "d": 64, "T": 32768, "pad": 0, "docs": 1, "mix": 3,
         "window": 4096, "sinks": 0, "grad": False},
        # positions of one small image between two lines of text
        {"name": "rope_tiny", "kind": "rope", "hq": 4, "hk": 2, "d": 64, "T": 97, "pairs": False, "cyclic": False, "inverse": False},
        # a micro-batch of images and text, heads of the 0.5B model
        {"name": "rope_0.5b", "kind": "rope", "hq": 14, "hk": 2, "d": 64, "T": 8192, "pairs": False, "cyclic": False, "inverse": False},
        # the gradient of a long video, 28 / 4 heads of 128, frequencies dealt to the axes in turn
        {"name": "rope_video_7b", "kind": "rope", "hq": 28, "hk": 4, "d": 128, "T": 32768, "pairs": False, "cyclic": True, "inverse": True},
        # a few tokens of a small vocabulary, fp32 logits
        {"name": "kd_logits_tiny", "kind": "kd_logits", "T": 37, "V": 32000, "K": 8, "fp32": True, "temperature": 1.0},
        # logits of a micro-batch over the full vocabulary
        {"name": "kd_logits_bf16", "kind": "kd_logits", "T": 4095, "V": 151936, "K": 64, "fp32": False, "temperature": 2.0},
        # one short answer of a tiny student
        {"name": "kd_linear_tiny", "kind": "kd_linear", "T": 120, "H": 256, "V": 32000, "K": 16, "temperature": 1.0},
        # a packed micro-batch with an odd number of tokens
        {"name": "kd_linear_1k", "kind": "kd_linear", "T": 1021, "H": 896, "V": 151936, "K": 32, "temperature": 2.0},
        # the head of a 0.5B student, 8 x 1024 tokens
        {"name": "kd_linear_0.5b", "kind": "kd_linear", "T": 8192, "H": 896, "V": 151936, "K": 64, "temperature": 1.5},
    ]


# ------------------------------------------------------------------------------------------------ drawn cases
def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_one(rng):
    kind = rng.choice(["attention", "attention", "rope", "kd_logits", "kd_linear"])
    hq, hk, d = rng.choice(HEADS)
    if kind == "attention":
        T = _log(rng, 1, 16384)
        return {"kind": kind, "hq": hq, "hk": hk, "d": d, "T": T, "pad": rng.choice([0, 0, rng.randint(1, 200)]),
                "docs": min(T, rng.choice([1, 1, 2, 5, 16, 40])), "mix": rng.randint(0, 999), "window": _log(rng, 1, 4096),
                "sinks": rng.choice([0, 0, 1, 4, 64, rng.randint(1, 64)]), "grad": rng.random() < 0.7}
    if kind == "rope":
        return {"kind": kind, "hq": hq, "hk": hk, "d": d, "T": _log(rng, 1, 32768), "pairs": rng.random() < 0.3,
                "cyclic": rng.random() < 0.4, "inverse": rng.random() < 0.5}
    V = rng.choice([32000, 102400, 128256, 151936, rng.randint(4000, 152000)])
    case = {"kind": kind, "T": _log(rng, 1, 8192), "V": V, "K": rng.choice([1, 8, 32, 64, rng.randint(2, 128)]),
            "temperature": rng.choice([1.0, 1.0, 2.0, round(rng.uniform(0.5, 4.0), 2)])}
    if kind == "kd_logits":
        return {**case, "fp32": rng.random() < 0.4}
    return {**case, "V": V // 8 * 8, "H": rng.choice([256, 896, 1536, 2048])}


def _cost(case):
    w = work(case)
    return max(w["flops"] / 1.0e15, w["bytes"] / 5e12)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw_one(rng)
        if _cost(c) <= most:
            return c


# ------------------------------------------------------------------------------------------------ inputs
def _lens(case):
    """Lengths of the documents, the same for every seed: shares of log-normal size, at least one token each."""
    n, total = case["docs"], case["T"]
    rng = random.Random(case["mix"])
    w = [math.exp(rng.gauss(0.0, 0.8)) for _ in range(n)]
    out = [1 + int(x / sum(w) * (total - n)) for x in w]
    out[-1] += total - sum(out)
    return out


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, scale=1.0, dtype=BF):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def _positions(T):
    """Text, a grid of frames x height x width, text: the positions of three axes, as models of images and video count them."""
    head = T // 8
    side = max(1, min(32, int(math.sqrt(T / 6))))
    grid = max(0, (T - head) * 3 // 4) // (side * side) * side * side
    t = torch.arange(T, device=DEV)
    i = (t - head).clamp_min(0)
    vis = (t >= head) & (t < head + grid)
    frames = grid // (side * side)
    axes = torch.stack((i // (side * side), i // side % side, i % side)) + head
    after = t - head - grid + head + max(frames, side if grid else 0)
    return torch.where(vis, axes, torch.where(t < head, t, after).expand(3, T)).contiguous()


def _teacher(g, T, V, K):
    """Distinct indices, frequent words more often, in no order; a few rows carry fewer entries and one none; logits that fall off."""
    k = torch.arange(K, device=DEV)
    u = (k + torch.rand(T, K, device=DEV, generator=g)) / K
    idx = torch.cummax((u.square().double() * V).long() - k, 1).values + k
    idx = torch.minimum(idx, V - K + k)
    idx = idx.gather(1, torch.rand(T, K, device=DEV, generator=g).argsort(1))
    drop = -torch.empty(T, K, device=DEV).exponential_(1.0, generator=g).cumsum(1) * 6.0 / K
    lg = 12.0 + _randn(g, T, 1, dtype=torch.float32) + drop
    short = torch.rand(T, 1, device=DEV, generator=g) < 0.05
    idx = torch.where(short & (k >= (K + 1) // 2), -1, idx)
    if T > 4:
        idx[T // 2] = -1
    labels = torch.randint(0, V, (T,), device=DEV, generator=g)
    labels[: T // 5] = IGNORE                                        # the prompt takes no part in the loss
    return idx, lg, labels


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    if case["kind"] == "attention":
        T, lens = case["T"] + case["pad"], _lens(case)
        s["qkv"] = _randn(g, T, (case["hq"] + 2 * case["hk"]) * case["d"])
        s["do"] = _randn(g, T, case["hq"] * case["d"])
        s["cu"] = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
        s["qkv"].requires_grad_(case["grad"])
    elif case["kind"] == "rope":
        s["qkv"] = _randn(g, case["T"], (case["hq"] + 2 * case["hk"]) * case["d"])
        s["pos"] = _positions(case["T"])
        n = int(s["pos"].max()) + 1
        inv = 1.0 / 1e6 ** (torch.arange(0, case["d"], 2, dtype=torch.float64, device=DEV) / case["d"])
        ang = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * inv
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        s["sections"] = SECTIONS[case["d"], case["cyclic"]]
    else:
        T, V = case["T"], case["V"]
        s["idx"], s["lg"], s["labels"] = _teacher(g, T, V, case["K"])
        if case["kind"] == "kd_logits":
            s["logits"] = _randn(g, T, V, scale=2.0, dtype=torch.float32 if case["fp32"] else BF).requires_grad_()
        else:
            s["hidden"] = _randn(g, T, case["H"]).requires_grad_()
            s["weight"] = _randn(g, V, case["H"], scale=1.5 / math.sqrt(case["H"])).requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return {"attention": _attention, "rope": _rope, "kd_logits": _kd_logits, "kd_linear": _kd_linear}[s["kind"]](s)


def _attention(s):
    if own:
        from chronicals_b200 import ops
        if not s["grad"]:
            with torch.no_grad():
                return ops.attention_qkv_packed(s["qkv"], s["cu"], s["hq"], s["hk"], s["d"], window=s["window"], sinks=s["sinks"])
        o = ops.attention_qkv_packed(s["qkv"], s["cu"], s["hq"], s["hk"], s["d"], window=s["window"], sinks=s["sinks"])
        return [o.detach(), torch.autograd.grad(o, s["qkv"], s["do"])[0]]
    return _attention_plain(s)


def _rope(s):
    if own:
        from chronicals_b200 import ops
        return ops.qk_rope_axes_(s["qkv"], s["cos"], s["sin"], s["pos"], s["hq"], s["hk"], s["d"], s["sections"], cyclic=s["cyclic"],
                                 interleaved=s["pairs"], inverse=s["inverse"])
    return _rope_plain(s)


def _kd_logits(s):
    if own:
        from chronicals_b200 import ops
        loss = ops.distillation_logits(s["logits"], s["idx"], s["lg"], s["temperature"], s["labels"], IGNORE)
        return [loss.detach(), torch.autograd.grad(loss, s["logits"])[0]]
    loss, d = _kd_plain(s["logits"].detach().float(), s)
    return [loss, d.to(s["logits"].dtype)]


def _kd_linear(s):
    if own:
        from chronicals_b200 import ops
        loss = ops.linear_distillation(s["hidden"], s["weight"], s["idx"], s["lg"], s["temperature"], s["labels"], IGNORE)
        return [loss.detach(), *torch.autograd.grad(loss, (s["hidden"], s["weight"]))]
    h, w = s["hidden"].detach().float(), s["weight"].detach().float()
    loss, d = _kd_plain(h @ w.t(), s)
    return [loss, (d @ w).to(BF), (d.t() @ h).to(BF)]


# ------------------------------------------------------------------------------------------------ plain forms, 32 bits
def _attention_plain(s):
    """Blocks of `window` queries against the keys of their own block and the one before, and against the sinks apart."""
    hq, hk, d, W, S = s["hq"], s["hk"], s["d"], s["window"], s["sinks"]
    x, T, G = s["qkv"].detach(), s["qkv"].shape[0], hq // hk
    cu = s["cu"].long()
    B = min(W, T)
    n = -(-T // B)
    P = n * B
    t = torch.arange(P, device=DEV)
    doc = torch.searchsorted(cu, t, right=True) - 1
    doc = torch.where(t < cu[-1], doc, -1)                           # behind the last document: of no document
    start = cu[doc.clamp_min(0)]
    q, k, v = (torch.nn.functional.pad(a.float().view(T, -1, d), (0, 0, 0, 0, 0, P - T)) for a in x.split([hq * d, hk * d, hk * d], 1))
    q = q.view(n, B, hk, G, d).permute(2, 0, 3, 1, 4).reshape(hk, n, G * B, d)

    def pair(a):                                                     # [P, hk, d] -> [hk, n, 2B, d]: the block before, and the own
        a = a.view(n, B, hk, d).permute(2, 0, 1, 3)
        return torch.cat((torch.nn.functional.pad(a, (0, 0, 0, 0, 1, 0))[:, :n], a), 2)

    def unpair(a):                                                   # the sum over the places that a key stands in
        own_, before = a[:, :, B:], a[:, :, :B]
        return (own_ + torch.nn.functional.pad(before, (0, 0, 0, 0, 0, 1))[:, 1:]).permute(1, 2, 0, 3).reshape(P, hk, d)

    k2, v2 = pair(k), pair(v)
    qi = t.view(n, B, 1)
    ki = (torch.arange(n, device=DEV) * B - B).view(n, 1, 1) + torch.arange(2 * B, device=DEV)
    see = (ki >= 0) & (ki <= qi) & (qi - ki < W) & (doc[ki.clamp_min(0)] == doc.view(n, B, 1)) & (doc.view(n, B, 1) >= 0)
    see = see.view(1, n, 1, B, 2 * B)
    scale = 1.0 / math.sqrt(d)
    a = (q @ k2.transpose(-1, -2)).view(hk, n, G, B, 2 * B).mul_(scale).masked_fill_(~see, -math.inf)
    m = a.amax(-1, keepdim=True)
    if S:
        at = start[:, None] + torch.arange(S, device=DEV)            # [P, S]
        see_s = ((at <= t[:, None] - W) & (doc[:, None] >= 0)).view(1, n, 1, B, S)
        at = at.clamp_max(P - 1)
        ks, vs = (y[at].view(n, B, S, hk, d).permute(3, 0, 1, 2, 4).reshape(hk, n, B, S, d) for y in (k, v))
        qs = q.view(hk, n, G, B, d).transpose(2, 3)                  # [hk, n, B, G, d]
        b = (qs @ ks.transpose(-1, -2)).transpose(2, 3).mul(scale).masked_fill(~see_s, -math.inf)     # [hk, n, G, B, S]
        m = torch.maximum(m, b.amax(-1, keepdim=True))
    m = torch.where(m == -math.inf, 0.0, m)
    a.sub_(m).exp_()
    z = a.sum(-1, keepdim=True)
    if S:
        b = (b - m).exp()
        z = z + b.sum(-1, keepdim=True)
    z = torch.where(z == 0, 1.0, z)
    a.div_(z)
    o = (a.view(hk, n, G * B, 2 * B) @ v2).view(hk, n, G, B, d)
    if S:
        b = b / z
        o = o + (b.transpose(2, 3) @ vs).transpose(2, 3)

    def rows(y):                                                     # [hk, n, G, B, d] -> [T, hq d]
        return y.permute(1, 3, 0, 2, 4).reshape(P, hq * d)[:T]

    if not s["grad"]:
        return rows(o).to(BF)
    do = torch.nn.functional.pad(s["do"].float().view(T, hk, G, d), (0, 0, 0, 0, 0, 0, 0, P - T))
    do = do.view(n, B, hk, G, d).permute(2, 0, 3, 1, 4) * (doc >= 0).view(1, n, 1, B, 1)
    dof = do.reshape(hk, n, G * B, d)
    delta = (do * o).sum(-1, keepdim=True)
    dv = unpair(a.view(hk, n, G * B, 2 * B).transpose(-1, -2) @ dof)
    ds = (dof @ v2.transpose(-1, -2)).view(hk, n, G, B, 2 * B).sub_(delta).mul_(a).mul_(scale)
    dsf = ds.view(hk, n, G * B, 2 * B)
    dq = (dsf @ k2).view(hk, n, G, B, d)
    dk = unpair(dsf.transpose(-1, -2) @ q)
    if S:
        dos = do.transpose(2, 3)                                     # [hk, n, B, G, d]
        dbs = b.transpose(2, 3) * (dos @ vs.transpose(-1, -2) - delta.transpose(2, 3)) * scale
        dq = dq + (dbs @ ks).transpose(2, 3)
        at = at.reshape(-1)
        dk = dk.index_add(0, at, (dbs.transpose(-1, -2) @ qs).permute(1, 2, 3, 0, 4).reshape(-1, hk, d))
        dv = dv.index_add(0, at, (b.transpose(2, 3).transpose(-1, -2) @ dos).permute(1, 2, 3, 0, 4).reshape(-1, hk, d))
    return [rows(o).to(BF), torch.cat((rows(dq), dk[:T].reshape(T, -1), dv[:T].reshape(T, -1)), 1).to(BF)]


def _axis_of(s):
    """The axis of every frequency: blocks one behind the other, or dealt in turn as long as an axis has frequencies left."""
    sec, half = s["sections"], s["d"] // 2
    if not s["cyclic"]:
        return torch.repeat_interleave(torch.arange(len(sec), device=DEV), torch.tensor(sec, device=DEV))
    f = torch.arange(half, device=DEV)
    turn = f % len(sec)
    return torch.where(f < torch.tensor(sec, device=DEV)[turn] * len(sec), turn, 0)


def _rope_plain(s):
    d, T, nqk = s["d"], s["T"], (s["hq"] + s["hk"]) * s["d"]
    axis = _axis_of(s)
    row = s["pos"][axis].t()                                         # [T, d / 2]: the table's row of each frequency
    f = torch.arange(d // 2, device=DEV)
    c, sn = s["cos"][row, f][:, None], s["sin"][row, f][:, None]
    sn = -sn if s["inverse"] else sn
    x = s["qkv"][:, :nqk].float().view(T, -1, d)
    if s["pairs"]:
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack((a * c - b * sn, b * c + a * sn), -1).flatten(-2)
    else:
        a, b = x[..., : d // 2], x[..., d // 2:]
        y = torch.cat((a * c - b * sn, b * c + a * sn), -1)
    s["qkv"][:, :nqk] = y.reshape(T, nqk).to(BF)
    return s["qkv"]


def _kd_plain(z, s):
    """Loss and gradient of fp32 logits `z` (in 32 bits; the sums over rows in 64)."""
    tau, T = s["temperature"], z.shape[0]
    has = s["idx"] >= 0
    valid = has.any(1) & (s["labels"] != IGNORE)
    n = valid.sum().clamp_min(1)
    at = s["idx"].clamp_min(0)
    t = torch.where(has, s["lg"] / tau, -math.inf)
    t = torch.where(valid[:, None], t, 0.0)
    q = (t - t.amax(1, keepdim=True)).exp()
    q = q / q.sum(1, keepdim=True)
    y = z / tau
    m = y.amax(1, keepdim=True)
    e = (y - m).exp()
    sm = e.sum(1, keepdim=True)
    logq = torch.where(q > 0, q, 1.0).log()
    logp = y.gather(1, at) - m - sm.log()
    rows = tau * tau * (q * (logq - logp)).sum(1)
    loss = torch.where(valid, rows, 0.0).double().sum().div(n).float()
    g = tau * valid.float()[:, None] / n
    return loss, (e / sm).mul_(g).scatter_add_(1, at, -(q * g * has))


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _attention64, "rope": _rope64, "kd_logits": _kd64, "kd_linear": _kd64}[case["kind"]](s)


def _attention64(s):
    """Document by document and a stretch of queries at a time, every key up to the last query under one mask."""
    hq, hk, d, W, S = s["hq"], s["hk"], s["d"], s["window"], s["sinks"]
    T = s["qkv"].shape[0]
    q, k, v = (a.double().view(T, -1, d).transpose(0, 1) for a in s["qkv"].detach().split([hq * d, hk * d, hk * d], 1))
    do = s["do"].double().view(T, hq, d).transpose(0, 1)
    o, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    cu, R, G = s["cu"].tolist(), 512, hq // hk
    for a, b in zip(cu, cu[1:]):
        for r0 in range(a, b, R):
            r1 = min(b, r0 + R)
            i = torch.arange(r0, r1, device=DEV)
            lo = max(a, r0 - W + 1)
            j = torch.cat((torch.arange(a, max(a, min(a + S, lo)), device=DEV), torch.arange(lo, r1, device=DEV)))
            see = (j <= i[:, None]) & ((i[:, None] - j < W) | (j < a + S))
            for g in range(hk):
                hs = slice(g * G, (g + 1) * G)
                sc = torch.einsum("gid,jd->gij", q[hs, r0:r1], k[g, j]) / math.sqrt(d)
                p = torch.softmax(sc.masked_fill(~see, -math.inf), -1)
                o[hs, r0:r1] = p @ v[g, j]
                if s["grad"]:
                    dO = do[hs, r0:r1]
                    dP = torch.einsum("gid,jd->gij", dO, v[g, j])
                    dS = p * (dP - (dP * p).sum(-1, keepdim=True)) / math.sqrt(d)
                    dq[hs, r0:r1] = dS @ k[g, j]
                    dk[g].index_add_(0, j, torch.einsum("gij,gid->jd", dS, q[hs, r0:r1]))
                    dv[g].index_add_(0, j, torch.einsum("gij,gid->jd", p, dO))
    out = o.transpose(0, 1).reshape(T, -1)
    return out if not s["grad"] else [out, torch.cat([x.transpose(0, 1).reshape(T, -1) for x in (dq, dk, dv)], 1)]


def _rope64(s):
    """Every pair as one complex number, turned by the unit number of its axis's position."""
    d, T, sec = s["d"], s["T"], s["sections"]
    axis = []
    for f in range(d // 2):
        if s["cyclic"]:
            axis.append(f % 3 if f // 3 < sec[f % 3] else 0)
        else:
            axis.append(sum(f >= sum(sec[:i + 1]) for i in range(len(sec))))
    turn = torch.stack([torch.complex(s["cos"][s["pos"][a], f].double(), s["sin"][s["pos"][a], f].double()) for f, a in enumerate(axis)], 1)
    if s["inverse"]:
        turn = turn.conj()
    x = s["qkv"].double().view(T, -1, d)
    n = s["hq"] + s["hk"]
    if s["pairs"]:
        z = torch.view_as_complex(x[:, :n].reshape(T, n, d // 2, 2).contiguous()) * turn[:, None]
        y = torch.view_as_real(z).reshape(T, n, d)
    else:
        z = torch.complex(x[:, :n, : d // 2], x[:, :n, d // 2:]) * turn[:, None]
        y = torch.cat((z.real, z.imag), -1)
    return torch.cat((y, x[:, n:]), 1).reshape(T, -1)


def _kd64(s):
    """Row by row in stretches: cross-entropy of the two distributions over the whole vocabulary, less the teacher's entropy."""
    tau, linear = s["temperature"], s["kind"] == "kd_linear"
    w = s["weight"].detach().double() if linear else None
    x = (s["hidden"] if linear else s["logits"]).detach()
    T, V = s["idx"].shape[0], s["V"]
    valid = [bool(a) for a in ((s["idx"] >= 0).any(1) & (s["labels"] != IGNORE)).tolist()]
    n, loss = max(1, sum(valid)), 0.0
    dx = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
    dw = torch.zeros_like(w) if linear else None
    for r0 in range(0, T, 1024):
        r1 = min(T, r0 + 1024)
        z = (x[r0:r1].double() @ w.t() if linear else x[r0:r1].double()) / tau
        t = torch.full((r1 - r0, V + 1), -math.inf, dtype=torch.float64, device=DEV)     # the last column takes the absent entries
        idx = s["idx"][r0:r1]
        t.scatter_(1, torch.where(idx < 0, V, idx), s["lg"][r0:r1].double() / tau)
        t[:, V] = -math.inf
        on = torch.tensor(valid[r0:r1], device=DEV)[:, None]
        q = torch.softmax(torch.where(on, t, 0.0), 1)[:, :V]
        logp = torch.log_softmax(z, 1)
        loss += tau * tau * float(torch.where(on, torch.xlogy(q, q) - q * logp, 0.0).sum()) / n
        d = torch.where(on, tau / n * (logp.exp() - q), 0.0)
        dx[r0:r1] = d @ w if linear else d
        if linear:
            dw.addmm_(d.t(), x[r0:r1].double())
    loss = torch.tensor(loss, dtype=torch.float64)
    return [loss, dx, dw] if linear else [loss, dx]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def _pairs(case):
    """Visible (query, key) pairs of one head."""
    total = 0
    for n in _lens(case):
        w = min(case["window"], n)
        total += w * (w + 1) // 2 + (n - w) * w                       # within the window
        m, k = n - w, min(case["sinks"], n)                           # the i-th query behind the window sees min(i, sinks) sinks besides
        total += sum(range(1, min(m, k) + 1)) + max(0, m - k) * k
    return total


def work(case):
    kind = case["kind"]
    if kind == "attention":
        T, rows = case["T"] + case["pad"], (case["hq"] + 2 * case["hk"]) * case["d"] * 2
        out = case["hq"] * case["d"] * 2
        macs = _pairs(case) * case["hq"] * case["d"]
        return {"bytes": T * (rows + out + (out + rows if case["grad"] else 0)), "flops": 2 * macs * (7 if case["grad"] else 2)}
    if kind == "rope":
        n = case["T"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 4 * n + 24 * case["T"], "flops": 3 * n}
    T, V, K = case["T"], case["V"], case["K"]
    teacher = T * K * 12 + T * 8
    if kind == "kd_logits":
        return {"bytes": 2 * T * V * (4 if case["fp32"] else 2) + teacher, "flops": 6 * T * V}
    H = case["H"]
    return {"bytes": 4 * H * (T + V) + teacher, "flops": 6 * T * V * H}
