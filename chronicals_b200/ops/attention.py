"""Varlen causal GQA attention over packed documents.

Replaces the reference's calls into flash-attn / SDPA
(chronicals/kernels/flash_attention_optimizer.py:845-994, :1388-1462).
Inputs are packed ``q [T, Hq, D]``, ``k/v [T, Hk, D]`` plus ``cu_seqlens``;
the KV head of a query head is ``hq // (Hq // Hk)`` (no ``repeat_interleave``).
Tokens before ``cu_seqlens[0]`` and at or after ``cu_seqlens[-1]`` are padding
and produce zeros.
"""
from __future__ import annotations

import math
import operator
from typing import Optional, Sequence

import torch
import torch.nn.functional as F

from . import ref
from . import _ext


def _sdpa_docs(q, k, v, bounds: Sequence[int], causal: bool, scale: float) -> torch.Tensor:
    """Library path: one SDPA call when all documents have equal length, else one per document."""
    T, hq, d = q.shape
    hk = k.shape[1]
    if bounds[0] > 0:                                  # tokens before the first document
        a = bounds[0]
        return torch.cat((q.new_zeros(a, hq, d), _sdpa_docs(q[a:], k[a:], v[a:], [b - a for b in bounds], causal, scale)))
    lens = [b - a for a, b in zip(bounds[:-1], bounds[1:])]
    out = torch.zeros_like(q) if bounds[-1] < T else torch.empty_like(q)
    if lens and all(l == lens[0] for l in lens) and lens[0] > 0:
        n, L = len(lens), lens[0]
        tot = n * L
        qq = q[:tot].view(n, L, hq, d).transpose(1, 2)
        kk = k[:tot].view(n, L, hk, d).transpose(1, 2)
        vv = v[:tot].view(n, L, hk, d).transpose(1, 2)
        o = F.scaled_dot_product_attention(qq, kk, vv, is_causal=causal, scale=scale, enable_gqa=hq != hk)
        out[:tot] = o.transpose(1, 2).reshape(tot, hq, d)
        return out
    pieces = []
    for a, b in zip(bounds[:-1], bounds[1:]):
        if b <= a:
            continue
        o = F.scaled_dot_product_attention(q[a:b].transpose(0, 1)[None], k[a:b].transpose(0, 1)[None],
                                           v[a:b].transpose(0, 1)[None], is_causal=causal, scale=scale,
                                           enable_gqa=hq != hk)
        pieces.append(o[0].transpose(0, 1))
    if pieces:
        cat = torch.cat(pieces, dim=0)
        out = torch.cat((cat, out[bounds[-1]:]), dim=0) if bounds[-1] < T else cat
    return out


def window_band(op: str, window: Optional[int], sinks: int, causal: bool = True) -> tuple:
    """``()`` without a window, else the checked ``(window, sinks)``."""
    try:
        if isinstance(window, bool) or isinstance(sinks, bool):
            raise TypeError
        window, sinks = None if window is None else operator.index(window), operator.index(sinks)
    except TypeError:
        raise ValueError(f"{op}: window {window!r} and sinks {sinks!r} must be whole numbers") from None
    if sinks < 0:
        raise ValueError(f"{op}: sinks {sinks} must not be negative")
    if window is None:
        if sinks:
            raise ValueError(f"{op}: {sinks} sinks without a window: every earlier token is visible then")
        return ()
    if window < 1:
        raise ValueError(f"{op}: window {window} must be at least 1, the token itself")
    if not causal:
        raise ValueError(f"{op}: a window needs causal attention")
    return min(window, 2 ** 31 - 1), min(sinks, 2 ** 31 - 1)


def _windowed(q, k, v, cu_seqlens, max_seqlen, scale, band, seqlens_host):
    T, hq, d = q.shape
    if k.shape != v.shape or k.dim() != 3 or k.shape[0] != T or k.shape[2] != d or k.shape[1] == 0 or hq % k.shape[1]:
        raise ValueError(f"attention_varlen: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not fit")
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"attention_varlen: softmax_scale {scale} must be positive and finite")
    from . import _same_device
    _same_device("attention_varlen", q, k, v, cu_seqlens)
    from .attention_cuda import attention_varlen_cuda, kernel_supports
    if T and cu_seqlens.numel() > 1 and all(kernel_supports(t, d) for t in (q, k, v)):
        return attention_varlen_cuda(q, k, v, cu_seqlens, max_seqlen, scale, band, seqlens_host)
    return ref.attention_window(q, k, v, cu_seqlens, *band, scale)


def attention_varlen(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                     max_seqlen: Optional[int] = None, causal: bool = True, softmax_scale: Optional[float] = None,
                     seqlens_host: Optional[Sequence[int]] = None, window: Optional[int] = None, sinks: int = 0) -> torch.Tensor:
    d = q.shape[-1]
    scale = softmax_scale if softmax_scale is not None else 1.0 / math.sqrt(d)
    band = window_band("attention_varlen", window, sinks, causal)
    if band:
        return _windowed(q, k, v, cu_seqlens, max_seqlen, scale, band, seqlens_host)
    if q.is_cuda and not _ext.reference_forced() and q.dtype == torch.bfloat16 and _ext.available() and _ext.has_symbol("cb_attn_fwd") \
            and d in (64, 128) and causal:
        from .attention_cuda import attention_varlen_cuda
        return attention_varlen_cuda(q, k, v, cu_seqlens, max_seqlen, scale)
    if q.is_cuda:
        # lengths of another number of documents: those of a typical batch, where the boundaries were filled up with empty ones
        if seqlens_host is not None and len(seqlens_host) == cu_seqlens.numel() - 1:
            bounds = [0]
            for l in seqlens_host:
                bounds.append(bounds[-1] + int(l))
        else:
            bounds = cu_seqlens.tolist()
        return _sdpa_docs(q, k, v, bounds, causal, scale)
    return ref.attention_varlen(q, k, v, cu_seqlens, max_seqlen, causal, scale)
