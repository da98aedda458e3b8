"""autograd wrappers of the tcgen05 varlen attention kernels (``csrc/attention.cu``)."""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _ext


def _cu32(cu_seqlens: torch.Tensor) -> torch.Tensor:
    cu = cu_seqlens
    if cu.dtype != torch.int32:
        cu = cu.to(torch.int32)
    return cu.contiguous()


class _AttnPackedFn(torch.autograd.Function):
    """Attention on a fused ``[T, (hq + 2 hk) * D]`` QKV buffer; the gradient comes back as one
    fused buffer too, so autograd never has to stitch three slice gradients together.
    ``band``: () or (window, sinks).  ``documents``: how many of the boundaries' documents are not empty, as a rule; 0: all."""

    @staticmethod
    def forward(ctx, qkv, cu, hq, hk, d, scale, band=(), documents=0):
        T, ld = qkv.shape[0], qkv.stride(0)
        nq, nk = hq * d, hk * d
        o = torch.empty(T, nq, dtype=qkv.dtype, device=qkv.device)     # the kernel writes the zeros of the padding rows
        lse = torch.empty(hq, T, dtype=torch.float32, device=qkv.device)
        esz = qkv.element_size()
        o_lo = None                                    # what the rounding of O leaves out, where few keys are visible
        if band and ctx.needs_input_grad[0]:
            rows = _ext.lib().cb_attn_window_lo_rows(T, cu.numel() - 1, band[0])
            o_lo = torch.empty(2 * rows * nq + 4 * T, dtype=torch.uint8, device=qkv.device)
        fwd = _ext.lib().cb_attn_window_fwd if band else _ext.lib().cb_attn_fwd
        code = fwd(qkv.data_ptr(), qkv.data_ptr() + nq * esz, qkv.data_ptr() + (nq + nk) * esz,
                   o.data_ptr(), lse.data_ptr(), cu.data_ptr(), cu.numel() - 1, T, hq, hk, d,
                   ld, ld, ld, nq, scale, *((*band, _ext.ptr(o_lo)) if band else ()), _ext.status_buffer(qkv.device).data_ptr(),
                   _ext.stream_ptr())
        _ext.check(code, "attn_window_fwd" if band else "attn_fwd")
        ctx.save_for_backward(qkv, o, lse, cu, *(() if o_lo is None else (o_lo,)))
        ctx.cfg = (hq, hk, d, scale, band, documents)
        return o

    @staticmethod
    def backward(ctx, do):
        qkv, o, lse, cu, *o_lo = ctx.saved_tensors
        hq, hk, d, scale, band, documents = ctx.cfg
        T, ld = qkv.shape[0], qkv.stride(0)
        nq, nk = hq * d, hk * d
        if not do.is_contiguous():
            do = do.contiguous()
        if do.data_ptr() % 16:                         # a slice of a larger buffer: TMA loads want 16-byte boundaries
            do = do.clone()
        dev = qkv.device
        # the kernels use 16-byte vector accesses on dq_acc / dk_acc / dv_acc: every region must start on a
        # 16-byte boundary whatever T is (T * nq and T * nk are multiples of 4 because D is 64 or 128)
        n_delta = (hq * T + 63) // 64 * 64
        # The accumulators are cleared by the entry point right before the kernel.  Keeping them between calls and
        # letting the finalize kernel write the zeros back (``scratch_is_zero``) was measured slower (forward +
        # backward 0.191 -> 0.229 ms on 8 x 1024 tokens, 1.53 -> 1.94 ms on the 7B shape): the clears leave the lines
        # in L2, where the TMA reduce-adds of dQ then land without fetching them from memory first.
        scratch = torch.empty(n_delta + T * nq + 2 * T * nk, dtype=torch.float32, device=dev)
        delta = scratch.data_ptr()
        dq_acc = delta + 4 * n_delta
        dk_part = dq_acc + 4 * T * nq                  # per kv head, accumulated by the kernel
        dv_part = dk_part + 4 * T * nk
        dqkv = torch.empty(T, nq + 2 * nk, dtype=qkv.dtype, device=dev)
        esz = qkv.element_size()
        lib = _ext.lib()
        bwd = lib.cb_attn_window_bwd_filled if documents else lib.cb_attn_window_bwd if band else lib.cb_attn_bwd
        code = bwd(qkv.data_ptr(), qkv.data_ptr() + nq * esz, qkv.data_ptr() + (nq + nk) * esz,
                   o.data_ptr(), do.data_ptr(), lse.data_ptr(), cu.data_ptr(), cu.numel() - 1, T,
                   hq, hk, d, ld, ld, ld, nq, do.stride(0), scale, *((*band, _ext.ptr(o_lo[0]) if o_lo else None) if band else ()), delta,
                   dq_acc, dk_part, dv_part, dqkv.data_ptr(),
                   dqkv.stride(0), *((documents,) if documents else ()), _ext.status_buffer(dev).data_ptr(), _ext.stream_ptr(),
                   *(() if band else (0,)))
        _ext.check(code, "attn_window_bwd" if band else "attn_bwd")
        return dqkv, None, None, None, None, None, None, None


def kernel_supports(t: torch.Tensor, d: int) -> bool:
    return (t.is_cuda and not _ext.reference_forced() and t.dtype == torch.bfloat16 and d in (64, 128) and _ext.available()
            and _ext.has_symbol("cb_attn_fwd"))


def attention_qkv_packed(qkv: torch.Tensor, cu_seqlens: torch.Tensor, num_q_heads: int, num_kv_heads: int,
                         head_dim: int, softmax_scale: Optional[float] = None, band: tuple = (), seqlens_host=None) -> torch.Tensor:
    """Causal GQA attention over packed documents; ``qkv [T, (hq + 2 hk) * D]`` → ``[T, hq * D]``.  With a window ``seqlens_host``
    tells the documents that hold tokens from those that a list of boundaries was filled up with, for the choice of the kernel."""
    scale = float(softmax_scale) if softmax_scale is not None else 1.0 / math.sqrt(head_dim)
    assert qkv.dim() == 2 and qkv.stride(1) == 1 and qkv.stride(0) % 8 == 0
    documents = 0
    if band and seqlens_host is not None:
        documents = len(seqlens_host) - list(seqlens_host).count(0)
        documents = documents if 0 < documents < cu_seqlens.numel() - 1 else 0
    return _AttnPackedFn.apply(qkv, _cu32(cu_seqlens), num_q_heads, num_kv_heads, head_dim, scale, band, documents)


def attention_varlen_cuda(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens: torch.Tensor,
                          max_seqlen: Optional[int], scale: float, band: tuple = (), seqlens_host=None) -> torch.Tensor:
    """Separate q / k / v tensors: packed into one buffer (a copy) and run through the fused-buffer path."""
    T, hq, d = q.shape
    hk = k.shape[1]
    qkv = torch.cat((q.reshape(T, hq * d), k.reshape(T, hk * d), v.reshape(T, hk * d)), dim=1)
    return attention_qkv_packed(qkv, cu_seqlens, hq, hk, d, scale, band, seqlens_host).view(T, hq, d)
