"""A teacher's top logits on their way from samples to batches.

A sample may carry ``teacher_indices`` and ``teacher_logits [tokens, K]``: the teacher's top logits for the token that follows each
one.  Packers and collators lay them beside the tokens; rows without a teacher (padding, samples that carry none) get entries that are
absent, with the index -1.
"""
from __future__ import annotations

from typing import Any, Dict, Optional, Sequence, Tuple

import torch

TEACHER_KEYS = ("teacher_indices", "teacher_logits")
Pair = Tuple[torch.Tensor, torch.Tensor]


def teacher_of(sample: Any) -> Optional[Pair]:
    """The sample's teacher, or None.  Positions with several axes are refused: batches here count their own, one a token."""
    if not isinstance(sample, dict):
        return None
    pos = sample.get("position_ids")
    if pos is not None and torch.as_tensor(pos).dim() > 1 and torch.as_tensor(pos).shape[0] > 1:
        raise ValueError("a sample with positions of several axes: packers and collators lay out one position a token; pass batches with "
                         "position_ids [axes, B, S] instead")
    idx, lg = (sample.get(k) for k in TEACHER_KEYS)
    if idx is None and lg is None:
        return None
    if idx is None or lg is None:
        raise ValueError("teacher_indices and teacher_logits come together")
    idx, lg = torch.as_tensor(idx), torch.as_tensor(lg)
    n = torch.as_tensor(sample["input_ids"]).numel()
    if idx.dim() != 2 or idx.shape != lg.shape or idx.shape[0] != n or idx.shape[1] < 1:
        raise ValueError(f"teacher_indices {tuple(idx.shape)} and teacher_logits {tuple(lg.shape)} of a sample, wanted {(n, 'K')}")
    if idx.dtype.is_floating_point or idx.dtype.is_complex or idx.dtype == torch.bool or not lg.dtype.is_floating_point:
        raise ValueError(f"teacher_indices {idx.dtype} and teacher_logits {lg.dtype} of a sample, wanted whole and floating-point numbers")
    return idx.long(), lg


def join_teachers(pieces: Sequence[Tuple[Optional[Pair], int]]) -> Dict[str, torch.Tensor]:
    """Pieces ``(teacher, tokens)`` one behind the other: the first ``tokens`` rows of each, or as many without an entry.  Empty where no
    piece has a teacher."""
    pairs = [p for p, _ in pieces if p is not None]
    if not pairs:
        return {}
    K, total = max(i.shape[1] for i, _ in pairs), sum(n for _, n in pieces)
    dtype = pairs[0][1].dtype
    for _, lg in pairs:
        dtype = torch.promote_types(dtype, lg.dtype)
    idx, out, at = torch.full((total, K), -1, dtype=torch.long), torch.zeros(total, K, dtype=dtype), 0
    for p, n in pieces:
        if p is not None:
            idx[at:at + n, : p[0].shape[1]] = p[0][:n]
            out[at:at + n, : p[1].shape[1]] = p[1][:n]
        at += n
    return dict(zip(TEACHER_KEYS, (idx, out)))
