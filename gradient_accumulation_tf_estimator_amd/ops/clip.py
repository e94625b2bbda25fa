"""Global norm over many tensors, and clipping by it.

The engine clips its own flat fp32 buffer inside the apply kernel. These two
are for gradients that live in tensors of their own: any number, of any shape,
bf16, fp16 and fp32 in one list. Semantics are ``tf.clip_by_global_norm``'s,
which the reference calls on its list of gradients (optimization.py:84):

    norm = sqrt(sum_i sum(t_i^2));  out_i = t_i * clip_norm / max(norm, clip_norm)

and where the norm is infinite or NaN every output is NaN. ``None`` entries are
passed through. Sums, and the norm that the outputs are clipped by, are held in
64 bits; the results have no gradient. Nothing waits for the GPU: the norm
stays on the device, and a call can be captured into a graph (which then holds
the tensors' addresses).
"""

from __future__ import annotations

import math
from typing import List, Optional, Sequence, Tuple

import torch

from . import require_hip

Tensors = Sequence[Optional[torch.Tensor]]


def _present(tensors: Tensors) -> List[torch.Tensor]:
    if isinstance(tensors, torch.Tensor):
        raise TypeError("expected a list of tensors")
    return [t for t in tensors if t is not None]


def _plain_norm(tensors: List[torch.Tensor]) -> torch.Tensor:
    for t in tensors:
        if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise ValueError(f"tensors must be fp32, bf16 or fp16, got {t.dtype}")
        if t.device != tensors[0].device:
            raise ValueError("tensors must be on one device")
    return torch.stack([t.detach().double().square().sum() for t in tensors]).sum().sqrt()


def global_norm(tensors: Tensors) -> torch.Tensor:
    """2-norm of all elements of all tensors, an fp32 scalar on their device."""
    got = _present(tensors)
    if not got:
        return torch.zeros(())
    if got[0].is_cuda:
        return require_hip().global_norm(got, [], False, 1.0)[0]
    return _plain_norm(got).float()


def clip_by_global_norm(tensors: Tensors, clip_norm: float, *,
                        out: Optional[Tensors] = None) -> Tuple[List[Optional[torch.Tensor]], torch.Tensor]:
    """-> (clipped tensors, norm before clipping). ``out`` takes the results:
    tensors like the inputs (same dtype, shape and strides), or the inputs
    themselves to clip in place; an output may share memory with its own input
    alone. Without it new tensors are returned."""
    if not (clip_norm > 0):
        raise ValueError(f"clip_norm must be positive, got {clip_norm}")
    got = _present(tensors)
    if out is not None and (len(out) != len(tensors) or any((a is None) != (b is None) for a, b in zip(out, tensors))):
        raise ValueError("out must have an entry for each tensor, and None where it has None")
    if not got:
        return [None] * len(tensors), torch.zeros(())
    dst = [] if out is None else _present(out)
    if got[0].is_cuda:
        norm, dst = require_hip().global_norm(got, dst, True, float(clip_norm))
    else:
        norm, dst = _plain_clip(got, dst, clip_norm)
    if out is not None:
        return list(out), norm
    if len(dst) < len(tensors):
        rest = iter(dst)
        dst = [None if t is None else next(rest) for t in tensors]
    return dst, norm


def _check_apart(got, dst):
    """No output over another output, or over another tensor's input."""
    def span(t):
        size = 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + size * t.element_size()

    spans = sorted((*span(t), is_out) for d, t in zip(dst, got) if t.numel()
                   for t, is_out in ((d, True), (t, False)) if is_out or t.data_ptr() != d.data_ptr())
    out_end = any_end = 0
    for lo, hi, is_out in spans:
        if lo < (any_end if is_out else out_end):
            raise RuntimeError("an output shares memory with another tensor of the list (is one listed twice?)")
        any_end = max(any_end, hi)
        out_end = max(out_end, hi) if is_out else out_end


@torch.no_grad()
def _plain_clip(got, dst, clip_norm):
    norm = _plain_norm(got)
    n = float(norm)
    coef = math.nan if not math.isfinite(n) else 1.0 if n <= clip_norm else clip_norm / n
    coef = torch.tensor(coef, dtype=torch.float32)
    for d, t in zip(dst, got):
        if d.shape != t.shape or d.dtype != t.dtype or d.device != t.device:
            raise ValueError("an output must have its tensor's device, dtype and shape")
    _check_apart(got, dst)
    dst = dst or [torch.empty_like(t) for t in got]
    for d, t in zip(dst, got):
        d.copy_(t.detach().float() * coef)  # detached: no_grad leaves tangents on
    return norm.float(), dst
