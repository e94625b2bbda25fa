"""Root-mean-square norm with the residual's addition, and its 8-bit form.

    h = x + residual
    y = h / sqrt(mean(h^2) + eps) * weight

``add_rms_norm`` returns ``(y, h)``: ``h`` is the residual stream that the next
layer adds to. Both have gradients; the residual's is x's. The kernels
(ops/csrc/rms_norm.hip) take bf16, fp16 and fp32, any number of rows, widths
from 1 to 8192 and rows with any stride, and keep sums and statistics in 32
bits. Tensors on the CPU run the same formulas in plain PyTorch.

``rms_norm_fp8`` is the serving form: it writes ``y`` as e4m3 with one fp32
scale a row, or one for each ``group`` columns (``y ~ q * scale``), ready for a
scaled matrix product such as ``torch._scaled_mm``.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.nn as nn

from . import refuse_tangents, require_hip

FP8_MAX = 448.0  # the largest finite e4m3 value
GROUPS = (0, 32, 64, 128)


def _check(x, weight, residual):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x must have a last dimension of at least 1")
    if weight.shape != x.shape[-1:]:
        raise ValueError(f"weight must have shape {tuple(x.shape[-1:])}, got {tuple(weight.shape)}")
    if residual is not None and residual.shape != x.shape:
        raise ValueError(f"residual {tuple(residual.shape)} must have x's shape {tuple(x.shape)}")
    for t, name in ((weight, "weight"), (residual, "residual")):
        if t is not None and (t.dtype != x.dtype or t.device != x.device):
            raise ValueError(f"{name} must have x's dtype and device "
                             f"({x.dtype}, {x.device}), got ({t.dtype}, {t.device})")


def _plain(x, weight, residual, eps):
    up = torch.promote_types(x.dtype, torch.float32)
    h = x if residual is None else x + residual
    f = x.to(up) if residual is None else x.to(up) + residual.to(up)
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps) * weight.to(up)
    return y, h


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
                 eps: float = 1e-6, _dw_acc: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """x, residual [..., hidden]; weight [hidden], all of one dtype -> (y, h).
    Without a residual, h is x."""
    _check(x, weight, residual)
    if eps < 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if x.is_cuda:
        return tuple(require_hip().add_rms_norm(x, residual, weight, eps, _dw_acc))
    y, h = _plain(x, weight, residual, eps)
    return y.to(x.dtype), h


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
                 eps: float = 1e-6, group: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> (q e4m3 [..., hidden], scales fp32 [..., groups], h). ``group`` columns
    share a scale (0: the whole row, groups = 1); a group of zeros has scale 1,
    others at least 2^-126.
    For serving: nothing here has a gradient, so inputs that need one are
    refused while gradients are recorded, and those with a tangent at all times."""
    _check(x, weight, residual)
    if eps < 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if group not in GROUPS:
        raise ValueError(f"group must be one of {GROUPS}, got {group}")
    if group and x.shape[-1] % group:
        raise ValueError(f"hidden {x.shape[-1]} is no multiple of group {group}")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    if x.is_cuda:
        return tuple(require_hip().rms_norm_fp8(x, residual, weight, eps, group))
    refuse_tangents("rms_norm_fp8", x, weight, residual)
    groups = x.shape[-1] // group if group else 1
    y, h = _plain(x, weight, residual, eps)
    y = y.reshape(*x.shape[:-1], groups, x.shape[-1] // groups)
    top = y.abs().amax(-1)
    s = torch.where(top == 0, 1.0, (top / FP8_MAX).clamp_min(torch.finfo(top.dtype).tiny))
    q = (y / s[..., None]).to(torch.float8_e4m3fn)
    return q.view(x.shape), s, h


class FusedAddRMSNorm(nn.Module):
    """y = RMSNorm(x + residual) * weight; ``return_sum=True`` returns the sum
    too (the residual stream of pre-norm models). Bound to an engine, the
    weight's gradient is added to the flat fp32 accumulation buffer by the
    backward itself, as FusedAddLayerNorm's is."""

    def __init__(self, hidden: int, eps: float = 1e-6):
        super().__init__()
        self.hidden = hidden
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(hidden))
        self._accum_view = None

    def forward(self, x, residual=None, return_sum: bool = False):
        if self._accum_view is not None and not x.is_cuda:
            raise RuntimeError("bound FusedAddRMSNorm got a non-GPU input")
        y, h = add_rms_norm(x, self.weight, residual, eps=self.eps, _dw_acc=self._accum_view)
        return (y, h) if return_sum else y

    def forward_fp8(self, x, residual=None, group: int = 0):
        """The serving form: (q, scales, h), see rms_norm_fp8."""
        return rms_norm_fp8(x, self.weight, residual, eps=self.eps, group=group)
