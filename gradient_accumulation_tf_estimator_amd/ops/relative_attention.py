"""Attention with a learned relative position bias by buckets.

    s_ij = scale * <q_i, k_j> + table[map[clamp(j - i, -M, M) + M], head]
    out  = softmax_j(s) v          (zeros for a query with no key allowed)

``map`` gives each offset from -M to M (M = max_distance) its bucket; offsets
beyond M take the outermost one. ``relative_position_buckets`` builds the usual
map: half of a side's buckets hold one distance each, the others are spread over
the logarithm of the distance. Any other int32 map may be passed; bucket
numbers outside the table are taken as the nearest one inside.

* ``fused_relative_attention`` -- over the packed projection [B, S, (NH + 2 NKV)
  D], beside ``fused_attention``: any S, head size 64 or 128, key/value heads
  shared by NH / NKV query heads, a u8 key mask and a causal form; gradients of
  qkv and of the table (summed in 32 bits in a fixed order).
* ``relative_attention_decode`` -- the serving form: a few new tokens of each
  sequence over its K/V cache.

A table value from -2^29 down (-1e9, the type's lowest value, -inf) masks its
offsets; others are meant to be below 2^29. What stands at a key that the key
mask drops or behind a sequence's end, NaN too, reaches no result. (Keys that
only the causal order hides are ordinary data: a NaN in such a value row
reaches the queries before it, as 0 * NaN.) The kernels (ops/csrc/rel_attn.hip) take bf16; tensors on the CPU run
the same formulas in plain PyTorch.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn as nn

from . import refuse_tangents, require_hip

MAX_DISTANCE = 512
MAX_BUCKETS = 256
_LOWEST = -(2.0**29)  # a table value from here down masks its offsets


def relative_position_buckets(num_buckets: int = 32, max_distance: int = 128,
                              bidirectional: bool = True) -> torch.Tensor:
    """int32 [2 * max_distance + 1]: the bucket of each offset key - query from
    -max_distance on. With ``bidirectional`` the second half of the buckets is
    for keys behind the query; without it all are for keys before it and the
    later ones share bucket 0. Computed in whole numbers, so that no offset
    lies on the wrong side of a border."""
    side = num_buckets // 2 if bidirectional else num_buckets
    if bidirectional and num_buckets % 2:
        raise ValueError(f"num_buckets must be even for both directions, got {num_buckets}")
    if side < 2 or num_buckets > MAX_BUCKETS:
        raise ValueError(f"num_buckets must give each direction at least 2 and be at most {MAX_BUCKETS}, got {num_buckets}")
    one_each = side // 2
    if not one_each < max_distance <= MAX_DISTANCE:
        raise ValueError(f"max_distance must be above {one_each} and at most {MAX_DISTANCE}, got {max_distance}")
    rest = side - one_each
    # bucket one_each + t begins where (n / one_each)^rest >= (max_distance / one_each)^t
    of, t = [], 0
    for n in range(max_distance + 1):
        while n >= one_each and t < rest - 1 and \
                n ** rest * one_each ** (t + 1) >= max_distance ** (t + 1) * one_each ** rest:
            t += 1
        of.append(n if n < one_each else one_each + t)
    before = of[:0:-1]
    behind = [side + b for b in of[1:]] if bidirectional else [0] * max_distance
    return torch.tensor(before + [of[0]] + behind, dtype=torch.int32)


def _check_bias(table, buckets, nh, like):
    if table.dim() != 2 or table.shape[1] != nh:
        raise ValueError(f"the bias table must be [buckets, {nh}], got {tuple(table.shape)}")
    if not 1 <= table.shape[0] <= MAX_BUCKETS:
        raise ValueError(f"the bias table must have 1..{MAX_BUCKETS} buckets")
    if buckets.dim() != 1 or buckets.dtype != torch.int32 or buckets.numel() % 2 == 0 \
            or not 3 <= buckets.numel() <= 2 * MAX_DISTANCE + 1:
        raise ValueError("buckets must be an int32 tensor of 2 * max_distance + 1 entries, "
                         f"max_distance 1..{MAX_DISTANCE}")
    if table.dtype != like.dtype or table.device != like.device or buckets.device != like.device:
        raise ValueError("the bias table must have the operands' dtype, and table and buckets their device")


def _check_scale(scale, head_dim):
    scale = head_dim ** -0.5 if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def _check_gpu(t, head_dim):
    if t.dtype != torch.bfloat16:
        raise ValueError(f"the attention kernels take bf16, got {t.dtype}")
    if head_dim not in (64, 128):
        raise ValueError(f"the attention kernels take head size 64 or 128, got {head_dim}")


def _bias(table, buckets, rows, cols):
    """[NH, rows, cols] for positions of queries and keys."""
    far = buckets.numel() // 2
    which = buckets.long().clamp(0, table.shape[0] - 1)
    table = table.masked_fill(table <= _LOWEST, -math.inf)
    d = (cols[..., None, :] - rows[..., :, None]).clamp(-far, far) + far
    return table[which[d]].movedim(-1, -3)


def _softmax(s, keep):
    """softmax over the last axis of what ``keep`` allows; zeros where it allows nothing."""
    if s.shape[-1] == 0:  # no keys at all
        return s
    s = s.masked_fill(~keep, -math.inf)
    top = s.detach().amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top) & (top < 0), 0.0, top))
    z = p.sum(-1, keepdim=True)
    return p / torch.where(z == 0, 1.0, z)


def _plain_attention(qkv, nh, nkv, table, buckets, mask8, causal, scale):
    B, S, width = qkv.shape
    D = width // (nh + 2 * nkv)
    up = torch.promote_types(qkv.dtype, torch.float32)
    x = qkv.to(up).view(B, S, nh + 2 * nkv, D).transpose(1, 2)
    q = x[:, :nh]
    k, v = (t.repeat_interleave(nh // nkv, 1) for t in (x[:, nh:nh + nkv], x[:, nh + nkv:]))
    at = torch.arange(S, device=qkv.device)
    keep = torch.ones(B, 1, 1, S, dtype=torch.bool, device=qkv.device) if mask8 is None else (mask8 != 0)[:, None, None, :]
    k, v = (torch.where(keep.transpose(2, 3), t, 0.0) for t in (k, v))
    if causal:
        keep = keep & (at[None, :] <= at[:, None])
    s = torch.matmul(q, k.transpose(2, 3)) * scale + _bias(table.to(up), buckets, at, at)
    return torch.matmul(_softmax(s, keep), v).transpose(1, 2).reshape(B, S, nh * D).to(qkv.dtype)


def fused_relative_attention(qkv: torch.Tensor, nh: int, table: torch.Tensor, buckets: torch.Tensor, *,
                             nkv: Optional[int] = None, mask8: Optional[torch.Tensor] = None,
                             causal: bool = False, scale: Optional[float] = None) -> torch.Tensor:
    """qkv [B, S, (nh + 2 nkv) * D] (all query heads, then key heads, then value
    heads) -> [B, S, nh * D]. ``nkv`` key/value heads (nh if not given) are each
    shared by nh / nkv neighbouring query heads. ``mask8``: [B, S] u8 or bool,
    1 = attend. ``scale`` defaults to D ** -0.5; the kernels take 2^-96 to
    2^96. On a GPU there are first derivatives backward alone: forward-mode
    ones are refused."""
    nkv = nh if nkv is None else nkv
    if qkv.dim() != 3 or nh < 1 or nkv < 1 or nh % nkv or qkv.shape[2] < 1 or qkv.shape[2] % (nh + 2 * nkv):
        raise ValueError(f"qkv must be [B, S, (nh + 2 nkv) * D] with nh a multiple of nkv; got "
                         f"{tuple(qkv.shape)}, nh {nh}, nkv {nkv}")
    D = qkv.shape[2] // (nh + 2 * nkv)
    _check_bias(table, buckets, nh, qkv)
    scale = _check_scale(scale, D)
    if mask8 is not None:
        if mask8.shape != qkv.shape[:2] or mask8.dtype not in (torch.uint8, torch.bool) or mask8.device != qkv.device:
            raise ValueError(f"mask8 must be a u8 or bool {tuple(qkv.shape[:2])} tensor on qkv's device")
    if not qkv.is_cuda:
        return _plain_attention(qkv, nh, nkv, table, buckets, mask8, causal, scale)
    _check_gpu(qkv, D)
    if mask8 is not None:
        mask8 = (mask8.view(torch.uint8) if mask8.dtype == torch.bool else mask8).contiguous()
    return require_hip().rel_attention(qkv, table, buckets.contiguous(), mask8, nh, nkv, causal, scale)


def relative_attention_decode(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
                              buckets: torch.Tensor, lengths: torch.Tensor, *,
                              scale: Optional[float] = None) -> torch.Tensor:
    """New tokens over a K/V cache. q [B, Sq, NH, D]: the last Sq tokens of each
    sequence; k, v [B, S, NKV, D]: caches with the new tokens' rows in place, of
    any strides with contiguous heads; lengths int32 [B] on the same device:
    how many rows of the cache each sequence holds, the new ones among them
    (0 gives zeros; taken as at most S). Row i of sequence b stands at position
    lengths[b] - Sq + i and attends to the keys up to itself; a row before the
    start gives zeros. -> [B, Sq, NH, D]. For serving: it has no gradient.
    Nothing waits for the GPU, so lengths may change between replays of a graph."""
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3] \
            or k.shape[2] < 1 or q.shape[2] < 1 or q.shape[2] % k.shape[2]:
        raise ValueError(f"need q [B, Sq, NH, D] and k, v [B, S, NKV, D], NH a multiple of NKV; got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    B, Sq, NH, D = q.shape
    _check_bias(table, buckets, NH, q)
    scale = _check_scale(scale, D)
    if lengths.shape != (B,) or lengths.dtype != torch.int32 or lengths.device != q.device:
        raise ValueError(f"lengths must be an int32 [{B}] tensor on q's device")
    if any(t.dtype != q.dtype or t.device != q.device for t in (k, v)):
        raise ValueError("k and v must have q's dtype and device")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, table)):
        raise RuntimeError("relative_attention_decode has no gradient: call it under torch.no_grad()")
    if q.is_cuda:
        _check_gpu(q, D)
        return require_hip().rel_attn_token(q, k, v, table.contiguous(), buckets.contiguous(), lengths.contiguous(), scale)
    refuse_tangents("relative_attention_decode", q, k, v, table)
    S, NKV = k.shape[1:3]
    up = torch.promote_types(q.dtype, torch.float32)
    n = lengths.long().clamp(0, S)
    keys = torch.arange(S)
    held = (keys[None] < n[:, None])[:, :, None, None]
    kk, vv = (torch.where(held, t.to(up), 0.0).transpose(1, 2).repeat_interleave(NH // NKV, 1) for t in (k, v))
    rows = n[:, None] - Sq + torch.arange(Sq)[None]
    keep = (keys[None, None] <= rows[:, :, None])[:, None]
    s = torch.matmul(q.to(up).transpose(1, 2), kk.transpose(2, 3)) * scale + _bias(table.to(up), buckets, rows, keys)
    return torch.matmul(_softmax(s, keep), vv).transpose(1, 2).to(q.dtype)


class RelativePositionBias(nn.Module):
    """The learned table [num_buckets, heads] and its bucket map, shared by the
    layers of a model. The engine's rule for weight decay reads the parameter's
    name, so keep ``bias`` in the attribute that holds this module to exclude
    it, as the reference does for biases (optimization.py:65)."""

    def __init__(self, num_heads: int, num_buckets: int = 32, max_distance: int = 128, bidirectional: bool = True):
        super().__init__()
        self.num_heads = num_heads
        self.weight = nn.Parameter(torch.zeros(num_buckets, num_heads))
        self.register_buffer("buckets", relative_position_buckets(num_buckets, max_distance, bidirectional),
                             persistent=False)

    def dense(self, S: int) -> torch.Tensor:
        """[heads, S, S], for attention that takes an additive mask."""
        at = torch.arange(S, device=self.weight.device)
        return _bias(self.weight, self.buckets, at, at)

    def forward(self, qkv, *, nkv=None, mask8=None, causal=False, scale=None):
        return fused_relative_attention(qkv, self.num_heads, self.weight, self.buckets, nkv=nkv, mask8=mask8,
                                        causal=causal, scale=scale)
