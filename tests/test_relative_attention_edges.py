"""Relative-bias attention at the ends of its ranges: no rows, no distance to
speak of, more new tokens than the cache holds, the smallest and largest scales."""

import math

import pytest
import torch

from gradient_accumulation_tf_estimator_amd.ops.relative_attention import (
    fused_relative_attention,
    relative_attention_decode,
    relative_position_buckets,
)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("B,S", [(0, 5), (2, 0), (0, 0)])
def test_empty_batches(B, S, masked, causal):
    m = relative_position_buckets()
    qkv, table = torch.zeros(B, S, 4 * 64, requires_grad=True), torch.randn(32, 2, requires_grad=True)
    mask = torch.ones(B, S, dtype=torch.uint8) if masked else None
    out = fused_relative_attention(qkv, 2, table, m, nkv=1, mask8=mask, causal=causal)
    dqkv, dtable = torch.autograd.grad(out.sum(), (qkv, table))
    assert out.shape == (B, S, 2 * 64) and dqkv.shape == qkv.shape and (dtable == 0).all()


@pytest.mark.parametrize("B,Sq,S", [(0, 1, 4), (2, 0, 4), (2, 1, 0), (2, 3, 0)])
def test_empty_caches(B, Sq, S):
    m = relative_position_buckets(32, 128, False)
    k = torch.zeros(B, S, 2, 8)
    out = relative_attention_decode(torch.randn(B, Sq, 4, 8), k, k, torch.randn(32, 4), m, torch.ones(B, dtype=torch.int32))
    assert out.shape == (B, Sq, 4, 8) and (out == 0).all()


def maps(far, buckets):
    return (torch.arange(2 * far + 1) % buckets).to(torch.int32)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("far,buckets", [(1, 1), (1, 3), (2, 4), (512, 1), (512, 256), (37, 5)])
@pytest.mark.parametrize("causal", [False, True])
def test_any_map(far, buckets, causal, D):
    """Short and long distances, one bucket and many, in no order of theirs: against 64 bits, with the CPU's formulas."""
    torch.manual_seed(far)
    B, S, NH = 2, 150, 2
    m = maps(far, buckets)
    qkv, table, dout = torch.randn(B, S, 3 * NH * D).bfloat16(), torch.randn(buckets, NH).bfloat16(), torch.randn(B, S, NH * D).bfloat16()

    def run(qkv, table, m, dout):
        a, t = qkv.detach().requires_grad_(), table.detach().requires_grad_()
        out = fused_relative_attention(a, NH, t, m, causal=causal)
        return [out.detach(), *torch.autograd.grad(out, (a, t), dout)]

    want = run(qkv.double(), table.double(), m, dout.double())
    got = run(qkv.cuda(), table.cuda(), m.cuda(), dout.cuda())
    # out: P and the result rounded to bf16; the gradients: D's, P's, dS's and the result's roundings, 2^-8 each of parts
    # that are at most some four times the result's own size (norms over all elements). One bucket's gradient is zero:
    # a row's dS sums to nothing; what is left is what D is off by, a rounding of out for each row.
    zero = 2.0**-8 * float(dout.double().norm()) if buckets == 1 else 0.0
    for g, w, roundings, more in zip(got, want, (2, 8, 16), (0.0, 0.0, zero)):
        assert float((g.cpu().double() - w).norm()) <= roundings * 2.0**-8 * float(w.norm()) + more + 1e-30


@pytest.mark.gpu
@pytest.mark.parametrize("Sq,S", [(5, 3), (40, 7), (3, 1)])
def test_more_new_tokens_than_the_cache_holds(Sq, S):
    torch.manual_seed(Sq)
    m, table = relative_position_buckets(32, 128, False), torch.randn(32, 4).bfloat16()
    q, k, v = torch.randn(3, Sq, 4, 64).bfloat16(), torch.randn(3, S, 2, 64).bfloat16(), torch.randn(3, S, 2, 64).bfloat16()
    n = torch.tensor([S, 1, 0], dtype=torch.int32)
    want = relative_attention_decode(q.double(), k.double(), v.double(), table.double(), m, n)
    got = relative_attention_decode(q.cuda(), k.cuda(), v.cuda(), table.cuda(), m.cuda(), n.cuda()).cpu().double()
    # P and the result rounded; sums of at most S terms
    most = float(v.double().abs().max())
    assert ((got - want).abs() <= 2 * 2.0**-8 * most + 2.0**-8 * want.abs()).all()
    assert (got[2] == 0).all() and (got[:, :Sq - S] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-300, 1e-50, 1e-38, 2.0**-97, 2.0**97, 1e39, 1e300])
def test_scales_beyond_32_bits_are_refused(scale):
    """In 32 bits they are zero or infinite, or a bias divided by them is."""
    m, table = relative_position_buckets().cuda(), torch.ones(32, 2, device="cuda").bfloat16()
    qkv = torch.ones(1, 5, 6 * 64, device="cuda").bfloat16()
    with pytest.raises(ValueError, match="scale"):
        fused_relative_attention(qkv, 2, table, m, scale=scale)
    k, n = torch.ones(1, 5, 2, 64, device="cuda").bfloat16(), torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="scale"):
        relative_attention_decode(k[:, :1], k, k, table, m, n, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [1.0, -3.0, 2.0**28, -(2.0**28)])
def test_the_smallest_scale_leaves_the_bias(bias):
    """Scores that vanish beside a bias that all keys share: the values' mean, and dv is dout's."""
    torch.manual_seed(1)
    S = 100
    m, table = relative_position_buckets().cuda(), torch.full((32, 1), bias, device="cuda").bfloat16()
    qkv, dout = torch.randn(1, S, 3 * 64).bfloat16(), torch.randn(1, S, 64).bfloat16()
    a = qkv.cuda().requires_grad_()
    out = fused_relative_attention(a, 1, table, m, scale=2.0**-96)
    dv = torch.autograd.grad(out, a, dout.cuda())[0][..., 128:].cpu().double()
    v, g = qkv[..., 128:].double(), dout.double()
    # P, dO where the sum stands apart, and the result, a rounding each of the values' absolute sums
    for got, x in ((out.detach().cpu().double(), v), (dv, g)):
        assert ((got - x.mean(1, keepdim=True)).abs() <= 3 * 2.0**-8 * x.abs().mean(1, keepdim=True)).all()
    q, n = qkv.cuda().view(1, S, 3, 64), torch.full((1,), S, dtype=torch.int32, device="cuda")
    got = relative_attention_decode(q[:, -1:, :1], q[:, :, 1:2], q[:, :, 2:], table, m, n, scale=2.0**-96).cpu().double()
    assert ((got[0, 0] - v.mean(1)).abs() <= 3 * 2.0**-8 * v.abs().mean(1)).all()
