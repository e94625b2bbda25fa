"""Relative-bias attention on the CPU without rows: as the kernels take it."""

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
