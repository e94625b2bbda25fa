"""Relative-bias attention on the CPU: the bucket map, gradients against
differences, masks, the cache form against the full one, and refusals."""

import math

import pytest
import torch

from gradient_accumulation_tf_estimator_amd.ops.relative_attention import (
    RelativePositionBias,
    fused_relative_attention,
    relative_attention_decode,
    relative_position_buckets,
)


@pytest.mark.parametrize("num,far", [(32, 128), (16, 64), (64, 200), (8, 5), (256, 512), (4, 3)])
@pytest.mark.parametrize("both", [True, False])
def test_bucket_map(num, far, both):
    m = relative_position_buckets(num, far, both)
    side = num // 2 if both else num
    first = side // 2
    assert m.shape == (2 * far + 1,) and m.dtype == torch.int32 and m[far] == 0
    for n in range(1, far + 1):
        want = n
        if n >= first:
            x = math.log(n / first) / math.log(far / first) * (side - first)
            # next to a whole number the logarithms decide nothing: the powers do
            if abs(x - round(x)) < 1e-9:
                t = round(x)
                x = t if n ** (side - first) * first ** t >= far ** t * first ** (side - first) else t - 1
            want = min(first + int(x), side - 1)
        assert m[far - n] == want
        assert m[far + n] == (side + want if both else 0)
    assert int(m.max()) == num - 1


def test_bucket_refusals():
    for num, far, both in ((3, 128, True), (2, 128, True), (512, 128, True), (32, 8, True), (32, 2000, True), (1, 9, False)):
        with pytest.raises(ValueError):
            relative_position_buckets(num, far, both)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("masked", [False, True])
def test_gradients_against_differences(causal, masked):
    torch.manual_seed(0)
    B, S, NH, NKV, D = 2, 5, 4, 2, 3
    qkv = torch.randn(B, S, (NH + 2 * NKV) * D, dtype=torch.float64, requires_grad=True)
    table = torch.randn(8, NH, dtype=torch.float64, requires_grad=True)
    m = relative_position_buckets(8, 5, not causal)
    mask = torch.tensor([[1, 0, 1, 1, 0], [0, 0, 0, 0, 0]], dtype=torch.uint8) if masked else None

    def f(a, t):
        return fused_relative_attention(a, NH, t, m, nkv=NKV, mask8=mask, causal=causal)

    assert torch.autograd.gradcheck(f, (qkv, table))
    if masked:
        assert (f(qkv, table)[1] == 0).all()


def test_masked_keys_reach_nothing():
    torch.manual_seed(1)
    qkv = torch.randn(1, 6, 3 * 8)
    mask = torch.tensor([[1, 1, 0, 1, 0, 1]], dtype=torch.bool)
    table, m = torch.randn(8, 1), relative_position_buckets(8, 4)
    out = fused_relative_attention(qkv, 1, table, m, mask8=mask)
    bad = qkv.clone()
    bad[0, 2, 8:] = math.nan
    bad[0, 4, 8:] = math.inf
    assert torch.equal(fused_relative_attention(bad, 1, table, m, mask8=mask), out)


def test_table_values_that_mask():
    torch.manual_seed(2)
    qkv = torch.randn(1, 6, 3 * 8)
    m = relative_position_buckets(8, 3)
    outs = []
    for low in (-math.inf, torch.finfo(torch.float32).min):
        table = torch.zeros(8, 1)
        table[m.unique()[4:].long()] = low  # all keys behind the query
        outs.append(fused_relative_attention(qkv, 1, table, m))
    causal = fused_relative_attention(qkv, 1, torch.zeros(8, 1), m, causal=True)
    assert torch.allclose(outs[0], causal, atol=1e-6) and torch.equal(outs[0], outs[1])
    table = torch.full((8, 1), torch.finfo(torch.float32).min)
    assert (fused_relative_attention(qkv, 1, table, m) == 0).all()


def test_decode_is_the_full_form_row_by_row():
    torch.manual_seed(3)
    B, S, NH, NKV, D = 3, 9, 4, 2, 8
    qkv = torch.randn(B, S, (NH + 2 * NKV) * D)
    table, m = torch.randn(16, NH), relative_position_buckets(16, 9, False)
    full = fused_relative_attention(qkv, NH, table, m, nkv=NKV, causal=True).view(B, S, NH, D)
    x = qkv.view(B, S, NH + 2 * NKV, D)
    k, v = x[:, :, NH:NH + NKV], x[:, :, NH + NKV:]
    lengths = torch.tensor([9, 4, 1], dtype=torch.int32)
    for Sq in (1, 2):
        q = torch.stack([x[b, [max(0, int(n) - Sq + i) for i in range(Sq)], :NH] for b, n in enumerate(lengths)])
        out = relative_attention_decode(q, k, v, table, m, lengths)
        for b, n in enumerate(lengths):
            for i in range(Sq):
                at = int(n) - Sq + i
                want = full[b, at] if at >= 0 else torch.zeros(NH, D)
                torch.testing.assert_close(out[b, i], want, rtol=1e-5, atol=1e-6)
    assert (relative_attention_decode(q, k, v, table, m, torch.zeros(B, dtype=torch.int32)) == 0).all()
    assert relative_attention_decode(q, k[:, :0], v[:, :0], table, m, lengths).abs().sum() == 0


def test_refusals():
    m = relative_position_buckets(8, 4)
    t = torch.zeros(8, 2)
    qkv = torch.zeros(1, 4, 2 * 3 * 8)
    with pytest.raises(ValueError, match="qkv"):
        fused_relative_attention(qkv, 2, t, m, nkv=3)
    with pytest.raises(ValueError, match="qkv"):
        fused_relative_attention(torch.zeros(1, 4, 10), 2, t, m)
    with pytest.raises(ValueError, match="table"):
        fused_relative_attention(qkv, 2, torch.zeros(8, 3), m)
    with pytest.raises(ValueError, match="buckets"):
        fused_relative_attention(qkv, 2, t, m.long())
    with pytest.raises(ValueError, match="buckets"):
        fused_relative_attention(qkv, 2, t, m[1:])
    with pytest.raises(ValueError, match="dtype"):
        fused_relative_attention(qkv, 2, t.double(), m)
    with pytest.raises(ValueError, match="mask8"):
        fused_relative_attention(qkv, 2, t, m, mask8=torch.ones(1, 3, dtype=torch.uint8))
    with pytest.raises(ValueError, match="mask8"):
        fused_relative_attention(qkv, 2, t, m, mask8=torch.ones(1, 4))
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            fused_relative_attention(qkv, 2, t, m, scale=bad)
    q, k = torch.zeros(1, 1, 2, 8), torch.zeros(1, 4, 2, 8)
    n = torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="lengths"):
        relative_attention_decode(q, k, k, t, m, n.long())
    with pytest.raises(ValueError, match="lengths"):
        relative_attention_decode(q, k, k, t, m, torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="need q"):
        relative_attention_decode(q, k, k[:, :3], t, m, n)
    with pytest.raises(ValueError, match="dtype"):
        relative_attention_decode(q, k, k.double(), t, m, n)
    with pytest.raises(RuntimeError, match="no gradient"):
        relative_attention_decode(q.requires_grad_(), k, k, t, m, n)


def test_module():
    torch.manual_seed(4)
    mod = RelativePositionBias(2, 8, 4)
    with torch.no_grad():
        mod.weight.normal_()
    qkv = torch.randn(2, 5, 3 * 2 * 8)
    q, k, v = qkv.view(2, 5, 3, 2, 8).permute(2, 0, 3, 1, 4)
    want = torch.nn.functional.scaled_dot_product_attention(q, k, v, attn_mask=mod.dense(5)[None])
    torch.testing.assert_close(mod(qkv), want.transpose(1, 2).reshape(2, 5, 16))
    assert "buckets" not in mod.state_dict()
