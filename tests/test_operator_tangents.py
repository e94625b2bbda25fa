"""Forward-mode derivatives of the norm, clipping and relative-attention
operators: right where there is a plain form, refused where they would be lost
without a word."""

import pytest
import torch
import torch.autograd.forward_ad as fw

from gradient_accumulation_tf_estimator_amd import clip_by_global_norm, global_norm
from gradient_accumulation_tf_estimator_amd.ops.relative_attention import (
    fused_relative_attention,
    relative_attention_decode,
    relative_position_buckets,
)
from gradient_accumulation_tf_estimator_amd.ops.rms_norm import add_rms_norm, rms_norm_fp8


def test_eight_bit_norm_refuses_tangents():
    x, w = torch.randn(2, 64), torch.ones(64)
    with fw.dual_level():
        for args in ((fw.make_dual(x, x), w), (x, fw.make_dual(w, w)), (x, w, fw.make_dual(x, x))):
            with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
                rms_norm_fp8(*args)
        rms_norm_fp8(x, w)  # others are taken inside the level too


def test_decode_refuses_tangents():
    m, n = relative_position_buckets(8, 5, False), torch.full((1,), 4, dtype=torch.int32)
    args = [torch.randn(1, 1, 2, 8), torch.randn(1, 4, 2, 8), torch.randn(1, 4, 2, 8), torch.randn(8, 2)]
    with fw.dual_level():
        for i, x in enumerate(args):
            with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):
                relative_attention_decode(*args[:i], fw.make_dual(x, x), *args[i + 1:], m, n)
        relative_attention_decode(*args, m, n)


def test_clipped_results_have_no_tangent():
    """Nor a gradient: the factor's own derivative is in neither."""
    x = torch.randn(2, 64)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        out, norm = clip_by_global_norm([dual], 1.0)
        for t in (out[0], norm, global_norm([dual])):
            assert fw.unpack_dual(t).tangent is None


def test_plain_forms_against_differences():
    torch.manual_seed(5)
    m, t = relative_position_buckets(8, 5, False), torch.randn(8, 2, dtype=torch.float64)
    w = torch.randn(48, dtype=torch.float64)
    x, d = torch.randn(1, 6, 48, dtype=torch.float64), torch.randn(1, 6, 48, dtype=torch.float64)
    for f in (lambda x: fused_relative_attention(x, 2, t, m, causal=True), lambda x: add_rms_norm(x, w)[0]):
        with fw.dual_level():
            got = fw.unpack_dual(f(fw.make_dual(x, d))).tangent
        # central differences of 1e-5: its square of the third derivative, and 2^-53 / 1e-5 of the values
        torch.testing.assert_close(got, (f(x + 1e-5 * d) - f(x - 1e-5 * d)) / 2e-5, rtol=1e-6, atol=1e-8)


@pytest.mark.gpu
def test_kernels_refuse_tangents():
    def rand(*shape):
        return torch.randn(shape, device="cuda").bfloat16()

    m = relative_position_buckets().cuda()
    qkv, table = rand(1, 40, 6 * 64), rand(32, 2)
    with fw.dual_level():
        dual, dual_table = fw.make_dual(qkv, rand(1, 40, 6 * 64)), fw.make_dual(table, rand(32, 2))
        for a, t in ((dual, table), (qkv, dual_table), (dual, table.clone().requires_grad_())):
            with pytest.raises(RuntimeError, match="forward-mode"):
                fused_relative_attention(a, 2, t, m)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                fused_relative_attention(a, 2, t, m)
        k = rand(1, 8, 2, 64)
        with pytest.raises(RuntimeError, match="no gradient"):
            relative_attention_decode(fw.make_dual(rand(1, 1, 2, 64), rand(1, 1, 2, 64)), k, k, table, m,
                                      torch.ones(1, dtype=torch.int32, device="cuda"))
        x, w = rand(3, 64), rand(64)
        for args in ((fw.make_dual(x, x), w), (x, fw.make_dual(w, w)), (x, w, fw.make_dual(x, x))):
            with pytest.raises(RuntimeError):
                add_rms_norm(*args)
            with torch.no_grad(), pytest.raises(RuntimeError):
                add_rms_norm(*args)
            with pytest.raises(RuntimeError, match="no gradient"):
                rms_norm_fp8(*args)
        out, norm = clip_by_global_norm([fw.make_dual(x, x)], 1.0)
        assert fw.unpack_dual(out[0]).tangent is None and fw.unpack_dual(norm).tangent is None
        fused_relative_attention(qkv, 2, table, m)  # others are taken inside the level too
