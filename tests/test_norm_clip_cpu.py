"""RMS norm and global-norm clipping on the CPU: formulas, gradients against
differences, and what the entry points refuse."""

import math

import pytest
import torch

from gradient_accumulation_tf_estimator_amd import clip_by_global_norm, global_norm
from gradient_accumulation_tf_estimator_amd.ops.rms_norm import FusedAddRMSNorm, add_rms_norm, rms_norm_fp8


def test_rms_norm_gradients_against_differences():
    torch.manual_seed(0)
    x, r = torch.randn(3, 5, dtype=torch.float64), torch.randn(3, 5, dtype=torch.float64)
    w = torch.randn(5, dtype=torch.float64)
    leaves = [t.requires_grad_() for t in (x, r, w)]
    assert torch.autograd.gradcheck(lambda a, b, c: add_rms_norm(a, c, b), leaves)
    assert torch.autograd.gradcheck(lambda a, c: add_rms_norm(a, c), (x, w))


def test_rms_norm_module_and_sum():
    torch.manual_seed(1)
    mod = FusedAddRMSNorm(7, eps=1e-5)
    x, r = torch.randn(2, 3, 7), torch.randn(2, 3, 7)
    y, h = mod(x, residual=r, return_sum=True)
    want = (x + r) / ((x + r).square().mean(-1, keepdim=True) + 1e-5).sqrt()
    assert torch.equal(h, x + r)
    # fp32: a handful of roundings of 2^-24 each
    torch.testing.assert_close(y, want, rtol=16 * 2.0**-24, atol=0)
    torch.testing.assert_close(mod(x), add_rms_norm(x, mod.weight, eps=1e-5)[0])


@pytest.mark.parametrize("group", [0, 32])
def test_rms_norm_fp8_cpu(group):
    torch.manual_seed(2)
    x = torch.randn(4, 64)
    x[1] = 0
    w = torch.randn(64)
    q, s, h = rms_norm_fp8(x, w, group=group)
    assert q.dtype == torch.float8_e4m3fn and s.shape == (4, 64 // group if group else 1)
    assert (s[1] == 1).all() and (q[1].float() == 0).all() and h.shape == x.shape
    y = add_rms_norm(x, w)[0]
    back = q.float() * s.repeat_interleave(64 // s.shape[1], 1)
    # e4m3: half a step is 2^-4 of the value, 2^-10 of the scale below 2^-6
    assert ((back - y).abs() <= 2.0**-4 * y.abs() + 2.0**-10 * s.repeat_interleave(64 // s.shape[1], 1)).all()


def test_rms_norm_no_rows():
    q, s, h = rms_norm_fp8(torch.zeros(0, 3, 64), torch.ones(64), group=32)
    assert q.shape == (0, 3, 64) and s.shape == (0, 3, 2) and h.shape == (0, 3, 64)
    assert add_rms_norm(torch.zeros(0, 64), torch.ones(64))[0].shape == (0, 64)


def test_rms_norm_refusals():
    x, w = torch.zeros(2, 8), torch.ones(8)
    with pytest.raises(ValueError, match="weight"):
        add_rms_norm(x, torch.ones(4))
    with pytest.raises(ValueError, match="residual"):
        add_rms_norm(x, w, torch.zeros(8))
    with pytest.raises(ValueError, match="dtype"):
        add_rms_norm(x, w.double())
    with pytest.raises(ValueError, match="eps"):
        add_rms_norm(x, w, eps=-1.0)
    with pytest.raises(ValueError, match="group"):
        rms_norm_fp8(x, w, group=16)
    with pytest.raises(ValueError, match="multiple"):
        rms_norm_fp8(x, w, group=32)
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_fp8(x, w.clone().requires_grad_())
    with pytest.raises(ValueError, match="last dimension"):
        add_rms_norm(torch.zeros(2, 0), torch.ones(0))


def test_clip_matches_definition():
    torch.manual_seed(3)
    ts = [torch.randn(3, 4), None, torch.randn(5).bfloat16(), torch.randn(0), torch.randn(2, 2).half()]
    n = math.sqrt(sum(float(t.double().square().sum()) for t in ts if t is not None))
    assert float(global_norm(ts)) == pytest.approx(n, rel=1e-6)
    out, norm = clip_by_global_norm(ts, 0.5)
    assert float(norm) == pytest.approx(n, rel=1e-6) and out[1] is None
    for o, t in zip(out, ts):
        if t is not None:
            assert o.dtype == t.dtype
            torch.testing.assert_close(o.double(), t.double() * 0.5 / n, rtol=torch.finfo(t.dtype).eps, atol=1e-7)
    same, _ = clip_by_global_norm(ts, n * 2)
    assert all(torch.equal(a, b) for a, b in zip(same, ts) if b is not None)
    back = clip_by_global_norm(ts, 0.5, out=ts)[0]
    assert back[0] is ts[0] and torch.equal(ts[0], out[0])


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_clip_not_finite(bad):
    out, norm = clip_by_global_norm([torch.ones(4), torch.tensor([1.0, bad])], 1.0)
    assert not math.isfinite(float(norm))
    assert all(torch.isnan(o).all() for o in out)


def test_clip_refusals():
    t = torch.ones(3)
    for bad in (0.0, -1.0, math.nan):
        with pytest.raises(ValueError, match="clip_norm"):
            clip_by_global_norm([t], bad)
    with pytest.raises(TypeError):
        global_norm(t)
    with pytest.raises(ValueError, match="fp32"):
        global_norm([torch.ones(2, dtype=torch.int32)])
    with pytest.raises(ValueError, match="entry"):
        clip_by_global_norm([t], 1.0, out=[])
    with pytest.raises(ValueError, match="output"):
        clip_by_global_norm([t], 1.0, out=[torch.ones(4)])
    assert float(global_norm([])) == 0 and clip_by_global_norm([None], 1.0)[0] == [None]


def test_a_tensor_listed_twice_is_refused():
    t, u = torch.ones(4), torch.ones(4)
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_by_global_norm([t, t], 1.0, out=[t, t])
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_by_global_norm([t, u], 1.0, out=[u, t])
    big = torch.ones(8)
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_by_global_norm([big[:5], big[3:]], 1.0, out=[big[:5], big[3:]])
    assert (t == 1).all() and (u == 1).all() and (big == 1).all()
    clip_by_global_norm([big[:4], big[4:]], 1.0, out=[big[:4], big[4:]])  # neighbours share nothing
    assert abs(float(big.norm()) - 1.0) < 1e-6


def test_fp8_scales_stay_in_the_normal_range():
    x = torch.randn(3, 64)
    for w in (1e-44, 1e-42, 1e-40):
        q, s, _ = rms_norm_fp8(x, torch.full((64,), w))
        assert torch.isfinite(q.float()).all() and (s >= torch.finfo(torch.float32).tiny).all()
