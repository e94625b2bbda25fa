"""RMS norm and global-norm clipping kernels against plain forms in 64 bits.

Tolerances count roundings: a value rounded to type t is off by at most
eps(t)/2 of itself. In 32 bits a sum of n terms, each thread adding at most 64
in a row before the tree, is off by at most (64 + 16) * 2^-24 of the sum of
the terms' absolute values.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from gradient_accumulation_tf_estimator_amd import clip_by_global_norm, create_optimizer, global_norm
from gradient_accumulation_tf_estimator_amd.ops.rms_norm import FusedAddRMSNorm, add_rms_norm, rms_norm_fp8

TYPES = [torch.bfloat16, torch.float16, torch.float32]
U32 = 2.0**-24


def half_step(t):
    return torch.finfo(t).eps / 2


def rand(*shape, dtype, std=1.0):
    return (torch.randn(shape, device="cuda") * std).to(dtype)


def reference(x, w, r, eps):
    h = x.double() + (r.double() if r is not None else 0)
    rstd = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    return h, rstd, h * rstd * w.double()


def tiny(t):
    """what a value below the type's normal range may be off by"""
    return torch.finfo(t).tiny * half_step(t) * 2


def check_norm(x, w, r, dy, dh, eps=1e-6):
    dt = x.dtype
    leaves = [t.requires_grad_() for t in (x, r, w) if t is not None]
    y, h = add_rms_norm(x, w, r, eps=eps)
    grads = torch.autograd.grad((y, h), leaves, (dy, dh))
    h64, rstd, y64 = reference(x.detach(), w.detach(), None if r is None else r.detach(), eps)
    n = h64 * rstd
    u = half_step(dt)
    # y: the sum's 80 U32 halves under the root, six more operations, one rounding to the type
    assert ((y.double() - y64).abs() <= (u + 48 * U32) * y64.abs() + tiny(dt)).all()
    assert ((h.double() - h64).abs() <= (u + U32) * h64.abs() + tiny(dt)).all()
    a = dy.double() * w.detach().double()
    c = (a * n).mean(-1, keepdim=True)
    c_abs = (a * n).abs().mean(-1, keepdim=True)
    dx64 = rstd * (a - n * c) + dh.double()
    # n and c come from h as it was rounded (u of each term) and 80 U32 of sums
    e = u + 90 * U32
    dx_tol = u * dx64.abs() + rstd * (8 * U32 * a.abs() + n.abs() * (2 * e * c_abs + e * c.abs())) + 4 * U32 * dh.double().abs()
    for g in grads[:-1]:
        assert ((g.double() - dx64).abs() <= dx_tol * (1 + u) + tiny(dt)).all()
    if r is not None:
        assert torch.equal(grads[0], grads[1])
    dw64 = (dy.double() * n).sum(0)
    # a block adds its rows one after another, then slabs in 16 groups
    rows = math.ceil(x.shape[0] / 512) + 64 + 16
    dw_tol = u * dw64.abs() + (u + (rows + 50) * U32) * (dy.double() * n).abs().sum(0) * (1 + u) + tiny(dt)
    assert ((grads[-1].double() - dw64).abs() <= dw_tol).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H", [1, 7, 8, 64, 511, 512, 1000, 1024, 1025, 2048, 2056, 4095, 4096, 8191, 8192])
def test_norm_widths(H, dt):
    torch.manual_seed(H)
    for R in (1, 5):
        x, r = rand(R, H, dtype=dt), rand(R, H, dtype=dt, std=3.0)
        check_norm(x, rand(H, dtype=dt), r, rand(R, H, dtype=dt), rand(R, H, dtype=dt))
        check_norm(rand(R, H, dtype=dt), rand(H, dtype=dt), None, rand(R, H, dtype=dt), rand(R, H, dtype=dt))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("R,H", [(1023, 512), (2049, 768), (5000, 96), (1500, 1500), (700, 4096)])
def test_norm_many_rows(R, H, dt):
    torch.manual_seed(R)
    check_norm(rand(R, H, dtype=dt), rand(H, dtype=dt), rand(R, H, dtype=dt), rand(R, H, dtype=dt, std=0.1), rand(R, H, dtype=dt, std=0.1))


@pytest.mark.parametrize("dt", TYPES)
def test_norm_strides_and_alignment(dt):
    torch.manual_seed(5)
    R, H = 33, 256
    wide = rand(R, 2 * H + 8, dtype=dt)
    for at in (0, 8, 3):  # 3: rows that start off 16 bytes
        x = wide[:, at:at + H].detach()
        r = rand(R, H + 5, dtype=dt)[:, 1:H + 1].detach()
        w = rand(H + 1, dtype=dt)[1:].detach()
        y, h = add_rms_norm(x, w, r)
        y2, h2 = add_rms_norm(x.contiguous(), w.clone(), r.contiguous())
        # the same elements, another order of the sum: each side is off by at most (u + 48 U32) |y| (check_norm), so the
        # two differ by at most twice that, and |y| by as much from the value that it is taken of
        two = 2 * (half_step(dt) + 48 * U32) * (1 + 2.0**-6)
        torch.testing.assert_close(y, y2, rtol=two, atol=0)
        assert torch.equal(h, h2)
    x = rand(3, 4, H, dtype=dt).transpose(0, 1)
    torch.testing.assert_close(add_rms_norm(x, w)[0], add_rms_norm(x.contiguous(), w)[0], rtol=two, atol=0)
    g = rand(H, dtype=dt).requires_grad_()
    y, _ = add_rms_norm(rand(R, H, dtype=dt), g)
    y.sum().backward()  # an expanded gradient
    assert torch.isfinite(g.grad).all()


def test_norm_empty_and_unused_outputs():
    w = torch.ones(64, device="cuda").bfloat16().requires_grad_()
    x = torch.zeros(0, 64, device="cuda").bfloat16().requires_grad_()
    y, h = add_rms_norm(x, w)
    y.sum().backward()
    assert y.shape == (0, 64) and x.grad.shape == (0, 64) and (w.grad == 0).all()
    assert rms_norm_fp8(x.detach(), w.detach())[1].shape == (0, 1)
    x = rand(4, 64, dtype=torch.bfloat16).requires_grad_()
    r = rand(4, 64, dtype=torch.bfloat16).requires_grad_()
    _, h = add_rms_norm(x, w.detach(), r)
    h.sum().backward()  # y is not used
    assert (x.grad == 1).all() and (r.grad == 1).all()
    y, _ = add_rms_norm(x.detach(), w, r.detach())  # only the weight needs a gradient
    w.grad = None
    y.float().sum().backward()
    assert torch.isfinite(w.grad).all()


def test_norm_outputs_may_be_written_in_place():
    x, r = (rand(2, 4, 64, dtype=torch.float32).requires_grad_() for _ in range(2))
    w = rand(64, dtype=torch.float32).requires_grad_()
    y, h = add_rms_norm(x, w, r)
    y.mul_(2.0)
    y.sum().backward()
    assert torch.isfinite(x.grad).all()
    y, h = add_rms_norm(x, w, r)
    h.add_(1.0)  # the backward needs h as it was
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_no_second_derivative():
    x = rand(4, 64, dtype=torch.float32).requires_grad_()
    y, _ = add_rms_norm(x, rand(64, dtype=torch.float32))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_norm_not_finite_rows_stay_apart():
    x = rand(8, 512, dtype=torch.bfloat16)
    x[3, 5] = math.nan
    x[4, 7] = math.inf
    w = torch.ones(512, device="cuda").bfloat16()
    y, _ = add_rms_norm(x, w)
    assert torch.isnan(y[3]).all() and torch.isnan(y[4, 7])
    clean = [0, 1, 2, 5, 6, 7]
    assert torch.equal(y[clean], add_rms_norm(x[clean].contiguous(), w)[0])
    q, s, _ = rms_norm_fp8(x, w)
    assert torch.isnan(s[3]).all() and torch.isfinite(s[clean]).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("H,group", [(1, 0), (77, 0), (512, 0), (1024, 0), (4096, 0), (8192, 0), (32, 32), (96, 32), (1024, 64),
                                     (1152, 128), (2176, 64), (8192, 128)])
def test_norm_fp8(H, group, dt):
    torch.manual_seed(H + group)
    R = 37
    x, w, r = rand(R, H, dtype=dt), rand(H, dtype=dt), rand(R, H, dtype=dt)
    x[2], r[2] = 0, 0
    for xx, rr in ((x, r), (x, None), (rand(R, H + 3, dtype=dt)[:, 1:H + 1], None)):
        q, s, h = rms_norm_fp8(xx, w, rr, group=group)
        h64, _, y64 = reference(xx, w, rr, 1e-6)
        g = group or H
        assert q.dtype == torch.float8_e4m3fn and q.shape == xx.shape and s.shape == (R, H // g)
        top = y64.view(R, -1, g).abs().amax(-1) / 448
        top = torch.where(top == 0, 1.0, top)
        assert ((s.double() - top).abs() <= 60 * U32 * top).all()
        per = s.double().repeat_interleave(g, 1)
        # half a step of e4m3: 2^-4 of the value, 2^-10 below the normal range
        assert ((q.double() * per - y64).abs() <= (2.0**-4 + 60 * U32) * y64.abs() + 2.0**-10 * per).all()
        assert ((h.double() - h64).abs() <= (half_step(dt) + U32) * h64.abs() + tiny(dt)).all()


def test_norm_refusals_gpu():
    x, w = torch.zeros(2, 64, device="cuda"), torch.ones(64, device="cuda")
    with pytest.raises(ValueError, match="device"):
        add_rms_norm(x, w.cpu())
    with pytest.raises(RuntimeError, match="fp32, bf16 or fp16"):
        add_rms_norm(x.double(), w.double())
    with pytest.raises(RuntimeError, match="width"):
        add_rms_norm(torch.zeros(1, 8193, device="cuda"), torch.ones(8193, device="cuda"))


def test_norm_bound_to_an_engine():
    torch.manual_seed(7)
    for K in (1, 2):
        mod = torch.nn.Sequential()
        mod.LayerNorm = FusedAddRMSNorm(256)
        mod.add_module("lin", torch.nn.Linear(256, 8))
        mod = mod.cuda().bfloat16()
        op = create_optimizer(mod, 1e-3, 10, gradient_accumulation_multiplier=4, clip_norm=None)
        x = rand(40, 256, dtype=torch.bfloat16)
        want = torch.zeros(256, device="cuda", dtype=torch.float64)
        for _ in range(K):
            y = mod.LayerNorm(x)
            dy = rand(40, 256, dtype=torch.bfloat16)
            want += (dy.double() * reference(x, torch.ones(256, device="cuda"), None, 1e-6)[2]).sum(0)
            y.backward(dy)
        got = op.engine.state.accum_view(mod.LayerNorm.weight).double()
        # h is x itself and is not rounded: fp32 sums alone
        tol = 200 * U32 * K * 40 * 16
        assert ((got - want).abs() <= tol).all()


# ---------------------------------------------------------------- clipping


def shapes():
    return [(1000, 33), (7,), (), (64, 64), (3,), (12345,), (2, 3, 5), (0, 4), (8192,), (8193,), (100001,)]


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32", "mixed"])
@pytest.mark.parametrize("clip", [0.25, 1e9, math.inf])
def test_clip_lists(kind, clip):
    torch.manual_seed(11)
    types = {"bf16": [torch.bfloat16], "fp16": [torch.float16], "fp32": [torch.float32], "mixed": TYPES}[kind]
    ts = [rand(*s, dtype=types[i % len(types)], std=0.1) for i, s in enumerate(shapes())] + [None]
    n = math.sqrt(sum(float(t.double().square().sum()) for t in ts if t is not None))
    assert abs(float(global_norm(ts)) - n) <= 2 * U32 * n  # 64-bit sums, one rounding
    keep = [None if t is None else t.clone() for t in ts]
    out, norm = clip_by_global_norm(ts, clip)
    assert abs(float(norm) - n) <= 2 * U32 * n and out[-1] is None
    c = min(1.0, clip / n)
    for o, t, k in zip(out[:-1], ts, keep):
        assert torch.equal(t, k)  # inputs are left alone
        assert o.shape == t.shape and o.dtype == t.dtype
        assert ((o.double() - t.double() * c).abs() <= (half_step(t.dtype) + 3 * U32) * t.double().abs() * c + tiny(t.dtype)).all()
        if c == 1:
            assert torch.equal(o, t)
    clip_by_global_norm(ts, clip, out=ts)  # in place
    assert all(torch.equal(a, b) for a, b in zip(ts[:-1], out))


@pytest.mark.parametrize("count", [1, 127, 128, 129, 400])
def test_clip_many_tensors(count):
    torch.manual_seed(count)
    ts = [rand(1 + 37 * i % 501, dtype=TYPES[i % 3]) for i in range(count)]
    n = math.sqrt(sum(float(t.double().square().sum()) for t in ts))
    out, norm = clip_by_global_norm(ts, 1.0)
    assert abs(float(norm) - n) <= 2 * U32 * n
    c = 1 / max(n, 1.0)
    for o, t in zip(out, ts):
        assert ((o.double() - t.double() * c).abs() <= (half_step(t.dtype) + 3 * U32) * t.double().abs() * c + tiny(t.dtype)).all()


def test_clip_alignment_and_orders():
    flat = rand(5000, dtype=torch.bfloat16)
    ts = [flat[1:1000], flat[1001:2048], flat[2048:4000].view(61, 32).t(), flat[4000:4000]]
    n = math.sqrt(sum(float(t.double().square().sum()) for t in ts))
    want = [t.double() / n for t in ts]
    edge = flat[[0, 1000, 4000, 4999]].clone()
    _, norm = clip_by_global_norm(ts, 1.0, out=ts)
    assert abs(float(norm) - n) <= 2 * U32 * n
    for t, w in zip(ts, want):
        assert ((t.double() - w).abs() <= (2.0**-8 + 3 * U32) * w.abs()).all()
    assert torch.equal(flat[[0, 1000, 4000, 4999]], edge)  # what lies between them is left alone


def test_clip_range():
    # squares beyond 32 bits' range, and below it
    big = torch.full((1000,), 1e25, device="cuda")
    assert float(global_norm([big])) == pytest.approx(1e25 * math.sqrt(1000), rel=1e-6)
    out, _ = clip_by_global_norm([big], 1.0)
    assert float(out[0][0]) == pytest.approx(1 / math.sqrt(1000), rel=1e-6)
    small = torch.full((1000,), 1e-30, device="cuda")
    assert float(global_norm([small])) == pytest.approx(1e-30 * math.sqrt(1000), rel=1e-6)
    zero = torch.zeros(10, device="cuda")
    out, norm = clip_by_global_norm([zero], 1.0)
    assert float(norm) == 0 and (out[0] == 0).all()
    assert float(global_norm([torch.zeros(0, device="cuda")])) == 0


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_clip_not_finite_gpu(bad):
    ts = [torch.ones(4000, device="cuda"), torch.tensor([1.0, bad], device="cuda").bfloat16()]
    out, norm = clip_by_global_norm(ts, 1.0)
    assert not math.isfinite(float(norm)) and all(torch.isnan(o).all() for o in out)


def test_clip_refusals_gpu():
    t = torch.ones(64, device="cuda")
    with pytest.raises(RuntimeError, match="gaps"):
        global_norm([torch.ones(8, 8, device="cuda")[:, :4]])
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_by_global_norm([t, t], 1.0, out=[t, t])
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_by_global_norm([t[:32], t[32:]], 1.0, out=[t[32:], t[:32]])
    with pytest.raises(RuntimeError, match="shares memory"):
        clip_by_global_norm([t[:32]], 1.0, out=[t[16:48]])
    with pytest.raises(RuntimeError, match="output"):
        clip_by_global_norm([t], 1.0, out=[t.half()])
    with pytest.raises(RuntimeError, match="output"):
        clip_by_global_norm([t.view(8, 8)], 1.0, out=[t.view(8, 8).t().clone(memory_format=torch.preserve_format)])
    with pytest.raises(ValueError, match="one device"):
        global_norm([t, torch.ones(3)])
    a, b = clip_by_global_norm([t, t], 1.0)[0]  # the same input twice is fine where it is only read
    assert torch.equal(a, b)


def test_clip_captured_and_on_a_stream():
    torch.manual_seed(13)
    ts = [rand(5000, dtype=torch.bfloat16), rand(333, dtype=torch.float32)]
    out = [torch.empty_like(t) for t in ts]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clip_by_global_norm(ts, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, norm = clip_by_global_norm(ts, 1.0, out=out)
    for i in range(4):
        for t in ts:
            t.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want, n = clip_by_global_norm(ts, 1.0)
        assert torch.equal(norm, n) and all(torch.equal(a, b) for a, b in zip(out, want))


def test_clip_the_gradients_of_a_step():
    """As a training step uses it: backward, clip in place, update."""
    torch.manual_seed(17)
    model = torch.nn.Sequential(torch.nn.Linear(64, 64), torch.nn.Linear(64, 8)).cuda()
    mod = FusedAddRMSNorm(64).cuda()
    x = rand(32, 64, dtype=torch.float32)
    model[1](mod(model[0](x))).square().sum().backward()
    params = [*model.parameters(), *mod.parameters()]
    n = math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))
    want = [p.grad.double() / n for p in params]
    clip_by_global_norm([p.grad for p in params], 1.0, out=[p.grad for p in params])
    for p, w in zip(params, want):
        assert ((p.grad.double() - w).abs() <= 5 * U32 * w.abs() + 1e-30).all()


@pytest.mark.parametrize("H,group", [(64, 0), (256, 32), (2048, 0), (4096, 128)])
def test_norm_fp8_below_the_normal_range(H, group):
    torch.manual_seed(17)
    x = rand(5, H, dtype=torch.float32)
    for w in (1e-44, 1e-42, 1e-40, 1e-37):
        w = torch.full((H,), w, device="cuda")
        q, s, _ = rms_norm_fp8(x, w, group=group)
        _, _, y64 = reference(x, w, None, 1e-6)
        per = s.double().repeat_interleave(group or H, 1)
        assert (s >= torch.finfo(torch.float32).tiny).all()
        # half a step of e4m3, and of a 32-bit value below the normal range
        assert ((q.double() * per - y64).abs() <= (2.0**-4 + 60 * U32) * y64.abs() + 2.0**-10 * per + 2.0**-149).all()


def test_norm_and_clip_in_inference_mode_on_a_stream():
    torch.manual_seed(18)
    norm = FusedAddRMSNorm(512).cuda().bfloat16()
    x, r = rand(33, 512, dtype=torch.bfloat16), rand(33, 512, dtype=torch.bfloat16)

    def both():
        y, h = norm(x, r, return_sum=True)
        q, s, _ = norm.forward_fp8(x, r, group=64)
        out, n = clip_by_global_norm([y, h], 1.0)
        return [y, h, q.view(torch.uint8), s, *out, n]

    with torch.no_grad():
        want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.inference_mode():
        got = both()
        kept = got[0].clone()
        clip_by_global_norm([kept], 0.5, out=[kept])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert abs(float(kept.double().norm()) - 0.5) <= 0.5 * (half_step(torch.bfloat16) + U32)
