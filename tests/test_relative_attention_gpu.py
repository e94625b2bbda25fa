"""Relative-bias attention kernels against the formulas in 64 bits.

Tolerances count roundings, element by element. With u = 2^-8 (half a step of
bf16, relative) and e = 2^-24:

* a score is a sum of D products in 32 bits: off by (D + 8) e of the sum of
  their absolute values, so a probability is off by a relative
  r = 2 (D + 8) e max|q||k| scale + 64 e (both of its scores; exp2, sums);
* out: probabilities rounded once (u of sum P|v|), and the result (u of it);
* dsum = <dout, out> takes out as it was rounded: off by sum |dout| tol(out);
* dS = P (dP - dsum): P times what dsum is off by, r and (D + 8) e of its
  parts, and one rounding u before it is multiplied; gradients are rounded once.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from gradient_accumulation_tf_estimator_amd.ops.relative_attention import (
    RelativePositionBias,
    fused_relative_attention,
    relative_attention_decode,
    relative_position_buckets,
)

U, E32 = 2.0**-8, 2.0**-24


def rand(*shape, std=1.0):
    return (torch.randn(shape, device="cuda") * std).bfloat16()


def split(qkv, NH, NKV):
    """q, k, v in 64 bits, [B, NH, S, D], shared heads repeated"""
    B, S, W = qkv.shape
    x = qkv.detach().double().view(B, S, NH + 2 * NKV, W // (NH + 2 * NKV)).transpose(1, 2)
    n = NH // NKV
    return x[:, :NH].contiguous(), x[:, NH:NH + NKV].repeat_interleave(n, 1), x[:, NH + NKV:].repeat_interleave(n, 1)


def probabilities(q, k, bias, keep, scale):
    s = (q @ k.transpose(2, 3).contiguous() * scale + bias).masked_fill(~keep, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    z = p.sum(-1, keepdim=True)
    most = (q.abs() @ k.abs().transpose(2, 3).contiguous() * scale + bias.nan_to_num(neginf=0).abs()).masked_fill(~keep, 0.0)
    r = 2 * (q.shape[-1] + 8) * E32 * most.amax() + 64 * E32
    return p / torch.where(z == 0, 1.0, z), float(r)


def check(B, S, NH, NKV, D, causal, mask, nb=32, far=128, scale=None, qkv=None, table=None, grad=True, poison=False):
    m = relative_position_buckets(nb, far, not causal).cuda()
    qkv = rand(B, S, (NH + 2 * NKV) * D) if qkv is None else qkv
    table = rand(nb, NH, std=0.5) if table is None else table
    dout = rand(B, S, NH * D)
    c = D ** -0.5 if scale is None else scale
    at = torch.arange(S, device="cuda")
    bias = table.detach().double()[m.long()[(at[None] - at[:, None]).clamp(-far, far) + far]].permute(2, 0, 1)
    keep = torch.ones(B, 1, S, S, dtype=torch.bool, device="cuda")
    if mask is not None:
        keep = keep & (mask != 0)[:, None, None, :]
    if causal:
        keep = keep & (at[None] <= at[:, None])
    keep = keep & (bias > -math.inf)[None]
    q, k, v = split(qkv, NH, NKV)
    given, gout = qkv, dout
    if poison:  # what must not count
        x = qkv.detach().clone().view(B, S, -1, D)
        off = mask == 0
        y = x[off]
        y[:, NH:] = math.nan
        y[::2, NH:] = math.inf
        x[off] = y
        empty = ~keep.any(-1).any(1)  # [B, S]: rows that no head has a key for
        y = x[empty]
        y[:, :NH] = math.nan
        x[empty] = y
        given = x.view(B, S, -1)
        gout = dout.clone()
        gout[empty] = math.nan
        dout = dout.masked_fill(empty[..., None], 0.0)
    leaf, tleaf = given.detach().requires_grad_(grad), table.detach().requires_grad_(grad)
    out = fused_relative_attention(leaf, NH, tleaf, m, nkv=NKV, mask8=mask, causal=causal, scale=scale)
    p, r = probabilities(q, k, bias[None], keep, c)
    o = p @ v
    tol_o = (2 * U + 2 * r) * (p @ v.abs()) + U * o.abs()
    got = out.detach().double().view(B, S, NH, D).transpose(1, 2)
    assert ((got - o).abs() <= tol_o + 1e-30).all()
    if not grad:
        return out
    dqkv, dtable = torch.autograd.grad(out, (leaf, tleaf), gout)
    do = dout.double().view(B, S, NH, D).transpose(1, 2).contiguous()
    t = lambda z: z.transpose(2, 3).contiguous()  # noqa: E731
    dp = do @ t(v)
    dsum = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - dsum)
    off_sum = (do.abs() * tol_o).sum(-1, keepdim=True) + (D + 8) * E32 * (do.abs() * o.abs()).sum(-1, keepdim=True)
    off_ds = p * off_sum + p * ((D + 8) * E32 * (do.abs() @ t(v.abs())) + 2 * r * (dp.abs() + dsum.abs()))
    n, e = NH // NKV, S * E32  # sums over S in 32 bits
    fold = lambda z: z.view(B, NKV, n, S, D).sum(2)  # noqa: E731

    def near(got, want, tol):
        assert ((got - want).abs() <= tol * (1 + U) + U * want.abs() + 1e-30).all(), float(((got - want).abs() / (tol + 1e-30)).max())

    g = dqkv.double().view(B, S, NH + 2 * NKV, D).transpose(1, 2)
    near(g[:, :NH], ds @ k * c, c * ((off_ds + (U + e) * (ds.abs() + off_ds)) @ k.abs()))
    near(g[:, NH:NH + NKV], fold(t(ds) @ q * c), fold(c * (t(off_ds + (U + n * e) * (ds.abs() + off_ds)) @ q.abs())))
    near(g[:, NH + NKV:], fold(t(p) @ do), fold(t(p * (U + 2 * r + n * e)) @ do.abs()))
    idx = m.long()[(at[None] - at[:, None]).clamp(-far, far) + far].reshape(-1)
    by = lambda z: torch.zeros(nb, NH, device="cuda", dtype=torch.float64).index_add_(0, idx, z.sum(0).reshape(NH, -1).t().contiguous())  # noqa: E731
    near(dtable.double(), by(ds), by(off_ds + (B * S + 64) * E32 * (ds.abs() + off_ds)))
    return out


def padded(B, S, least=1):
    n = torch.linspace(least, S, B).round().long()
    return (torch.arange(S)[None] < n[:, None]).to(torch.uint8).cuda()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S", [2, 3, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 191, 257, 400])
def test_lengths(S, causal, D):
    torch.manual_seed(S)
    check(2, S, 4, 2, D, causal, None)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["padded", "empty", "holes", "one", "left", "all"])
def test_masks(kind, causal, D):
    torch.manual_seed(7)
    B, S = 3, 170
    mask = padded(B, S, 5)
    if kind == "empty":
        mask[1] = 0
    elif kind == "holes":
        mask = (torch.rand(B, S, device="cuda") < 0.3).to(torch.uint8)
    elif kind == "one":
        mask = torch.zeros(B, S, dtype=torch.uint8, device="cuda")
        mask[:, 77] = 1
    elif kind == "left":
        mask = mask.flip(1).contiguous()
    elif kind == "all":
        mask = torch.zeros(B, S, dtype=torch.uint8, device="cuda")
    out = check(B, S, 4, 4, D, causal, mask, poison=True)
    if kind == "all":
        assert (out == 0).all()
    check(B, S, 4, 4, D, causal, mask * 255 if kind == "padded" else mask.bool(), grad=False)


@pytest.mark.parametrize("NH,NKV", [(1, 1), (3, 1), (8, 8), (8, 2), (12, 4)])
@pytest.mark.parametrize("causal", [False, True])
def test_shared_heads(NH, NKV, causal):
    torch.manual_seed(NH)
    check(2, 150, NH, NKV, 64, causal, padded(2, 150, 60))


@pytest.mark.parametrize("nb,far", [(4, 3), (8, 5), (32, 64), (64, 300), (256, 512)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [64, 128])
def test_bucket_tables(nb, far, causal, D):
    torch.manual_seed(far)
    check(1, 450, 2, 1, D, causal, None, nb=nb, far=far)


@pytest.mark.parametrize("scale", [1.0, 0.02, 3e-3])
def test_scales(scale):
    torch.manual_seed(3)
    check(1, 140, 2, 2, 64, False, None, scale=scale, qkv=rand(1, 140, 6 * 64, std=0.4))


@pytest.mark.parametrize("D", [64, 128])
def test_long(D):
    torch.manual_seed(5)
    check(1, 1500, 2, 1, D, True, None)
    check(1, 1500, 2, 2, D, False, padded(1, 1500, 1337))


def test_one_key():
    """One key: the output is its value, dv is dout, and dq, dk and dtable are zero up to dsum's rounding."""
    torch.manual_seed(6)
    qkv, table = rand(3, 1, 3 * 2 * 64).requires_grad_(), rand(32, 2).requires_grad_()
    m = relative_position_buckets().cuda()
    out = fused_relative_attention(qkv, 2, table, m)
    assert torch.equal(out, qkv[:, :, 256:].detach())
    dout = rand(3, 1, 128)
    dqkv, dtable = torch.autograd.grad(out, (qkv, table), dout)
    assert torch.equal(dqkv[:, :, 256:], dout)
    v = qkv.detach()[:, :, 256:].double().abs().view(3, 2, 64)
    off = (72 * E32) * (dout.double().abs().view(3, 2, 64) * v).sum(-1)  # out is exact here: sums in 32 bits alone
    assert (dqkv[:, :, :256].double().view(3, 2, 2, 64).abs().amax((1, 3)) <= 0.125 * 2 * off * 8).all()
    assert (dtable.double().abs().sum(0) <= 2 * off.sum(0)).all()


def test_empty_batches():
    m = relative_position_buckets().cuda()
    for shape in ((0, 5, 3 * 64), (2, 0, 3 * 64)):
        qkv = torch.zeros(shape, device="cuda").bfloat16().requires_grad_()
        table = rand(32, 1).requires_grad_()
        out = fused_relative_attention(qkv, 1, table, m)
        dqkv, dtable = torch.autograd.grad(out.sum(), (qkv, table))
        assert out.shape == (*shape[:2], 64) and dqkv.shape == shape and (dtable == 0).all()


def test_table_values_that_mask():
    torch.manual_seed(8)
    m = relative_position_buckets(32, 128).cuda()
    for low in (-math.inf, torch.finfo(torch.bfloat16).min):
        table = rand(32, 2, std=0.5)
        table[17:] = -math.inf
        want = table.clone()
        if low > -math.inf:
            table[17:] = low
        qkv = rand(1, 200, 6 * 64)
        out = fused_relative_attention(qkv, 2, table, m)
        torch.manual_seed(9)
        assert torch.equal(out, check(1, 200, 2, 2, 64, False, None, qkv=qkv, table=want, grad=False))
    full = torch.full((32, 2), torch.finfo(torch.bfloat16).min, device="cuda").bfloat16()
    assert (fused_relative_attention(qkv, 2, full, m) == 0).all()
    # bucket numbers outside the table are taken as the nearest inside
    wild = m.clone()
    wild[:100], wild[200:] = -5, 1000
    table = rand(32, 2)
    assert torch.equal(fused_relative_attention(qkv, 2, table, wild), fused_relative_attention(qkv, 2, table, wild.clamp(0, 31)))


def test_layout_of_operands():
    torch.manual_seed(10)
    m = relative_position_buckets().cuda()
    table = rand(32, 2)
    qkv = rand(2, 70, 6 * 64)
    want = fused_relative_attention(qkv, 2, table, m)
    odd = torch.empty(qkv.numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view_as(qkv).copy_(qkv)
    wide = torch.empty(2, 70, 7 * 64, device="cuda", dtype=torch.bfloat16)[..., :6 * 64].copy_(qkv)
    for x in (odd, wide):
        x = x.detach().requires_grad_()
        out = fused_relative_attention(x, 2, table, m)
        assert torch.equal(out, want)
        out.sum().backward()  # an expanded gradient
        assert x.grad.shape == x.shape
    assert torch.equal(fused_relative_attention(qkv, 2, table.t().contiguous().t(), m), want)


def test_results_do_not_depend_on_timing():
    torch.manual_seed(11)
    m = relative_position_buckets(32, 128, False).cuda()
    qkv, table, dout = rand(4, 333, 8 * 64).requires_grad_(), rand(32, 4).requires_grad_(), rand(4, 333, 4 * 64)
    first = None
    for _ in range(3):
        out = fused_relative_attention(qkv, 4, table, m, nkv=2, causal=True)
        got = [out, *torch.autograd.grad(out, (qkv, table), dout)]
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_gradients_against_differences():
    """Along one direction each: (f(x + h d) - f(x - h d)) / 2h of sum(out * w) against <grad, d>."""
    torch.manual_seed(12)
    m = relative_position_buckets(32, 20).cuda()
    B, S, NH, D = 1, 48, 2, 64
    qkv, table = rand(B, S, 3 * NH * D), rand(32, NH, std=0.5)
    w = rand(B, S, NH * D)
    leaf, tleaf = qkv.clone().requires_grad_(), table.clone().requires_grad_()
    out = fused_relative_attention(leaf, NH, tleaf, m)
    g, gt = torch.autograd.grad(out, (leaf, tleaf), w)

    def f(x, t):
        q, k, v = split(x, NH, NH)
        at = torch.arange(S, device="cuda")
        bias = t.double()[m.long()[(at[None] - at[:, None]).clamp(-20, 20) + 20]].permute(2, 0, 1)
        p = torch.softmax(q @ k.transpose(2, 3).contiguous() / 8 + bias, -1)
        return float(((p @ v).transpose(1, 2).reshape(B, S, -1) * w.double()).sum())

    for x, t, grad, d in ((qkv, None, g, torch.randn_like(qkv, dtype=torch.float64)), (None, table, gt, torch.randn_like(table, dtype=torch.float64))):
        h = 1e-4
        if t is None:
            diff = (f(qkv.double() + h * d, table) - f(qkv.double() - h * d, table)) / (2 * h)
        else:
            diff = (f(qkv, table.double() + h * d) - f(qkv, table.double() - h * d)) / (2 * h)
        got = float((grad.double() * d).sum())
        # three roundings of u on the way, in random directions: their sum over n elements grows as its root
        assert abs(got - diff) <= 3 * U * float((grad.double() * d).norm()) * 6 + 1e-3


def test_refusals_gpu():
    m = relative_position_buckets().cuda()
    t = rand(32, 2)
    with pytest.raises(ValueError, match="bf16"):
        fused_relative_attention(torch.zeros(1, 4, 6 * 64, device="cuda"), 2, t.float(), m)
    with pytest.raises(ValueError, match="head size"):
        fused_relative_attention(rand(1, 4, 6 * 32), 2, t, m)
    with pytest.raises(ValueError, match="device"):
        fused_relative_attention(rand(1, 4, 6 * 64), 2, t, m.cpu())
    with pytest.raises(ValueError, match="device"):
        fused_relative_attention(rand(1, 4, 6 * 64), 2, t, m, mask8=torch.ones(1, 4, dtype=torch.uint8))
    k = rand(1, 8, 2, 64)
    n = torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="16 bytes"):
        relative_attention_decode(rand(1, 1, 2, 64), rand(1, 8, 2, 65)[..., :64], k, t, m, n)
    with pytest.raises(RuntimeError, match="at most 32"):
        relative_attention_decode(rand(1, 1, 64, 64), rand(1, 8, 1, 64), rand(1, 8, 1, 64), rand(32, 64), m, n)


# ---------------------------------------------------------------- new tokens over a cache


def check_token(q, k, v, table, m, lengths, scale=None):
    B, Sq, NH, D = q.shape
    S, NKV = k.shape[1:3]
    far = m.numel() // 2
    out = relative_attention_decode(q, k, v, table, m, lengths, scale=scale)
    assert out.shape == q.shape
    for b in range(B):
        n = min(max(int(lengths[b]), 0), S)
        pos = torch.arange(n - Sq, n, device="cuda")
        keys = torch.arange(n, device="cuda")
        kk, vv = (x[b, :n].double().transpose(0, 1).repeat_interleave(NH // NKV, 0) for x in (k, v))
        bias = table.double()[m.long()[(keys[None] - pos[:, None]).clamp(-far, far) + far]].permute(2, 0, 1)
        keep = (keys[None] <= pos[:, None])[None, None]
        if n == 0:
            assert (out[b] == 0).all()
            continue
        p, r = probabilities(q[b].double().transpose(0, 1)[None].contiguous(), kk[None].contiguous(), bias[None], keep,
                             D ** -0.5 if scale is None else scale)
        o = (p @ vv[None])[0].transpose(0, 1)
        tol = (2 * U + 2 * r) * (p @ vv.abs()[None])[0].transpose(0, 1) + U * o.abs()
        assert ((out[b].double() - o).abs() <= tol + 1e-30).all(), (b, n)
    return out


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq", [1, 2, 7])
@pytest.mark.parametrize("NH,NKV", [(2, 2), (8, 2), (12, 1)])
@pytest.mark.parametrize("S", [1, 31, 33, 200, 700, 3001])
def test_token(S, NH, NKV, Sq, D):
    torch.manual_seed(S)
    B = 5
    q, k, v = rand(B, Sq, NH, D), rand(B, S, NKV, D), rand(B, S, NKV, D)
    m = relative_position_buckets(32, 128, False).cuda()
    lengths = torch.tensor([S, max(1, S // 2), min(S, 1), 0, S + 9], dtype=torch.int32, device="cuda")
    for b, n in enumerate(lengths.tolist()):  # behind the end: whatever was there
        k[b, max(n, 0):] = math.nan
        v[b, max(n, 0):] = math.inf
    check_token(q, k, v, rand(32, NH, std=0.5), m, lengths)


@pytest.mark.parametrize("Sq,NH,NKV", [(1, 32, 1), (33, 2, 2), (20, 8, 2)])
def test_token_many_rows(Sq, NH, NKV):
    torch.manual_seed(Sq)
    m = relative_position_buckets(16, 40, False).cuda()
    check_token(rand(2, Sq, NH, 64), rand(2, 150, NKV, 64), rand(2, 150, NKV, 64), rand(16, NH), m,
                torch.tensor([150, Sq + 1], dtype=torch.int32, device="cuda"))


def test_token_strides_and_far_offsets():
    torch.manual_seed(21)
    m = relative_position_buckets(32, 500, False).cuda()
    B, S, NKV, D = 2, 500, 2, 64
    both = rand(B, NKV, S, 2, D)  # heads first, keys and values interleaved
    k, v = both[:, :, :, 0].transpose(1, 2), both[:, :, :, 1].transpose(1, 2)
    q = rand(B, 3, 6, D)[:, 1:2]
    n = torch.tensor([500, 123], dtype=torch.int32, device="cuda")
    out = check_token(q, k, v, rand(32, 6), m, n, scale=1.0 / 20)
    # an offset of a sequence that passes 32 bits (in elements): the batch stride of a large cache
    far = torch.empty(2 * (1 << 31) // 2 + S * NKV * D, dtype=torch.bfloat16, device="cuda")
    at = 1 << 31
    big_k = far.as_strided((2, S, NKV, D), (at, NKV * D, D, 1))
    big_k.copy_(k)
    assert torch.equal(relative_attention_decode(q, big_k, v, table := rand(32, 6), m, n),
                       relative_attention_decode(q, k, v, table, m, n))
    assert out.shape == (B, 1, 6, D)


def test_token_captured_with_growing_lengths():
    """As a server uses it: one graph, the cache and the lengths grow between replays."""
    torch.manual_seed(22)
    B, S, NH, NKV, D = 3, 300, 4, 2, 64
    m = relative_position_buckets(32, 64, False).cuda()
    table = rand(32, NH)
    q, k, v = rand(B, 1, NH, D), torch.zeros(B, S, NKV, D, device="cuda").bfloat16(), torch.zeros(B, S, NKV, D, device="cuda").bfloat16()
    n = torch.zeros(B, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        relative_attention_decode(q, k, v, table, m, n)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = relative_attention_decode(q, k, v, table, m, n)
    for step in range(6):
        grow = 40 + 3 * step
        for t in (k, v):
            t[:, step * 45:step * 45 + grow] = rand(B, grow, NKV, D)
        n.fill_(step * 45 + grow)
        q.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, check_token(q, k, v, table, m, n))


def test_training_step_captured():
    torch.manual_seed(23)
    m = relative_position_buckets(32, 64).cuda()
    bias = RelativePositionBias(2, 32, 64).cuda().bfloat16()
    with torch.no_grad():
        bias.weight.normal_()
    qkv, dout = rand(2, 96, 6 * 64).requires_grad_(), rand(2, 96, 128)

    def step():
        out = fused_relative_attention(qkv, 2, bias.weight, m)
        return [out.detach(), *torch.autograd.grad(out, (qkv, bias.weight), dout)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            qkv.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("value", [2.0**11, 2.0**12, -(2.0**20), 2.0**20, -99614720.0, 99614720.0])
def test_one_large_bias_for_all(value, causal, D):
    """A table of one value, which softmax does not see: the oracle has none. Beside the tolerances above: what the
    scores lose next to such a value is at most the products themselves, so a probability is off by twice the largest
    one more; dO is rounded once more on its way to dK and dV (u of it)."""
    torch.manual_seed(13)
    B, S, NH = 2, 330, 2
    m = relative_position_buckets(32, 128, not causal).cuda()
    mask = padded(B, S, 150)
    qkv = rand(B, S, 3 * NH * D)
    qkv[:, :, :2 * NH * D] *= 2.0**-8
    dout = rand(B, S, NH * D)
    leaf, tleaf = qkv.clone().requires_grad_(), torch.full((32, NH), value, device="cuda").bfloat16().requires_grad_()
    out = fused_relative_attention(leaf, NH, tleaf, m, mask8=mask, causal=causal)
    dqkv, dtable = torch.autograd.grad(out, (leaf, tleaf), dout)
    at, c = torch.arange(S, device="cuda"), D ** -0.5
    keep = ((mask != 0)[:, None, None, :] & (at[None] <= at[:, None] if causal else torch.ones_like(at[None] <= at[:, None])))
    q, k, v = split(qkv, NH, NH)
    t = lambda z: z.transpose(2, 3).contiguous()  # noqa: E731
    p, r = probabilities(q, k, torch.zeros(1, NH, S, S, device="cuda", dtype=torch.float64), keep, c)
    r += 2.1 * float((q @ t(k) * c).abs().amax())
    do = dout.double().view(B, S, NH, D).transpose(1, 2).contiguous()
    o, va, da = p @ v, v.abs(), do.abs()
    tol_o = (2 * U + 2 * r) * (p @ va) + U * o.abs()
    dp, dsum = do @ t(v), (do * o).sum(-1, keepdim=True)
    ds = p * (dp - dsum)
    off = p * ((da * tol_o).sum(-1, keepdim=True) + ((D + 8) * E32 + U) * (da @ t(va)) + 2 * r * (dp.abs() + dsum.abs())
               + (D + 8) * E32 * (da * o.abs()).sum(-1, keepdim=True))
    off_ds = off + (U + S * E32) * (ds.abs() + off)
    got = [*dqkv.double().view(B, S, 3, NH, D).permute(2, 0, 3, 1, 4), out.detach().double().view(B, S, NH, D).transpose(1, 2)]
    want = [(ds @ k * c, off_ds @ k.abs() * c), (t(ds) @ q * c, t(off_ds) @ q.abs() * c),
            (t(p) @ do, t(p * (2 * U + 2 * r + S * E32)) @ da), (o, tol_o)]
    for name, g, (w, tol) in zip(("dq", "dk", "dv", "out"), got, want):
        assert ((g - w).abs() <= tol * (1 + U) + U * w.abs() + 1e-30).all(), name
    idx = m.long()[(at[None] - at[:, None]).clamp(-128, 128) + 128].reshape(-1)
    by = lambda z: torch.zeros(32, NH, device="cuda", dtype=torch.float64).index_add_(0, idx, z.sum(0).reshape(NH, -1).t().contiguous())  # noqa: E731
    w, tol = by(ds), by(off_ds)
    assert ((dtable.double() - w).abs() <= tol * (1 + U) + U * w.abs() + 1e-30).all()


def test_table_values_below_the_usable_range_mask():
    torch.manual_seed(14)
    m = relative_position_buckets(32, 128).cuda()
    qkv, dout = rand(1, 200, 6 * 64), rand(1, 200, 128)
    got = []
    for low in (-math.inf, -1e9, -(2.0**29), -1e30):
        table = rand(32, 2, std=0.5) if not got else table.detach().clone()
        table[17:] = low
        leaf, tleaf = qkv.clone().requires_grad_(), table.requires_grad_()
        out = fused_relative_attention(leaf, 2, tleaf, m)
        got.append([out, *torch.autograd.grad(out, (leaf, tleaf), dout)])
        token = relative_attention_decode(qkv[:, 9:10, :128].view(1, 1, 2, 64), qkv[:, :, 128:256].view(1, 200, 2, 64),
                                          qkv[:, :, 256:].view(1, 200, 2, 64), table.detach(), m.flip(0).contiguous(),
                                          torch.tensor([200], dtype=torch.int32, device="cuda"))
        got[-1].append(token)
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(other, got[0]))


@pytest.mark.parametrize("B,S,NH,NKV", [(1, 8321, 1, 1), (2, 300, 8, 4), (8, 129, 2, 1)])
def test_causal_orders_of_work(B, S, NH, NKV):
    """More tiles than one stretch of the longest-first order, and key heads that divide over the XCDs."""
    torch.manual_seed(15)
    check(B, S, NH, NKV, 64, True, None)


def test_inference_mode_and_another_stream():
    torch.manual_seed(16)
    bias = RelativePositionBias(4, 32, 64).cuda().bfloat16()
    with torch.no_grad():
        bias.weight.normal_()
    qkv, cache = rand(2, 300, 8 * 64), rand(2, 100, 2, 2, 64)
    n = torch.tensor([100, 41], dtype=torch.int32, device="cuda")

    def both():
        return (bias(qkv, nkv=2, causal=True),
                relative_attention_decode(qkv[:, :1, :256].view(2, 1, 4, 64), cache[:, :, 0], cache[:, :, 1], bias.weight, bias.buckets, n))

    with torch.no_grad():
        want = both()
    assert torch.equal(bias(qkv, nkv=2, causal=True), want[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.inference_mode():
        got = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_token_long_caches_of_different_lengths():
    torch.manual_seed(24)
    m = relative_position_buckets(32, 128, False).cuda()
    B, S, NH, NKV, D = 6, 9000, 4, 2, 64
    lengths = torch.tensor([9000, 1, 4097, 0, 8191, 260], dtype=torch.int32, device="cuda")
    check_token(rand(B, 2, NH, D), rand(B, S, NKV, D), rand(B, S, NKV, D), rand(32, NH), m, lengths)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,S,NH,NKV", [(1, 1031, 1, 1), (1, 640, 4, 2), (2, 777, 6, 2)])
def test_queries_cut_into_spans(B, S, NH, NKV, causal, D):
    torch.manual_seed(19)
    check(B, S, NH, NKV, D, causal, padded(B, S, 300) if B > 1 else None)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["empty", "holes", "left", "late"])
def test_masks_over_spans(kind, causal):
    """Keys cut over several workgroups, some of which find none that counts."""
    torch.manual_seed(20)
    B, S = 2, 700
    mask = padded(B, S, 90)
    if kind == "empty":
        mask[0] = 0
    elif kind == "holes":
        mask = (torch.rand(B, S, device="cuda") < 0.2).to(torch.uint8)
    elif kind == "left":
        mask = mask.flip(1).contiguous()
    elif kind == "late":
        mask = torch.zeros(B, S, dtype=torch.uint8, device="cuda")
        mask[:, 650:] = 1
    check(B, S, 2, 1, 64, causal, mask, poison=True)


@pytest.mark.parametrize("value", [-(2.0**20), 99614720.0])
def test_one_large_bias_over_spans(value):
    """As test_one_large_bias_for_all, for out and dv of a batch whose keys and queries are cut."""
    torch.manual_seed(21)
    S, NH, D = 1100, 2, 64
    m = relative_position_buckets(32, 128).cuda()
    qkv = rand(1, S, 3 * NH * D)
    qkv[:, :, :2 * NH * D] *= 2.0**-8
    dout = rand(1, S, NH * D)
    leaf, table = qkv.clone().requires_grad_(), torch.full((32, NH), value, device="cuda").bfloat16()
    out = fused_relative_attention(leaf, NH, table, m)
    dv = torch.autograd.grad(out, leaf, dout)[0].double().view(1, S, 3, NH, D)[:, :, 2].transpose(1, 2)
    q, k, v = split(qkv, NH, NH)
    keep = torch.ones(1, 1, S, S, dtype=torch.bool, device="cuda")
    p, r = probabilities(q, k, torch.zeros(1, NH, S, S, device="cuda", dtype=torch.float64), keep, D ** -0.5)
    r += 2.1 * float((q @ k.transpose(2, 3).contiguous()).abs().amax()) * D ** -0.5
    do = dout.double().view(1, S, NH, D).transpose(1, 2).contiguous()
    pt = p.transpose(2, 3).contiguous()
    for got, want, tol in ((out.detach().double().view(1, S, NH, D).transpose(1, 2), p @ v, (2 * U + 2 * r) * (p @ v.abs())),
                           (dv, pt @ do, (2 * U + 2 * r + S * E32) * (pt @ do.abs()))):
        assert ((got - want).abs() <= tol * (1 + U) + U * want.abs() + 1e-30).all()


def test_spans_captured_and_repeated():
    """The spans' workspaces inside a graph: every replay is the eager result, bit for bit."""
    torch.manual_seed(22)
    m = relative_position_buckets(32, 128, False).cuda()
    qkv, table, dout = rand(1, 900, 4 * 64).requires_grad_(), rand(32, 2).requires_grad_(), rand(1, 900, 128)

    def step():
        out = fused_relative_attention(qkv, 2, table, m, nkv=1, causal=True)
        return [out.detach(), *torch.autograd.grad(out, (qkv, table), dout)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            qkv.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_launches_beyond_the_grid_are_refused():
    m = relative_position_buckets().cuda()
    t = rand(32, 1)
    with pytest.raises(RuntimeError, match="too many rows"):
        fused_relative_attention(torch.zeros(1 << 22, 1, 192, dtype=torch.bfloat16, device="cuda"), 1, t, m)
    q, k = rand(1, 1, 1, 64).expand(1 << 22, 1, 1, 64), rand(1, 4, 1, 64).expand(1 << 22, 4, 1, 64)
    with pytest.raises(RuntimeError, match="too many rows"):
        relative_attention_decode(q, k, k, t, m, torch.ones(1 << 22, dtype=torch.int32, device="cuda"))
    n = 70000
    q, k = rand(1, 1, 1, 64).expand(n, 1, 1, 64), rand(1, 4, 1, 64).expand(n, 4, 1, 64)
    out = relative_attention_decode(q, k, k, t, m, torch.full((n,), 3, dtype=torch.int32, device="cuda"))
    assert torch.equal(out, out[:1].expand_as(out))
    out = fused_relative_attention(rand(1, 1, 192).expand(n, 1, 192).contiguous(), 1, t, m)
    assert torch.equal(out, out[:1].expand_as(out))
