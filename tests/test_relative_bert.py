"""The encoder with relative position bias and RMS norms: the operators run
together as a model, a training step and a server use them."""

import math

import pytest
import torch

from gradient_accumulation_tf_estimator_amd import clip_by_global_norm, create_optimizer
from gradient_accumulation_tf_estimator_amd.models.bert import BertConfig, BertForSequenceClassification
from gradient_accumulation_tf_estimator_amd.ops.relative_attention import fused_relative_attention
from gradient_accumulation_tf_estimator_amd.ops.rms_norm import FusedAddRMSNorm, add_rms_norm, rms_norm_fp8
from gradient_accumulation_tf_estimator_amd.serving import GraphedPredictor


def config(**kw):
    return BertConfig(**{**dict(vocab_size=50, hidden_size=256, num_layers=2, num_heads=4, intermediate_size=512,
                                max_position_embeddings=96, relative_buckets=16, relative_max_distance=20, norm="rms",
                                layer_norm_eps=1e-6), **kw})


def build(cfg, seed=0):
    torch.manual_seed(seed)
    model = BertForSequenceClassification(cfg)
    with torch.no_grad():
        if model.bert.relative_attention_bias is not None:
            model.bert.relative_attention_bias.weight.normal_(std=0.5)
        for m in model.modules():
            if isinstance(m, FusedAddRMSNorm):
                m.weight.add_(0.1 * torch.randn_like(m.weight))
    return model


def batch(B, S, device="cpu"):
    ids = torch.randint(0, 50, (B, S), device=device)
    labels = torch.randint(0, 2, (B,), device=device)
    n = torch.linspace(max(1, S // 3), S, B).round().long()
    mask = (torch.arange(S)[None] < n[:, None]).long().to(device)
    return ids, labels, mask


@pytest.mark.parametrize("fused", [True, False])
def test_model_gradients_against_differences(fused):
    model = build(config(hidden_size=16, intermediate_size=32, fused=fused)).double()
    ids, labels, mask = batch(3, 7)
    loss = lambda: torch.nn.functional.cross_entropy(model(ids, attention_mask=mask), labels)  # noqa: E731
    params = list(model.parameters())
    grads = torch.autograd.grad(loss(), params, allow_unused=True)
    names = [n for n, _ in model.named_parameters()]
    table = names.index("bert.relative_attention_bias.weight")
    assert grads[table].abs().sum() > 0
    for i, (p, g) in enumerate(zip(params, grads)):
        if g is None:
            continue
        d = torch.randn_like(p)
        with torch.no_grad():
            keep, ends = p.clone(), []
            for h in (1e-5, -1e-5):
                p.copy_(keep + h * d)
                ends.append(float(loss()))
            p.copy_(keep)
        diff = (ends[0] - ends[1]) / 2e-5
        # central differences: h^2 of the third derivative, and 2^-53 / h of the loss
        assert abs(diff - float((g * d).sum())) <= 1e-6 + 1e-5 * abs(diff), names[i]


def test_weight_decay_leaves_the_new_parameters_alone():
    model = build(config())
    op = create_optimizer(model, 1e-3, 10, gradient_accumulation_multiplier=1)
    state = op.engine.state
    decayed = {s.name for s in state.layout.slices if s.decay}
    assert not any("relative_attention_bias" in n or "LayerNorm" in n for n in decayed)


def test_config_refusals():
    with pytest.raises(ValueError, match="dropout"):
        build(config(dropout=0.1))
    with pytest.raises(ValueError, match="norm"):
        build(config(norm="batch"))


def test_the_defaults_are_the_model_that_was():
    model = BertForSequenceClassification(config(relative_buckets=0, norm="layer"))
    assert model.bert.relative_attention_bias is None
    assert not any(isinstance(m, FusedAddRMSNorm) for m in model.modules())


@pytest.mark.gpu
def test_model_is_its_operators():
    """A layer's output is that of its operators in turn, bit by bit."""
    model = build(config()).cuda().bfloat16().eval()
    bias, layer = model.bert.relative_attention_bias, model.bert.encoder[0]
    ids, _, mask = batch(4, 70, "cuda")
    with torch.no_grad():
        x = model.bert.embeddings(ids)
        got = layer(x, mask8=mask.to(torch.uint8), relative=bias)
        a = fused_relative_attention(layer.attention.qkv(x), 4, bias.weight, bias.buckets, mask8=mask.to(torch.uint8))
        h, _ = add_rms_norm(layer.attention_output(a), layer.attention_LayerNorm.weight, x, eps=1e-6)
        f = layer.output(layer.intermediate_act(layer.intermediate(h)))
        want, _ = add_rms_norm(f, layer.output_LayerNorm.weight, h, eps=1e-6)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("S", [33, 96])
def test_training_bound_to_an_engine_and_not(S):
    """The same model with its gradients in the engine's buffer and in .grad."""
    cfg = config()
    ids, labels, mask = batch(8, S, "cuda")
    free = build(cfg).cuda().bfloat16()
    torch.nn.functional.cross_entropy(free(ids, attention_mask=mask).float(), labels).backward()
    bound = build(cfg).cuda().bfloat16()
    op = create_optimizer(bound, 1e-3, 10, gradient_accumulation_multiplier=2, clip_norm=1.0)
    loss = torch.nn.functional.cross_entropy(bound(ids, attention_mask=mask).float(), labels)
    loss.backward()
    op.engine.accumulate()
    got = {n: op.engine.state.accum_view(p).view(p.shape) for n, p in bound.named_parameters()}
    for n, p in free.named_parameters():
        if p.grad is None or float(p.grad.float().norm()) == 0:
            continue
        # both compute in bf16 with different products: some twelve roundings of 2^-8 a layer, two layers, each side
        off = float((got[n] - p.grad.float()).norm()) / float(p.grad.float().norm())
        assert off <= 2 * 24 * 2.0**-8, (n, off)


@pytest.mark.gpu
def test_clip_and_step_without_an_engine():
    model = build(config()).cuda().bfloat16()
    ids, labels, mask = batch(8, 50, "cuda")
    torch.nn.functional.cross_entropy(model(ids, attention_mask=mask).float(), labels).backward()
    grads = [p.grad for p in model.parameters() if p.grad is not None]
    n = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    want = [g.double() * min(1.0, 1e-2 / n) for g in grads]
    _, norm = clip_by_global_norm(grads, 1e-2, out=grads)
    assert abs(float(norm) - n) <= 2.0**-23 * n
    for g, w in zip(grads, want):
        assert ((g.double() - w).abs() <= (2.0**-8 + 2.0**-22) * w.abs() + 1e-38).all()


@pytest.mark.gpu
def test_served_from_a_graph():
    model = build(config()).cuda().bfloat16().eval()
    ids, _, mask = batch(5, 64, "cuda")
    pred = GraphedPredictor(model, ids, example_mask=mask)
    for seed in range(3):
        torch.manual_seed(seed)
        ids = torch.randint(0, 50, ids.shape, device="cuda")
        mask = mask.flip(0).contiguous()
        with torch.no_grad():
            want = model(ids, attention_mask=mask)
        assert torch.equal(pred(ids, mask=mask), want)


@pytest.mark.gpu
def test_eight_bit_norm_into_a_scaled_product():
    """q and its row scales as torch's scaled product takes them: y @ w^T up to the 8-bit roundings of both sides."""
    torch.manual_seed(3)
    R, H, N = 64, 256, 128
    x, r = (torch.randn(R, H, device="cuda").bfloat16() for _ in range(2))
    g = torch.ones(H, device="cuda").bfloat16()
    w = torch.randn(N, H, device="cuda")
    ws = w.abs().amax(1, keepdim=True) / 448
    wq = (w / ws).to(torch.float8_e4m3fn)
    q, s, _ = rms_norm_fp8(x, g, r)
    out = torch._scaled_mm(q, wq.t(), scale_a=s, scale_b=ws.t().contiguous(), out_dtype=torch.bfloat16)
    a, b = q.double() * s.double(), wq.double() * ws.double()
    want = a @ b.t()
    # the product of the same 8-bit values: sums in 32 bits, one rounding to bf16
    tol = 2.0**-8 * want.abs() + (H + 8) * 2.0**-24 * (a.abs() @ b.abs().t())
    assert ((out.double() - want).abs() <= tol).all()
