"""Weight gradients on the side stream (set_wgrad_overlap): what it reads stays
as it was until it has run.

The CPU tests stand the library's products and the streams in by plain ones and
look at addresses alone: the side stream's product is taken to run as late as
it may, so memory that it was given must not be written before."""

import contextlib

import pytest
import torch

from gradient_accumulation_tf_estimator_amd import create_optimizer
from gradient_accumulation_tf_estimator_amd.engine.graphs import GraphedTrainLoop
from gradient_accumulation_tf_estimator_amd.models.bert import BertConfig, BertForSequenceClassification
from gradient_accumulation_tf_estimator_amd.ops import fused, gemm


class Products:
    """gemm's entry points on the CPU; what the weight gradients were given is kept as addresses."""

    def __init__(self):
        self.read = []  # (first byte, one past the last) of each dy

    def linear_fwd(self, x, w, bias):
        return torch.nn.functional.linear(x, w, bias)

    def dgrad(self, dy, w):
        return dy @ w

    def wgrad_acc(self, x, dy, accum, *rest):
        self.read.append((dy.data_ptr(), dy.data_ptr() + dy.numel() * dy.element_size()))


class Stream:
    def wait_stream(self, other):
        pass


@pytest.fixture
def overlap(monkeypatch):
    products = Products()
    for name in ("linear_fwd", "dgrad", "wgrad_acc"):
        monkeypatch.setattr(gemm, name, getattr(products, name))
    monkeypatch.setattr(fused, "wgrad_stream", Stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream())
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: None)
    monkeypatch.setattr(fused, "_GROUPED_WGRAD", False)
    monkeypatch.setattr(fused, "_WGRAD_OVERLAP", True)
    yield products
    fused.release_held_wgrads()


class OneGradientForBoth(torch.autograd.Function):
    """x + residual with one tensor as both gradients, as the RMS norm's node returns it."""

    @staticmethod
    def forward(ctx, x, residual):
        return x + residual

    @staticmethod
    def backward(ctx, dy):
        dx = dy * 1.0
        return dx, dx


class Sink(torch.autograd.Function):
    """Keeps the gradient that arrives."""

    @staticmethod
    def forward(ctx, x, kept):
        ctx.kept = kept
        return x.clone()

    @staticmethod
    def backward(ctx, dy):
        ctx.kept.append(dy)
        return dy, None


@pytest.mark.parametrize("join", [OneGradientForBoth.apply, torch.add])
@pytest.mark.parametrize("shape", [(6, 8), (2, 3, 8)])
def test_the_other_branch_is_not_added_into_what_the_side_stream_reads(overlap, join, shape):
    lin = fused.DirectLinear(8, 8, bias=False)
    lin._accum_view_w = torch.zeros(8, 8)
    leaf, kept = torch.randn(shape, requires_grad=True), []
    x = Sink.apply(leaf, kept)
    y = join(fused._DirectLinearFn.apply(x, lin.weight, None, lin), x)
    (y * 2.0).backward(torch.randn(shape))
    (lo, hi), summed = overlap.read[0], kept[0]
    at = summed.data_ptr()
    assert not lo <= at < hi


class Library:
    """The extension's products on the CPU; each call's stream and workspace are kept."""

    def __init__(self):
        self.on_side, self.calls = False, []

    @contextlib.contextmanager
    def side(self, stream):
        self.on_side = True
        yield
        self.on_side = False

    def lt_algo_count(self, *shape):
        return 3

    wgrad_algo_count = lt_algo_count

    def lt_linear(self, x, w, bias, algo):
        self.calls.append((self.on_side, 0))
        return x @ w.t()

    def lt_dgrad(self, dy, w, algo):
        self.calls.append((self.on_side, 0))
        return dy @ w

    def wgrad_acc(self, x, dy, accum, algo=0, workspace=0):
        self.calls.append((self.on_side, workspace))


def test_products_that_run_at_once_share_no_workspace(monkeypatch):
    """Among them those that the tuner times."""
    lib = Library()

    def tune(key, count, run):
        for i in range(count):
            run(i)
        return 0

    monkeypatch.setattr(gemm, "require_hip", lambda: lib)
    monkeypatch.setattr(gemm, "_tune", tune)
    monkeypatch.setattr(gemm, "_cache", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(fused, "wgrad_stream", Stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream())
    monkeypatch.setattr(torch.cuda, "stream", lib.side)
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: None)
    monkeypatch.setattr(fused, "_GROUPED_WGRAD", False)
    monkeypatch.setattr(fused, "_WGRAD_OVERLAP", True)
    lin = fused.DirectLinear(8, 8, bias=False)
    lin._accum_view_w = torch.zeros(8, 8)
    x = torch.randn(6, 8, requires_grad=True)
    for overlap in (True, False):
        monkeypatch.setattr(fused, "_WGRAD_OVERLAP", overlap)
        fused._DirectLinearFn.apply(x, lin.weight, None, lin).sum().backward()
    fused.release_held_wgrads()
    side, main = ({w for on, w in lib.calls if on == which} for which in (True, False))
    assert side and main and not side & main


STEPS = 3


def encoder(norm):
    torch.manual_seed(0)
    model = BertForSequenceClassification(BertConfig(
        vocab_size=50, hidden_size=256, num_layers=2, num_heads=4, intermediate_size=512, max_position_embeddings=96,
        relative_buckets=16, relative_max_distance=20, norm=norm, layer_norm_eps=1e-6))
    model = model.cuda().bfloat16()
    op = create_optimizer(model, 1e-3, 10, gradient_accumulation_multiplier=STEPS + 1, clip_norm=None)
    return model, op.engine


def near(model, engine, want):
    """Accumulated gradients against those of the main stream alone: the same kernels on the same values. Should the
    library's products add in another order, roundings to bf16 on the way may fall the other way: some twelve of 2^-8
    a layer and side, two layers."""
    for (name, p), w in zip(model.named_parameters(), want):
        got = engine.state.accum_view(p).float()
        assert float((got - w).norm()) <= 2 * 24 * 2.0**-8 * float(w.norm()) + 1e-30, name


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_encoder_with_the_side_stream_and_without(norm, monkeypatch):
    monkeypatch.setattr(fused, "_GROUPED_WGRAD", False)
    monkeypatch.setattr(fused, "_WGRAD_OVERLAP", False)
    ids = torch.randint(0, 50, (8, 96), device="cuda")
    labels = torch.randint(0, 2, (8,), device="cuda")
    mask = (torch.arange(96)[None] < torch.linspace(30, 96, 8)[:, None]).long().cuda()

    def loss(model):
        return torch.nn.functional.cross_entropy(model(ids, attention_mask=mask).float(), labels)

    model, engine = encoder(norm)
    want = []
    for _ in range(STEPS):
        loss(model).backward()
        engine.accumulate()
        want.append([engine.state.accum_view(p).float().clone() for p in model.parameters()])
    assert any(float(w.norm()) > 0 for w in want[0])

    fused.set_wgrad_overlap(True)
    model, engine = encoder(norm)
    for step in range(STEPS):
        loss(model).backward()
        assert fused._wgrad_held
        engine.accumulate()
        assert not fused._wgrad_held
        engine._join_wgrad_stream()
        near(model, engine, want[step])

    model, engine = encoder(norm)
    loop = GraphedTrainLoop(engine, lambda: loss(model))
    for step in range(STEPS):
        loop.step()
        torch.cuda.synchronize()
        near(model, engine, want[step])
        torch.randn(1000, device="cuda").sum().item()


def test_switching_it_off_waits_for_what_is_running(monkeypatch):
    """The engine joins the side stream only while the switch is on."""
    waited = []

    class Main:
        def wait_stream(self, other):
            waited.append(other)

    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Main())
    monkeypatch.setattr(fused, "_wgrad_stream", None)
    monkeypatch.setattr(fused, "_WGRAD_OVERLAP", False)
    fused.set_wgrad_overlap(True)
    fused.set_wgrad_overlap(False)  # nothing ran there
    assert not waited
    fused.set_wgrad_overlap(True)
    monkeypatch.setattr(fused, "_wgrad_stream", "side")
    fused.set_wgrad_overlap(True)
    assert not waited
    fused.set_wgrad_overlap(False)
    assert waited == ["side"]
    fused.set_wgrad_overlap(False)
    assert waited == ["side"]
