"""Weight gradients on the side stream (set_wgrad_overlap): what it reads stays
as it was until it has run.

The CPU tests stand the library's products and the streams in by plain ones and
look at addresses alone: the side stream's product is taken to run as late as
it may, so memory that it was given must not be written before."""

import contextlib

import pytest
import torch

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
