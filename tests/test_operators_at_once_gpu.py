"""Calls of the operators at the same time on several streams, and captured
calls replayed beside eager ones: every result is the lone call's, bit by bit
(their sums have a fixed order, and nothing is shared between calls)."""

import pytest
import torch

from gradient_accumulation_tf_estimator_amd import clip_by_global_norm
from gradient_accumulation_tf_estimator_amd.ops.relative_attention import (
    fused_relative_attention,
    relative_attention_decode,
    relative_position_buckets,
)
from gradient_accumulation_tf_estimator_amd.ops.rms_norm import add_rms_norm, rms_norm_fp8

pytestmark = pytest.mark.gpu


def rand(*shape, dtype=torch.bfloat16):
    return torch.randn(shape, device="cuda").to(dtype)


def attention(S):
    m, table = relative_position_buckets(32, 64, False).cuda(), rand(32, 4).requires_grad_()
    qkv, dout = rand(2, S, 8 * 64).requires_grad_(), rand(2, S, 4 * 64)

    def call():
        out = fused_relative_attention(qkv, 4, table, m, nkv=2, causal=True)
        return [out.detach(), *torch.autograd.grad(out, (qkv, table), dout)]
    return call, [qkv, dout]


def decode(S):
    m, table = relative_position_buckets(32, 64, False).cuda(), rand(32, 4)
    q, kv = rand(3, 2, 4, 128)[..., :64], rand(3, S, 2, 2, 64)
    n = torch.tensor([S, S // 2, 1], dtype=torch.int32, device="cuda")
    return lambda: [relative_attention_decode(q, kv[:, :, 0], kv[:, :, 1], table, m, n)], [q, kv]


def norm(R, H):
    x, r, w = rand(R, H).requires_grad_(), rand(R, H).requires_grad_(), rand(H).requires_grad_()
    dy, dh = rand(R, H), rand(R, H)

    def call():
        y, h = add_rms_norm(x, w, r)
        with torch.no_grad():
            q, s, _ = rms_norm_fp8(x, w, r, group=64)
        return [y.detach(), h.detach(), *torch.autograd.grad((y, h), (x, r, w), (dy, dh)), q.view(torch.uint8), s]
    return call, [x, r, dy]


def clip(count):
    ts = [rand(1000 + 37 * i, dtype=(torch.bfloat16, torch.float32)[i % 2]) for i in range(count)]
    out = [torch.empty_like(t) for t in ts]

    def call():
        got, n = clip_by_global_norm(ts, 1.0, out=out)
        return [t.clone() for t in got] + [n]
    return call, ts


MAKE = [lambda: attention(300), lambda: attention(1300), lambda: decode(900), lambda: norm(700, 1024), lambda: norm(50, 4096),
        lambda: clip(150)]


def same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_on_several_streams_at_once():
    torch.manual_seed(1)
    calls = [make()[0] for make in MAKE for _ in range(2)]  # two of each, with values of their own
    want = [call() for call in calls]
    streams = [torch.cuda.Stream() for _ in range(4)]
    for _ in range(3):
        got = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for i, call in enumerate(calls):
            with torch.cuda.stream(streams[i % 4]):
                got.append(call())
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("which", range(len(MAKE)))
def test_two_graphs_in_turn_with_eager_calls(which):
    torch.manual_seed(2)
    (one, inputs), (two, _) = MAKE[which](), MAKE[which]()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one(), two()
    torch.cuda.current_stream().wait_stream(side)
    graphs, got = [], []
    for call in (one, two):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=graphs[0].pool() if len(graphs) > 1 else None):
            got.append(call())
    for _ in range(3):
        with torch.no_grad():
            for t in inputs:
                t.normal_()
        for graph, call, result in zip(graphs, (one, two), got):
            graph.replay()
            torch.cuda.synchronize()
            assert same([t.clone() for t in result], call())
