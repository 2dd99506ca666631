"""Layer norm, the dense product with an epilogue and the mixture-of-experts layer recorded into graphs and on streams of their own.

Behind the other tests: torch hands out its streams in turn, and what those tests find on theirs should not change."""

import pytest
import torch

from tests import cases
from tests.test_gpu_dense_act import _inputs as dense_inputs
from tests.test_gpu_layer_norm import EPS
from tests.test_gpu_layer_norm import _inputs as norm_inputs
from tests.test_gpu_moe import _experts as moe_experts
from tests.test_gpu_moe import _layer as moe_weights

pytestmark = pytest.mark.gpu


def test_captured_dense_linear_act(gpu):
    from neuropress_amd import kernels

    for m, n, k in ((1, 512, 1024), (20, 512, 4096), (96, 256, 8192)):
        x, w, b, r = (t.to(gpu) for t in dense_inputs(m, n, k, torch.bfloat16))
        stream = torch.cuda.Stream()
        kernels.dense_linear_act(x, w, b, "silu", r)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y = kernels.dense_linear_act(x, w, b, "silu", r)
        for seed in range(4):
            nx, _, _, nr = dense_inputs(m, n, k, torch.bfloat16, seed)
            x.copy_(nx)
            r.copy_(nr)
            want = kernels.dense_linear_act(x, w, b, "silu", r)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


def test_captured_layer_norm_forward_and_backward(gpu):
    from neuropress_amd import kernels

    x, w, b, dy = (t.to(gpu) for t in norm_inputs(300, 1000, torch.bfloat16))

    def step():
        y, mean, rstd = kernels.layer_norm_stats(x, w, b, EPS)
        return (y, *kernels.layer_norm_backward(dy, x, w, mean, rstd))

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step()
    for seed in range(4):
        nx, _, _, ndy = norm_inputs(300, 1000, torch.bfloat16, seed=seed)
        x.copy_(nx)
        dy.copy_(ndy)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want))


def test_captured_training_step(gpu):
    """Forward and backward through autograd, recorded after a step on the same side stream whose graph is gone."""
    from neuropress_amd import kernels

    x, w, b, dy = (t.to(gpu) for t in norm_inputs(70, 640, torch.bfloat16))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]

    def step():
        for t in leaves:
            t.grad = None
        kernels.layer_norm(*leaves, EPS).backward(dy)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    for seed in range(3):
        nx, _, _, ndy = (t.to(gpu) for t in norm_inputs(70, 640, torch.bfloat16, seed=seed))
        with torch.no_grad():
            leaves[0].copy_(nx)
        dy.copy_(ndy)
        graph.replay()
        torch.cuda.synchronize()
        _, mean, rstd = kernels.layer_norm_stats(nx, w, b, EPS)
        assert all(torch.equal(t.grad, c) for t, c in zip(leaves, kernels.layer_norm_backward(ndy, nx, w, mean, rstd)))


def test_captured_twice_and_on_two_streams(gpu):
    """Two captured calls and eager ones, replayed in turn and side by side: each has scratch of its own."""
    from neuropress_amd import kernels

    layer, _ = moe_weights(9, 16, 256, 512, torch.float16, 4)
    experts = moe_experts(layer)
    xs = [torch.randn(m, 256, generator=cases.gen(m)).half().to(gpu) for m in (3, 12)]
    for x in xs:
        kernels.moe_layer(x, experts, 4)
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in xs], [torch.cuda.CUDAGraph() for _ in xs], []
    for x, st, graph in zip(xs, streams, graphs):
        with torch.cuda.graph(graph, stream=st):
            outs.append(kernels.moe_layer(x, experts, 4))
    for seed in range(5):
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=cases.gen(seed)).half())
        want = [kernels.moe_layer(x, experts, 4) for x in xs]
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens", [1, 5, 32])
def test_captured_feed_forward_half_of_a_block(gpu, tokens, dtype):
    from neuropress_amd import kernels

    h, i, g = 256, 512, cases.gen(tokens)
    rand = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).to(dtype).to(gpu)
    x, n1, b1, n2, b2, up, ub, down = rand(tokens, h), rand(h), rand(h), rand(h), rand(h), rand(i, h), rand(i), rand(h, i)
    experts = moe_experts(moe_weights(3, 8, h, 128, dtype, 4)[0])

    def block():
        hidden = kernels.dense_linear_act(kernels.layer_norm(x, n1, b1), up, ub, "gelu")
        mid = kernels.dense_linear_act(hidden, down, residual=x)
        return mid, kernels.moe_layer(kernels.layer_norm(mid, n2, b2), experts, 2)

    block()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block()
    for k in range(3):
        x.copy_(torch.randn(tokens, h, generator=cases.gen(k)))
        again = block()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, again))


def test_capture_beside_an_eager_graph_of_the_same_leaves(gpu):
    """Refused in the backward pass, before torch waits for the other graph's stream inside the capture; once that graph is gone the same step is captured."""
    from neuropress_amd import kernels

    x, w, b, dy = (t.to(gpu) for t in norm_inputs(20, 320, torch.bfloat16))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    alive = kernels.layer_norm(*leaves, EPS)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            kernels.layer_norm(*leaves, EPS).backward(dy)
    torch.cuda.synchronize()
    assert torch.equal(alive, kernels.layer_norm(*leaves, EPS)) and all(t.grad is None for t in leaves)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        kernels.layer_norm(*leaves, EPS).backward(dy)
    graph.replay()
    torch.cuda.synchronize()
    _, mean, rstd = kernels.layer_norm_stats(x, w, b, EPS)
    assert all(torch.equal(t.grad, c) for t, c in zip(leaves, kernels.layer_norm_backward(dy, x, w, mean, rstd)))
