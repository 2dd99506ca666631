"""Residual norm, gated product and adapters as a block uses them, recorded into graphs, and on streams of their own.

Behind the other tests: torch hands out its streams in turn, and what those tests find on theirs should not change."""

import pytest
import torch

from tests import cases

pytestmark = pytest.mark.gpu


def _block(gpu, dtype, h=256, i=384, seed=0):
    """A feed-forward half whose down projection is an int4 layer with adapters, between two residual norms."""
    from neuropress_amd import kernels
    from neuropress_amd.nn import NPAdapterLinear, NPLinear

    g = cases.gen(seed)
    rand = lambda *s, std=1.0, mean=0.0: (torch.randn(*s, generator=g) * std + mean).to(dtype).to(gpu)
    Q = cases.q4_layer(3, h, i)
    adapters = kernels.LowRankAdapters(rand(4, 8, i, std=i**-0.5), rand(4, h, 8, std=0.3), torch.tensor([0.5, 1.0, 2.0, 1.5], device=gpu))
    down = NPAdapterLinear(NPLinear(Q["blob"], Q["scale"], h, i, 32, 4, "sym", "cuda", compute_dtype=dtype).to(gpu), adapters)
    gate_up, bias = rand(2 * i, h, std=h**-0.5), rand(2 * i, std=0.1)
    w = [rand(h, std=0.1, mean=1.0) for _ in range(4)]
    gate = rand(h, std=0.3, mean=0.5)

    def run(x, attn, ids):
        stream, z = kernels.residual_norm(x, attn, w[0], w[1], gate, 0.5)
        y = down(kernels.gated_linear(z, gate_up, bias), ids)
        return (stream, y, *kernels.residual_norm(stream, y, w[2], w[3], gate, 0.5))

    return run


def _inputs(tokens, dtype, gpu, seed=0, h=256):
    g = cases.gen(seed)
    x, attn = (torch.randn(tokens, h, generator=g).to(dtype).to(gpu) for _ in range(2))
    return x, attn, torch.randint(-1, 4, (tokens,), generator=g).to(gpu)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens", [1, 5, 40, 300])
def test_captured_block(gpu, tokens, dtype):
    run, state = _block(gpu, dtype), _inputs(tokens, dtype, gpu)
    run(*state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*state)
    for seed in range(4):
        for t, new in zip(state, _inputs(tokens, dtype, gpu, seed)):
            t.copy_(new)
        want = run(*state)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(bool(t.isfinite().all()) for t in out)


@pytest.mark.parametrize("tokens", [3, 150])
def test_two_captured_blocks_side_by_side(gpu, tokens):
    """Replayed at once on two streams: each has scratch of its own."""
    run = _block(gpu, torch.bfloat16)
    states = [_inputs(tokens, torch.bfloat16, gpu, seed) for seed in (1, 2)]
    for s in states:
        run(*s)
    torch.cuda.synchronize()
    streams, graphs, outs = [torch.cuda.Stream() for _ in states], [torch.cuda.CUDAGraph() for _ in states], []
    for s, st, graph in zip(states, streams, graphs):
        with torch.cuda.graph(graph, stream=st):
            outs.append(run(*s))
    for seed in range(4):
        for k, s in enumerate(states):
            for t, new in zip(s, _inputs(tokens, torch.bfloat16, gpu, 10 * k + seed)):
                t.copy_(new)
        want = [run(*s) for s in states]
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o, w in zip(outs, want) for a, b in zip(o, w))


def test_eager_on_two_streams(gpu):
    run = _block(gpu, torch.float16)
    states = [_inputs(t, torch.float16, gpu, t) for t in (7, 90, 200)]
    want = [run(*s) for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(5):
        outs = []
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                outs.append(run(*s))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for o, w in zip(outs, want) for a, b in zip(o, w))


def _training(gpu, m, h, i):
    from neuropress_amd import kernels

    g = cases.gen(m)
    rand = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).bfloat16().to(gpu)
    leaves = [t.requires_grad_() for t in (rand(m, h), rand(m, h), rand(h, std=0.1), rand(h, std=0.1), rand(h), rand(2 * i, h, std=h**-0.5), rand(2 * i))]
    dh = rand(m, i)

    def step():
        for t in leaves:
            t.grad = None
        x, y, w, p, gate, gate_up, bias = leaves
        stream, z = kernels.residual_norm(x, y, w, p, gate, 0.7)
        torch.autograd.backward((kernels.gated_linear(z, gate_up, bias), stream), (dh, dh @ dh.new_ones(i, h)))

    return leaves, dh, step


def test_captured_training_step(gpu):
    """Forward and backward through autograd, recorded after a step on the same side stream whose graph is gone."""
    leaves, dh, step = _training(gpu, 70, 320, 200)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    captured = [t.grad for t in leaves]
    for seed in range(3):
        with torch.no_grad():
            leaves[0].copy_(torch.randn(70, 320, generator=cases.gen(seed)))
        dh.copy_(torch.randn(70, 200, generator=cases.gen(seed + 9)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        with torch.cuda.stream(stream):
            step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, t.grad) for a, t in zip(got, leaves))


def test_capture_beside_an_eager_graph_of_the_same_leaves(gpu):
    """Refused in the backward pass, before torch waits for the other graph's stream inside the capture; once that graph is gone the same step is captured."""
    from neuropress_amd import kernels

    leaves, dh, step = _training(gpu, 20, 64, 48)
    x, y, w, p, gate, gate_up, bias = leaves
    for make, back in ((lambda: kernels.gated_linear(x, gate_up, bias), dh), (lambda: kernels.residual_norm(x, y, w, p, gate)[1], x.detach())):
        alive = make()
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="cannot be captured"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
                make().backward(back)
        torch.cuda.synchronize()
        assert all(t.grad is None for t in leaves) and torch.equal(alive, make())
        del alive
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            make().backward(back)
        graph.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad(make(), x, back)[0]
        assert torch.equal(x.grad, want)
        for t in leaves:
            t.grad = None


@pytest.mark.parametrize("which", range(5))
def test_capture_beside_an_eager_graph_of_one_leaf(gpu, which):
    """The same where x, y, a weight or the gate is the only leaf, kept by the node or not."""
    from neuropress_amd import kernels

    g = cases.gen(which)
    given = [torch.randn(s, generator=g).bfloat16().to(gpu) for s in ((20, 64), (20, 64), (64,), (64,), (64,))]
    leaf = given[which].requires_grad_()
    make = lambda: kernels.residual_norm(*given, 0.7)[1]
    back = torch.ones(20, 64, device=gpu, dtype=torch.bfloat16)
    alive = make()
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=stream):
            make().backward(back)
    torch.cuda.synchronize()
    assert leaf.grad is None
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        make().backward(back)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(leaf.grad, torch.autograd.grad(make(), leaf, back)[0])


def test_captured_call_of_a_node_by_itself(gpu):
    """Nothing goes on to the leaves there, so another stream's graph of them is no hindrance."""
    from neuropress_amd import kernels

    g = cases.gen(4)
    x, y, w = (torch.randn(s, generator=g).bfloat16().to(gpu).requires_grad_() for s in ((20, 64), (20, 64), (64,)))
    ds, dz = (torch.randn(20, 64, generator=g).bfloat16().to(gpu) for _ in range(2))
    out = kernels.residual_norm(x, y, w)
    want = torch.autograd.grad(out, (x, y, w), (ds, dz), retain_graph=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = out[0].grad_fn(ds, dz)[:3]
    for _ in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
