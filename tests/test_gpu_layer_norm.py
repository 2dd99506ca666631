"""Layer norm and its backward pass against the formulas in 64 bits.

Tolerances: half a step of the output type, plus what f32 arithmetic may add: sums of n terms are off by at most n 2^-24 times the sum of their magnitudes
(n the longest chain of additions of any kernel: less than H / 64 + 16 over a row, M / 64 + 100 over rows), and a handful of roundings of 2^-24 on every factor."""

import pytest
import torch

from tests import cases

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
EPS32 = 2.0**-24
EPS = 1e-5


def _half_step(ref, dtype):
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return ref.abs() * (torch.finfo(dtype).eps / 2) + tiny / 2


def _check(got, ref, slack, dtype, what):
    assert got.dtype == dtype and got.shape == ref.shape
    err, tol = (got.double().cpu() - ref).abs(), _half_step(ref, dtype) * 1.0001 + slack * (1 + torch.finfo(dtype).eps)
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert bool((err <= tol).all()), f"{what}: {worst:.2f} of the tolerance"


def _inputs(m, h, dtype, seed=0, affine=True):
    g = cases.gen(seed + 31 * m + h)
    x = torch.randn(m, h, generator=g) * 2 + torch.randn(m, 1, generator=g)
    x[:, :: max(1, h // 3)] *= 9
    w, b = (torch.randn(h, generator=g) * 0.3 + 1, torch.randn(h, generator=g) * 0.2) if affine else (None, None)
    dy = torch.randn(m, h, generator=g)
    return [None if t is None else t.to(dtype) for t in (x, w, b, dy)]


def _reference(x, w, b, eps=EPS):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * rstd
    y = xh * (1.0 if w is None else w.double()) + (0.0 if b is None else b.double())
    # the mean is off by n 2^-24 mean|x|, rstd by n + 8 of 2^-24 relative (and by what the mean's error adds, far less)
    n = x.shape[-1] / 64 + 16
    wa = 1.0 if w is None else w.double().abs()
    slack = EPS32 * ((n + 12) * xh.abs() * wa + (n + 2) * rstd * x.abs().mean(-1, keepdim=True) * wa + 2 * y.abs())
    return y, mean[:, 0], rstd[:, 0], slack


def _reference_back(dy, x, w, mean, rstd):
    """From the mean and rstd that the backward pass is given."""
    dy, x, mean, rstd = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    m, h = x.shape
    xh = (x - mean) * rstd
    g = dy * (1.0 if w is None else w.double())
    c1, c2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dx = rstd * (g - c1 - xh * c2)
    xe = xh.abs() + 2 * mean.abs() * rstd  # x - mean is rounded once, relative to itself; products follow
    n, r = h / 64 + 20, m / 64 + 100
    slack = EPS32 * rstd * (6 * g.abs() + n * g.abs().mean(-1, keepdim=True) + (n + 8) * xe * (g * xh).abs().mean(-1, keepdim=True))
    dw, db = (dy * xh).sum(0), dy.sum(0)
    return (dx, slack), (dw, EPS32 * (r + 6) * (dy * xe).abs().sum(0)), (db, EPS32 * r * dy.abs().sum(0))


SHAPES = [(1, 1), (3, 2), (5, 7), (2, 8), (1, 640), (7, 4096), (130, 2048), (3, 8192), (5, 100), (2, 16384), (509, 333), (6, 12288 + 8), (2, 40000), (1025, 512),
          (4099, 72)]  # fmt: skip


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,h", SHAPES)
def test_forward(gpu, dtype, m, h):
    from neuropress_amd import kernels

    x, w, b, _ = _inputs(m, h, dtype)
    y, mean, rstd = kernels.layer_norm_stats(x.to(gpu), w.to(gpu), b.to(gpu), EPS)
    ref, mean_ref, rstd_ref, slack = _reference(x, w, b)
    _check(y, ref, slack, dtype, "y")
    assert torch.equal(kernels.layer_norm(x.to(gpu), w.to(gpu), b.to(gpu), EPS), y)
    n = h / 64 + 16
    assert bool(((mean.double().cpu() - mean_ref).abs() <= EPS32 * (n + 2) * x.double().abs().mean(-1)).all())
    # the variance: n roundings of its sum, and the square of the mean's own error
    assert bool(((rstd.double().cpu() - rstd_ref).abs() <= EPS32 * (n + 8) * rstd_ref + rstd_ref**3 * (EPS32 * (n + 2) * x.double().abs().mean(-1)) ** 2).all())


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("m,h", [(9, 1024), (9, 77)])
def test_without_weight_or_bias(gpu, m, h, weight, bias):
    from neuropress_amd import kernels

    x, w, b, dy = _inputs(m, h, torch.float16)
    w, b = (w if weight else None), (b if bias else None)
    on = [None if t is None else t.to(gpu) for t in (x, w, b, dy)]
    ref, _, _, slack = _reference(x, w, b)
    y, mean, rstd = kernels.layer_norm_stats(*on[:3])
    _check(y, ref, slack, torch.float16, "y")
    refs = _reference_back(dy, x, w, mean.cpu(), rstd.cpu())
    for got, (want, tol), name in zip(kernels.layer_norm_backward(on[3], on[0], on[1], mean, rstd), refs, ("dx", "dw", "db")):
        _check(got, want, tol, torch.float16, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,h", SHAPES)
def test_backward(gpu, dtype, m, h):
    from neuropress_amd import kernels

    x, w, _, dy = _inputs(m, h, dtype)
    _, mean, rstd = kernels.layer_norm_stats(x.to(gpu), None, None, EPS)
    got = kernels.layer_norm_backward(dy.to(gpu), x.to(gpu), w.to(gpu), mean, rstd)
    for t, (ref, slack), what in zip(got, _reference_back(dy, x, w, mean.cpu(), rstd.cpu()), ("dx", "dw", "db")):
        _check(t, ref, slack, dtype, what)
    again = kernels.layer_norm_backward(dy.to(gpu), x.to(gpu), w.to(gpu), mean, rstd)
    assert all(torch.equal(a, b) for a, b in zip(got, again)), "the same inputs, other bits"
    # every choice of what is asked for gives the same
    for needs in [(True, False, False), (False, True, False), (False, False, True), (False, False, False)]:
        some = kernels.layer_norm_backward(dy.to(gpu), x.to(gpu), w.to(gpu), mean, rstd, needs=needs)
        assert all((a is None) != n and (a is None or torch.equal(a, b)) for a, b, n in zip(some, got, needs))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h,ld,at", [(256, 512, 0), (256, 257, 1), (4096, 4100, 3), (1000, 1001, 0)])
def test_row_distances_and_odd_addresses(gpu, dtype, h, ld, at):
    from neuropress_amd import kernels

    m = 21
    x, w, b, dy = _inputs(m, h, dtype)

    def strided(t):
        room = torch.full((m * ld + at,), float("nan"), dtype=dtype, device=gpu)
        view = room[at:].as_strided((m, h), (ld, 1))
        view.copy_(t)
        return view

    xs, dys = strided(x), strided(dy)
    y, mean, rstd = kernels.layer_norm_stats(xs, w.to(gpu), b.to(gpu), EPS)
    ref, _, _, slack = _reference(x, w, b)
    _check(y, ref, slack, dtype, "y")
    for t, (want, tol), what in zip(kernels.layer_norm_backward(dys, xs, w.to(gpu), mean, rstd), _reference_back(dy, x, w, mean.cpu(), rstd.cpu()), ("dx", "dw", "db")):
        _check(t, want, tol, dtype, what)
    # weight and bias between two 16-byte addresses
    both = torch.cat([w[:1], w, b]).to(gpu)
    assert torch.equal(kernels.layer_norm(xs, both[1 : h + 1], both[h + 1 :], EPS), y)


def test_no_rows_and_leading_dimensions(gpu):
    from neuropress_amd import kernels

    w, b = torch.ones(64, device=gpu), torch.zeros(64, device=gpu)
    empty = torch.empty(2, 0, 64, device=gpu)
    y, mean, rstd = kernels.layer_norm_stats(empty, w, b)
    assert y.shape == (2, 0, 64) and mean.shape == rstd.shape == (2, 0)
    dx, dw, db = kernels.layer_norm_backward(empty, empty, w, mean, rstd)
    assert dx.shape == (2, 0, 64) and not dw.any() and not db.any() and dw.shape == db.shape == (64,)
    x = torch.randn(3, 5, 64, device=gpu)
    assert torch.equal(kernels.layer_norm(x, w, b), kernels.layer_norm(x.reshape(15, 64), w, b).reshape(3, 5, 64))
    assert torch.equal(kernels.layer_norm(x[:, ::2], w, b), kernels.layer_norm(x, w, b)[:, ::2])
    assert torch.equal(kernels.layer_norm(x[0, :1].expand(4, 64), w, b), kernels.layer_norm(x, w, b)[0, :1].expand(4, 64))
    assert kernels.layer_norm(x[0, 0], w, b).shape == (64,)


def test_rows_that_are_constant_not_finite_or_far_from_zero(gpu):
    from neuropress_amd import kernels

    x = torch.randn(5, 512, generator=cases.gen(3))
    x[0] = 3.0  # no variance: eps alone, exactly zero
    x[1, 7] = float("inf")
    x[2, 9] = float("nan")
    x[3] += 4096.0  # a mean far larger than the deviation
    y = kernels.layer_norm(x.to(gpu), None, None, EPS).cpu()
    assert not y[0].any() and y[1].isnan().all() and y[2].isnan().all()
    ref, _, _, slack = _reference(x[3:], None, None)
    _check(y[3:], ref, slack, torch.float32, "y")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weight,bias", [(True, True), (True, False), (False, False)])
def test_gradients_through_autograd(gpu, dtype, weight, bias):
    from neuropress_amd import kernels

    x, w, b, dy = (t.to(gpu) for t in _inputs(37, 200, dtype))
    leaves = [t.requires_grad_() for t, need in ((x, True), (w, weight), (b, bias)) if need]
    y = kernels.layer_norm(x, w if weight else None, b if bias else None, EPS)
    assert y.grad_fn is not None
    got = torch.autograd.grad(y, leaves, dy)
    _, mean, rstd = kernels.layer_norm_stats(x.detach(), None, None, EPS)
    want = kernels.layer_norm_backward(dy, x.detach(), w.detach() if weight else None, mean, rstd)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    # only the weight asks for a gradient
    if weight:
        y = kernels.layer_norm(x.detach(), w, None, EPS)
        assert torch.equal(torch.autograd.grad(y, [w], dy)[0], want[1])
    with torch.no_grad():
        assert kernels.layer_norm(x, w if weight else None, b if bias else None, EPS).grad_fn is None


def test_gradients_against_differences(gpu):
    """Central differences of the kernel's own forward pass in f32: off by their own rounding, 2^-24 |y| / step, and by step^2 of the third derivative."""
    from neuropress_amd import kernels

    g = cases.gen(11)
    x, w, b, dy = (torch.randn(*s, generator=g).to(gpu) for s in ((3, 24), (24,), (24,), (3, 24)))
    _, mean, rstd = kernels.layer_norm_stats(x, w, b, EPS)
    grads = kernels.layer_norm_backward(dy, x, w, mean, rstd)
    step = 2.0**-7
    for k, (t, grad) in enumerate(zip((x, w, b), grads)):
        for i in range(t.numel()):
            args = [x, w, b]
            ends = []
            for sign in (1, -1):
                moved = t.clone()
                moved.view(-1)[i] += sign * step
                args[k] = moved
                ends.append((kernels.layer_norm(*args, EPS).double() * dy.double()).sum().item())
            # 72 values of up to 4, each off by 2^-22, over 2 steps: 0.0015; third derivative of order 10 at most: 10 step^2 / 6 = 1e-4
            assert abs((ends[0] - ends[1]) / (2 * step) - grad.view(-1)[i].item()) < 2e-3 * max(1.0, grad.abs().max().item())


def test_calls_that_torch_follows_otherwise(gpu):
    from neuropress_amd import kernels

    x, w, b = torch.randn(4, 32, device=gpu), torch.randn(32, device=gpu), torch.randn(32, device=gpu)
    f = lambda t: kernels.layer_norm(t, w, b, EPS)
    want = torch.func.jvp(lambda t: torch.nn.functional.layer_norm(t, (32,), w, b, EPS), (x,), (x,))
    got = torch.func.jvp(f, (x,), (x,))
    assert all(torch.allclose(a, c, atol=1e-5) for a, c in zip(got, want))
    assert torch.allclose(torch.func.vmap(f)(x), f(x), atol=1e-5)
    assert torch.func.grad(lambda t: f(t).sum())(x).shape == x.shape
    # a second derivative is refused, not wrong
    x = x.requires_grad_()
    (dx,) = torch.autograd.grad(kernels.layer_norm(x, w, b).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


def test_in_place_and_rows_behind_the_last(gpu):
    """Through the C entry: out may be x, dx may be dy, and nothing behind the rows is written."""
    from neuropress_amd import _lib, kernels

    for m, h in ((5, 4096), (3, 77)):
        x, w, b, dy = (t.to(gpu) for t in _inputs(m, h, torch.bfloat16))
        y, mean, rstd = kernels.layer_norm_stats(x, w, b, EPS)
        dx, dw, db = kernels.layer_norm_backward(dy, x, w, mean, rstd)
        room = torch.full((m + 1, h + 8), 7.0, dtype=torch.bfloat16, device=gpu)
        room[:m, :h] = x
        st = torch.cuda.current_stream().cuda_stream
        _lib.call("npamd_layer_norm", room.data_ptr(), h + 8, w.data_ptr(), b.data_ptr(), room.data_ptr(), h + 8, None, None, m, h, EPS, 1, st)
        assert torch.equal(room[:m, :h], y) and bool((room[m] == 7).all()) and bool((room[:, h:] == 7).all())
        room[:m, :h] = dy
        need = _lib.load().npamd_layer_norm_workspace_bytes(m, h)
        ws = torch.empty(need // 4, device=gpu)
        _lib.call("npamd_layer_norm_backward", room.data_ptr(), h + 8, x.data_ptr(), h, w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), room.data_ptr(), h + 8, dw.data_ptr(),
                  db.data_ptr(), m, h, 1, ws.data_ptr(), need, st)  # fmt: skip
        assert torch.equal(room[:m, :h], dx) and bool((room[m] == 7).all()) and bool((room[:, h:] == 7).all())


@pytest.mark.parametrize("over", ["dy", "x"])
@pytest.mark.parametrize("m,h", [(5, 4096), (40, 321), (70, 640), (300, 5), (130, 17000)])
def test_gradient_in_the_place_of_an_input(gpu, over, m, h):
    """Through the C entry, with the gradients of weight and bias, which are sums over what dx replaces."""
    from neuropress_amd import _lib, kernels

    x, w, _, dy = (None if t is None else t.to(gpu) for t in _inputs(m, h, torch.float16))
    _, mean, rstd = kernels.layer_norm_stats(x, None, None, EPS)
    want = kernels.layer_norm_backward(dy, x, w, mean, rstd)
    dw, db = torch.empty_like(w), torch.empty_like(w)
    need = _lib.load().npamd_layer_norm_workspace_bytes(m, h)
    ws = torch.empty(need // 4, device=gpu)
    place = dy if over == "dy" else x
    _lib.call("npamd_layer_norm_backward", dy.data_ptr(), h, x.data_ptr(), h, w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), place.data_ptr(), h, dw.data_ptr(),
              db.data_ptr(), m, h, 0, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)  # fmt: skip
    assert all(torch.equal(a, c) for a, c in zip((place, dw, db), want))


def test_module_and_lowering(gpu):
    from neuropress_amd import AutoKernelLowering, is_lowered, unlower_model
    from neuropress_amd.nn import NPLayerNorm

    torch.manual_seed(0)

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm = torch.nn.LayerNorm(96, eps=1e-6)
            self.again = self.norm
            self.inner = torch.nn.Sequential(torch.nn.Linear(96, 96), torch.nn.LayerNorm(96, bias=False), torch.nn.LayerNorm((4, 24)))

        def forward(self, x):
            return self.inner[2](self.inner[1](self.inner[0](self.again(self.norm(x)))).unflatten(-1, (4, 24))).flatten(-2)

    model = Block().to(gpu)
    torch.nn.init.normal_(model.norm.weight)
    x = torch.randn(2, 9, 96, device=gpu)
    keys, before = list(model.state_dict()), model(x)
    weights = torch.randn(before.shape, device=gpu)

    def gradients(loss):
        model.zero_grad()
        loss(model(x)).backward()
        return {n: p.grad.clone() for n, p in model.named_parameters()}

    losses = (lambda y: y.square().sum(), lambda y: (y * weights).sum())
    grads = [gradients(loss) for loss in losses]
    AutoKernelLowering(norm_backend="auto").apply(model)
    assert not is_lowered(model), "only norm_backend='all' reaches nn.LayerNorm"
    norm = model.norm
    AutoKernelLowering(norm_backend="all").apply(model)
    assert is_lowered(model) and isinstance(model.norm, NPLayerNorm) and model.again is model.norm and isinstance(model.inner[1], NPLayerNorm)
    assert type(model.inner[2]) is torch.nn.LayerNorm and list(model.state_dict()) == keys and model.norm.weight is norm.weight
    # values of a few units through three norms and a linear layer in f32
    assert torch.allclose(model(x), before, atol=1e-4)
    for loss, want in zip(losses, grads):
        got = gradients(loss)
        for n, g in got.items():
            # The squares' sum is 4 * 18 * 24 whatever the parameters (the last norm has unit weight): that loss's true gradients are zero, and what either side
            # returns is its rounding, 2^-24 of some 18 * 96 terms of up to 6 * 4 each that average out: 2^-24 * 24 * sqrt(1728) = 6e-5.
            assert torch.allclose(g, want[n], rtol=1e-3, atol=max(1e-3 * want[n].abs().max().item(), 6e-5)), n
    unlower_model(model)
    assert model.norm is norm and model.again is norm and not is_lowered(model)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [8, 64, 321, 777, 2052, 4099, 8200])
@pytest.mark.parametrize("m", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 32, 33, 65])
def test_backward_of_few_rows(gpu, dtype, m, h):
    """As many rows as a block takes at once or in a second turn, one more and one less: its sums meet in other ways, or are all there is."""
    from neuropress_amd import kernels

    x, w, _, dy = _inputs(m, h, dtype, seed=3)
    _, mean, rstd = kernels.layer_norm_stats(x.to(gpu), None, None, EPS)
    got = kernels.layer_norm_backward(dy.to(gpu), x.to(gpu), w.to(gpu), mean, rstd)
    for t, (ref, slack), what in zip(got, _reference_back(dy, x, w, mean.cpu(), rstd.cpu()), ("dx", "dw", "db")):
        _check(t, ref, slack, dtype, what)


@pytest.mark.parametrize("h", [2, 8])
def test_more_rows_than_a_launch_has_blocks(gpu, h):
    from neuropress_amd import kernels

    m = (1 << 24) + 5
    g = torch.Generator(device=gpu).manual_seed(h)
    x, dy = (torch.randn(m, h, generator=g, device=gpu).to(torch.float16) for _ in range(2))
    y, mean, rstd = kernels.layer_norm_stats(x, None, None, EPS)
    dx, _, _ = kernels.layer_norm_backward(dy, x, None, mean, rstd, needs=(True, False, False))
    for first in (0, (1 << 23) - 3, (1 << 24) - 3):
        rows = slice(first, first + 8)
        xs, dys = x[rows].cpu(), dy[rows].cpu()
        ref, _, _, slack = _reference(xs, None, None)
        _check(y[rows], ref, slack, torch.float16, "y")
        _check(dx[rows], *_reference_back(dys, xs, None, mean[rows].cpu(), rstd[rows].cpu())[0], torch.float16, "dx")
    assert torch.equal(y, kernels.layer_norm(x, None, None, EPS)) and bool(torch.isfinite(dx).all())


def test_what_autograd_hands_to_the_backward_pass(gpu):
    """Gradients that are expanded, transposed or missing, inputs without rows or at no single distance, an input changed in between, one backward pass after another."""
    from neuropress_amd import kernels

    x, w, b, dy = (t.to(gpu) for t in _inputs(24, 160, torch.float32))
    xs = torch.randn(4, 6, 400, device=gpu)[:, ::2, 30:190].requires_grad_()
    w.requires_grad_(), b.requires_grad_()
    f = lambda t: torch.nn.functional.layer_norm(t, (160,), w, b, EPS)
    for t in (xs, x.view(2, 12, 160).transpose(0, 1).detach().requires_grad_()):
        for loss in (lambda y: y.sum(), lambda y: (y.transpose(0, 1) * 0.5).contiguous().square().sum(), lambda y: y[:, :2].mean()):
            got, want = torch.autograd.grad(loss(kernels.layer_norm(t, w, b, EPS)), [t, w, b]), torch.autograd.grad(loss(f(t)), [t, w, b])
            # both are f32 sums of up to 72 x 160 terms of about one
            assert all(torch.allclose(a, c, rtol=1e-4, atol=1e-4) for a, c in zip(got, want))
    none = x[:0].detach().requires_grad_()
    got = torch.autograd.grad(kernels.layer_norm(none, w, b, EPS).sum(), [none, w, b])
    assert got[0].shape == none.shape and not got[1].any() and not got[2].any()
    y = kernels.layer_norm(xs, w, b, EPS)
    y.sum().backward(retain_graph=True)
    first = w.grad.clone()
    y.sum().backward()
    assert torch.equal(w.grad, 2 * first)
    moved = x.clone()
    y = kernels.layer_norm(moved, w, b, EPS)
    moved.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = kernels.layer_norm(x, w, b, EPS)
    with pytest.raises(RuntimeError, match="at most 2\\*\\*31"):
        kernels.layer_norm(x[:1].expand(1 << 31, 160), w, b, EPS)
    del y


@pytest.mark.parametrize("auto", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtype", DTYPES)
def test_autocast_norms_in_float32(gpu, dtype, auto):
    """Whether its type is the inputs' or not; with and without a recorded gradient.  Two f32 norms of the same values: off by n 2^-24 of a few units each."""
    from neuropress_amd import kernels

    x, w, b, dy = (t.to(gpu) for t in _inputs(5, 64, dtype))
    with torch.autocast("cuda", auto):
        want = torch.nn.functional.layer_norm(x, (64,), w, b, EPS)
        got = kernels.layer_norm(x, w, b, EPS)
        recorded = kernels.layer_norm(x.requires_grad_(), w, b, EPS)
    assert got.dtype == recorded.dtype == want.dtype == torch.float32 and recorded.grad_fn is not None
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5) and torch.allclose(recorded, want, rtol=1e-5, atol=1e-5)


def _lowered(width, dtype):
    """A module with one norm, and its lowered copy."""
    import copy

    from neuropress_amd import AutoKernelLowering
    from neuropress_amd.nn import NPLayerNorm

    torch.manual_seed(1)
    plain = torch.nn.Sequential(torch.nn.LayerNorm(width))
    for p in plain.parameters():
        torch.nn.init.normal_(p)
    plain = plain.to("cuda", dtype)
    lowered = copy.deepcopy(plain)
    AutoKernelLowering(norm_backend="all").apply(lowered)
    assert type(lowered[0]) is NPLayerNorm
    return plain, lowered


@pytest.mark.parametrize("auto", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dtype", DTYPES)
def test_module_under_autocast(gpu, dtype, auto):
    """Mixed-precision training: float32 parameters, x of any type.  Results, their types and gradients are the replaced module's; both sides norm in f32."""
    x = _inputs(7, 96, dtype)[0].to(gpu)
    results = []
    for model in _lowered(96, torch.float32):
        leaf = x.clone().requires_grad_()
        with torch.autocast("cuda", auto):
            y = model(leaf)
            with torch.no_grad():
                silent = model(x)
        y.float().square().sum().backward()
        results.append((y, silent, leaf.grad, *(p.grad for p in model.parameters())))
    for want, got in zip(*results, strict=True):
        assert got.dtype == want.dtype
        # gradients in x's type: the same f32 values to a few 2^-24, so another rounding at most
        eps = torch.finfo(want.dtype).eps
        assert torch.allclose(got.float(), want.float(), rtol=max(eps, 1e-5), atol=1e-4)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_module_refuses_mixed_types_as_the_one_it_replaced(gpu, dtype):
    x = torch.randn(7, 96, device=gpu).to(dtype)
    for model in _lowered(96, torch.float32):
        with pytest.raises(RuntimeError):
            model(x)


def test_float64_norms_stay_torchs(gpu):
    """Left alone by the lowering, and computed as before by a module that is moved to float64 afterwards."""
    from neuropress_amd import AutoKernelLowering

    x = torch.randn(7, 96, dtype=torch.float64, device=gpu)
    model = torch.nn.Sequential(torch.nn.LayerNorm(96)).to("cuda", torch.float64)
    want = model(x)
    AutoKernelLowering(norm_backend="all").apply(model)
    assert type(model[0]) is torch.nn.LayerNorm and torch.equal(model(x), want)
    plain, lowered = _lowered(96, torch.float32)
    plain.double(), lowered.double()
    leaves = [x.clone().requires_grad_() for _ in range(2)]
    ys = [net(leaf) for net, leaf in zip((plain, lowered), leaves)]
    for y in ys:
        y.square().sum().backward()
    assert torch.equal(*ys) and torch.equal(leaves[0].grad, leaves[1].grad)


@pytest.mark.parametrize("kind", ["forward_hook", "forward_pre_hook", "full_backward_hook", "full_backward_pre_hook", "state_dict_post_hook", "load_state_dict_post_hook", "forward"])
def test_norms_with_hooks_are_left_alone(gpu, kind):
    from neuropress_amd import AutoKernelLowering
    from neuropress_amd.nn import NPLayerNorm

    model = torch.nn.Sequential(torch.nn.LayerNorm(64), torch.nn.LayerNorm(64)).to(gpu)
    seen = []
    if kind == "forward":
        forward = model[0].forward
        model[0].forward = lambda x: seen.append(kind) or forward(x)
    else:
        getattr(model[0], "register_" + kind)(lambda *args: seen.append(kind))
    AutoKernelLowering(norm_backend="all").apply(model)
    assert type(model[0]) is torch.nn.LayerNorm and type(model[1]) is NPLayerNorm
    model(torch.randn(3, 64, device=gpu, requires_grad=True)).sum().backward()
    model.load_state_dict(model.state_dict())
    assert seen


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,h", [(5, 64), (40, 1000), (3, 8192), (300, 512), (5, 12288), (2, 5), (3, 40000)])
def test_gradients_of_constant_rows(gpu, dtype, m, h):
    """x - mean is exactly zero there, whatever kernel takes the row: the weight's gradient is zero, and that of x is what the mean of dy * weight leaves."""
    from neuropress_amd import kernels

    x = (torch.arange(m) * 7 + 99.0)[:, None].expand(m, h).to(dtype)
    _, w, _, dy = _inputs(m, h, dtype)
    mean, rstd = x[:, 0].float(), torch.full((m,), EPS).rsqrt()
    dx, dw, db = kernels.layer_norm_backward(dy.to(gpu), x.to(gpu), w.to(gpu), mean.to(gpu), rstd.to(gpu))
    assert not dw.any()
    refs = _reference_back(dy, x, w, mean, rstd)
    for got, (ref, slack), what in zip((dx, db), (refs[0], refs[2]), ("dx", "db")):
        _check(got, ref, slack, dtype, what)


@pytest.mark.parametrize("h", [2, 3, 8])
def test_sums_over_very_many_rows(gpu, h):
    """Equal addends, whose roundings in a long f32 chain all go the same way.  Short rows: strips in f64, rounded once, then up to 64 + 16 of them in f32.  Others: a chain
    of M / 4096 rows for each of 256 blocks' 16 groups."""
    from neuropress_amd import kernels

    m = (1 << 24) + 5
    x = torch.zeros(m, h, device=gpu)
    x[:, ::2] = 1.0
    dy = torch.full((m, h), 1.001, device=gpu)
    mean, rstd = torch.full((m,), 0.5, device=gpu), torch.full((m,), 2.0, device=gpu)  # (x - mean) * rstd is 1 and -1
    _, dw, db = kernels.layer_norm_backward(dy, x, None, mean, rstd, needs=(False, True, True))
    want = m * dy[0, 0].double()
    off = EPS32 * (100 + (m / 4096 if h >= 4 else 0)) * want
    assert bool(((db.double() - want).abs() <= off).all()) and bool(((dw[::2].double() - want).abs() <= off).all()) and bool(((dw[1::2].double() + want).abs() <= off).all())
