"""The dense product with an epilogue against the formula in 64 bits.

Tolerances: half a step of the output type, plus what f32 adds: the product's sum of K terms is off by at most n 2^-24 sum |x w| with n = K / 16 + 40 (the longest chain of
additions of any kernel), times the activations' largest slope (1.13), and an activation is computed to 2^-20 of its argument."""

import pytest
import torch

from tests import cases

pytestmark = pytest.mark.gpu
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]
DTYPES = [torch.float16, torch.bfloat16]


def _act(name, v):
    f = torch.nn.functional
    return v if name is None else f.gelu(v, approximate="tanh") if name == "gelu_tanh" else getattr(f, name)(v)


def _inputs(m, n, k, dtype, seed=0):
    g = cases.gen(seed + m + 7 * n + 13 * k)
    return [t.to(dtype) for t in (torch.randn(m, k, generator=g), torch.randn(n, k, generator=g) * k**-0.5 * 2, torch.randn(n, generator=g), torch.randn(m, n, generator=g) * 2)]


def _check(y, x, w, b, act, r, what=""):
    dtype = x.dtype
    on = lambda t: None if t is None else t.to("cuda").double()
    xd, wd = on(x), on(w)
    v = xd @ wd.T
    spread = xd.abs() @ wd.abs().T
    if b is not None:
        v, spread = v + on(b), spread + on(b).abs()
    ref = _act(act, v)
    if r is not None:
        ref = ref + on(r)
    assert y.dtype == dtype and y.shape == ref.shape
    eps = torch.finfo(dtype).eps
    tol = ref.abs() * (eps / 2) * 1.0001 + torch.finfo(dtype).smallest_normal * eps / 2 + 1.13 * 2.0**-24 * (x.shape[-1] / 16 + 40) * spread + 2.0**-20 * v.abs()
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), f"{what}: {(err / tol).max().item():.2f} of the tolerance"


def _run(x, w, b, act, r):
    from neuropress_amd import kernels

    on = lambda t: None if t is None else t.to("cuda")
    return kernels.dense_linear_act(on(x), on(w), on(b), act, on(r))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(1, 640, 2048), (3, 257, 512), (17, 200, 136), (40, 129, 264), (300, 520, 1024)])
def test_epilogues(gpu, dtype, act, m, n, k):
    x, w, b, r = _inputs(m, n, k, dtype)
    for bias in (None, b, b.float() + 1e-3):
        for res in (None, r):
            _check(_run(x, w, bias, act, res), x, w, bias, act, res, f"bias {bias is not None and bias.dtype} residual {res is not None}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 2, 4, 5, 8, 9, 16, 17, 31, 32, 33, 64, 65, 129, 257])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 8), (63, 1003), (100, 64), (384, 520), (1030, 2312)])
def test_sizes(gpu, dtype, m, n, k):
    x, w, b, r = _inputs(m, n, k, dtype)
    _check(_run(x, w, b, "silu", r), x, w, b, "silu", r)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 14336), (16, 512, 8192), (5, 14336, 640), (33, 256, 14336), (96, 384, 8192), (2048, 1024, 512), (700, 2000, 4096)])
def test_large(gpu, m, n, k):
    x, w, b, r = _inputs(m, n, k, torch.bfloat16)
    _check(_run(x, w, b, "gelu", r), x, w, b, "gelu", r)
    assert torch.equal(_run(x, w, b, "gelu", r), _run(x, w, b, "gelu", r)), "the same inputs, other bits"


@pytest.mark.parametrize("tile", sorted(cases.DENSE_TILES))
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("k", [640, 584])
def test_every_tile(gpu, monkeypatch, tile, splits, k):
    from neuropress_amd import _lib

    monkeypatch.setenv("NPAMD_DENSE_TILE", str(tile))
    monkeypatch.setenv("NPAMD_DENSE_SPLITS", str(splits))
    _lib.load().npamd_diag_reload_tuning()
    for n in (330, 331):
        x, w, b, r = _inputs(270, n, k, torch.float16)
        _check(_run(x, w, b, "gelu_tanh", r), x, w, b, "gelu_tanh", r, f"n {n}")
        _check(_run(x, w, None, "relu", None), x, w, None, "relu", None, f"n {n}")


def _strided(t, ld, at):
    room = torch.full((t.shape[0] * ld + at,), float("nan"), dtype=t.dtype, device="cuda")
    view = room[at:].as_strided(t.shape, (ld, 1))
    view.copy_(t)
    return view


@pytest.mark.parametrize("m", [1, 7, 20, 50])
@pytest.mark.parametrize("at,pad", [(0, 0), (1, 3), (8, 8), (3, 16)])
def test_row_distances_and_odd_addresses(gpu, m, at, pad):
    from neuropress_amd import kernels

    n, k = 136, 264
    x, w, b, r = _inputs(m, n, k, torch.float16)
    y = kernels.dense_linear_act(_strided(x, k + pad, at), _strided(w, k + pad, at), _strided(b[None], n, at)[0], "silu", _strided(r, n + pad, at))
    _check(y, x, w, b, "silu", r)
    # rows that overlap or stand still
    one = x[:1].to(gpu).expand(m, k)
    _check(kernels.dense_linear_act(one, w.to(gpu), None, None, r[:1].to(gpu).expand(m, n)), x[:1].expand(m, k), w, None, None, r[:1].expand(m, n))
    wt = w.T.contiguous().to(gpu).T  # a weight kept [K, N]
    _check(kernels.dense_linear_act(x.to(gpu), wt), x, w, None, None, None)


def test_shapes_around(gpu):
    from neuropress_amd import kernels

    x, w, b, r = (t.to(gpu) for t in _inputs(24, 40, 64, torch.bfloat16))
    y = kernels.dense_linear_act(x, w, b, "relu", r)
    assert torch.equal(kernels.dense_linear_act(x.view(2, 3, 4, 64), w, b, "relu", r.view(2, 3, 4, 40)), y.view(2, 3, 4, 40))
    assert kernels.dense_linear_act(x[5], w, b, "relu", r[5]).shape == (40,)
    assert kernels.dense_linear_act(x[:0], w, b, "relu", r[:0]).shape == (0, 40)
    assert kernels.dense_linear_act(x.view(2, 12, 64), w[:0], b[:0], "relu", r.view(2, 12, 40)[..., :0]).shape == (2, 12, 0)


@pytest.mark.parametrize("m", [1, 20, 200])
def test_values_that_are_not_finite(gpu, m):
    """They reach their own row and column only, and go through the activations as torch's do."""
    x, w, b, r = _inputs(m, 256, 128, torch.bfloat16)
    x[0, 3], w[7, 5], b[9], r[0, 11], b[12], b[13] = float("nan"), float("inf"), float("-inf"), float("inf"), float("nan"), float("inf")
    for act in ACTS:
        y = _run(x, w, b, act, r).cpu()
        v = x.double() @ w.double().T + b.double()
        ref = _act(act, v) + r.double()
        assert torch.equal(y.isnan(), ref.isnan()) and torch.equal(y == float("inf"), ref == float("inf")) and torch.equal(y == float("-inf"), ref == float("-inf")), act


def test_activations_over_their_range(gpu):
    """x @ w is one exact product here, so the activation alone is seen: to 2^-20 of its argument, and to half a step."""
    from neuropress_amd import kernels

    for dtype, far in ((torch.float16, 60000.0), (torch.bfloat16, 3e38)):
        v = torch.cat([torch.linspace(-12, 12, 4001), torch.linspace(-100, 100, 501), torch.tensor([0.0, -0.0, far, -far])]).to(dtype)
        x, w = v[:, None], torch.ones(1, 1, dtype=dtype)
        for act in ACTS[1:]:
            y = kernels.dense_linear_act(x.to(gpu), w.to(gpu), None, act).cpu()[:, 0].double()
            ref = _act(act, v.double())
            tol = ref.abs() * torch.finfo(dtype).eps / 2 * 1.0001 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 + torch.where(v.abs() < 100, 2.0**-20 * v.double().abs(), 0.0)
            assert bool(((y - ref).abs() <= tol).all()), (act, v[((y - ref).abs() > tol)][:5])


def test_calls_that_torch_follows(gpu):
    from neuropress_amd import kernels

    x, w, b, r = (t.to(gpu) for t in _inputs(4, 24, 32, torch.float16))
    f = torch.nn.functional
    want = f.gelu(f.linear(x, w, b)) + r
    for t in (x, w, b, r):
        t.requires_grad_()
    y = kernels.dense_linear_act(x, w, b, "gelu", r)
    assert torch.equal(y, want)
    assert all(g is not None for g in torch.autograd.grad(y.sum(), [x, w, b, r]))


def test_the_residual_in_its_own_place(gpu):
    """Through the C entry: y may be the residual, and nothing outside the result is written."""
    from neuropress_amd import _lib, kernels

    for m, n, k in ((1, 96, 256), (9, 96, 256), (30, 100, 256), (130, 100, 256), (60, 64, 8192)):
        x, w, b, r = (t.to(gpu) for t in _inputs(m, n, k, torch.float16))
        want = kernels.dense_linear_act(x, w, b, "relu", r)
        room = torch.full((m + 1, n + 8), 5.0, dtype=torch.float16, device=gpu)
        room[:m, :n] = r
        need = _lib.load().npamd_dense_gemm_act_workspace_bytes(m, n, k)
        ws = torch.empty(max(need // 4, 4), device=gpu)
        _lib.call("npamd_dense_gemm_act", x.data_ptr(), k, w.data_ptr(), k, b.data_ptr(), 0, 1, room.data_ptr(), n + 8, room.data_ptr(), n + 8, m, n, k, 0, ws.data_ptr(), need,
                  torch.cuda.current_stream().cuda_stream)  # fmt: skip
        assert torch.equal(room[:m, :n], want) and bool((room[m] == 5).all()) and bool((room[:, n:] == 5).all())
        # without a workspace K is not split: another order of the same sum
        room[:m, :n] = r
        _lib.call("npamd_dense_gemm_act", x.data_ptr(), k, w.data_ptr(), k, b.data_ptr(), 0, 1, room.data_ptr(), n + 8, room.data_ptr(), n + 8, m, n, k, 0, None, 0,
                  torch.cuda.current_stream().cuda_stream)  # fmt: skip
        _check(room[:m, :n], x, w, b, "relu", r)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [2, 3, 15, 16, 17, 31, 32, 33, 48, 49, 64, 65])
@pytest.mark.parametrize("n,k", [(1, 8), (16, 120), (17, 128), (100, 1032), (40, 2560), (40, 2568), (4096, 264), (4100, 264), (8191, 136), (8192, 136), (8209, 1160), (2048, 1032), (2049, 1032), (2048, 1021)])
def test_where_one_kernel_takes_over_from_another(gpu, dtype, m, n, k):
    """Tokens and rows on both sides of where the kernel changes; columns that end inside a step, or before every wave has one."""
    x, w, b, r = _inputs(m, n, k, dtype)
    _check(_run(x, w, b, "silu", r), x, w, b, "silu", r)


@pytest.mark.parametrize("n", [4096, 4112])  # 2^24 weights of 4096 columns, and some more
@pytest.mark.parametrize("m", [16, 17, 32, 50])
def test_weights_on_both_sides_of_the_line(gpu, m, n):
    x, w, b, r = _inputs(m, n, 4096, torch.bfloat16)
    _check(_run(x, w, b, "gelu", r), x, w, b, "gelu", r)


def test_nothing_of_other_rows_reaches_a_result(gpu):
    """Infinities and NaN in the rows that a tile reads besides its own, and behind the columns."""
    x, w, b, r = _inputs(32, 48, 200, torch.bfloat16)
    for m, n in [(1, 48), (3, 47), (5, 17), (17, 33), (31, 1)]:
        xs, ws = torch.full((32, 208), float("nan"), dtype=x.dtype), torch.full((48, 208), float("inf"), dtype=x.dtype)
        xs[:m, :200], ws[:n, :200] = x[:m], w[:n]
        xs, ws = xs.to("cuda")[:m, :200], ws.to("cuda")[:n, :200]
        _check(_run(xs, ws, b[:n], "relu", r[:m, :n]), xs, ws, b[:n], "relu", r[:m, :n])


@pytest.mark.parametrize("m", [1, 2, 3, 17, 32, 40])
@pytest.mark.parametrize("k", [9, 11, 15, 523])
@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_values_in_the_columns_that_two_pieces_share(gpu, dtype, m, k):
    """A row's last piece of eight starts inside the one before; what it has of that counts once, also where it is not finite."""
    x, w, b, r = _inputs(m, 21, k, dtype)
    x = x.abs() + 0.5
    w[3, k // 8 * 8 - 8 + k % 8], w[4, k - 8], w[5, k // 8 * 8 - 1], w[6, k - 1] = float("-inf"), float("inf"), float("-inf"), float("inf")
    for act in ACTS:
        y = _run(x, w, b, act, r).cpu()
        ref = _act(act, x.double() @ w.double().T + b.double()) + r.double()
        assert torch.equal(y.isnan(), ref.isnan()) and torch.equal(y == float("inf"), ref == float("inf")) and torch.equal(y == float("-inf"), ref == float("-inf")), act
