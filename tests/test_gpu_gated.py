"""The gated product and its backward pass against the formulas in 64 bits.

Tolerances: half a step of the output type, plus what f32 adds.  A sum of K products is off by at most n 2^-24 of the sum of their absolute values, n = K / 16 + 40 (the longest chain of additions
of any kernel); activations' slopes are at most 1.13, and an activation is computed to 2^-20 of its argument.  Backward: an activation's slope is computed to 2^-19 (1 + |g|); what goes into
the products is rounded once to their type (half a step of each term); a bias's sum over M rows is a chain of at most M / 64 + 60 additions."""

import pytest
import torch

from tests import cases

pytestmark = pytest.mark.gpu
ACTS = [None, "relu", "gelu", "gelu_tanh", "silu"]
DTYPES = [torch.float16, torch.bfloat16]
U = 2.0**-24


def _act(name, v):
    f = torch.nn.functional
    return v if name is None else f.gelu(v, approximate="tanh") if name == "gelu_tanh" else getattr(f, name)(v)


def _half(ref, dtype):
    return ref.abs() * (torch.finfo(dtype).eps / 2) * 1.0001 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _within(got, ref, tol, dtype, what):
    assert got.dtype == dtype and got.shape == ref.shape, what
    bad = (got.double() - ref).abs() / (tol + _half(ref, dtype))
    assert bool((bad <= 1).all()), f"{what}: {bad.max().item():.2f} of the tolerance"


def _inputs(m, n, k, dtype, seed=0):
    g = cases.gen(seed + m + 7 * n + 13 * k)
    make = lambda *shape, std=1.0: (torch.randn(*shape, generator=g) * std).to(dtype).cuda()
    return make(m, k), make(2 * n, k, std=2 * k**-0.5), make(2 * n), make(m, n)


def _check_forward(x, w, b, act, what=""):
    from neuropress_amd import kernels

    h, pre = kernels.gated_linear_pre(x, w, b, act)
    assert torch.equal(h, kernels.gated_linear(x, w, b, act))
    xd, wd = x.double(), w.double()
    v, spread = xd @ wd.T, xd.abs() @ wd.abs().T
    if b is not None:
        v, spread = v + b.double(), spread + b.double().abs()
    e = (x.shape[-1] / 16 + 40) * U * spread
    _within(pre, v, e, x.dtype, f"pre {what}")
    (g, u), (eg, eu) = v.chunk(2, -1), e.chunk(2, -1)
    a = _act(act, g)
    ea = 1.13 * eg + 2.0**-20 * g.abs()
    _within(h, a * u, ea * u.abs() + (a.abs() + ea) * eu + 2 * U * (a * u).abs(), x.dtype, f"h {what}")
    return h, pre


def _pointwise(dh, pre, act):
    """[dg du] in 64 bits and its error in f32."""
    p = pre.double().requires_grad_()
    g, u = p.chunk(2, -1)
    d = torch.autograd.grad(_act(act, g) * u, p, dh.double())[0]
    g, u = g.detach(), u.detach()
    e = torch.cat(((dh.double() * u).abs() * 2.0**-19 * (1 + g.abs()), dh.double().abs() * 2.0**-20 * g.abs()), -1) + 3 * U * d.abs()
    return d, e


def _check_backward(dh, x, w, pre, act, bias_dtype=None, what=""):
    from neuropress_amd import kernels

    dx, dw, db = kernels.gated_linear_backward(dh, x, w, pre, act, bias_dtype=bias_dtype)
    dtype = x.dtype
    d, e = _pointwise(dh, pre, act)
    er = e + _half(d, dtype)
    m, n2 = d.shape
    xd, wd = x.double(), w.double()
    _within(dx, d @ wd, er @ wd.abs() + (n2 / 16 + 40) * U * ((d.abs() + er) @ wd.abs()), dtype, f"dx {what}")
    _within(dw, d.T @ xd, er.T @ xd.abs() + (m / 16 + 40) * U * ((d.abs() + er).T @ xd.abs()), dtype, f"dgate_up {what}")
    _within(db, d.sum(0), e.sum(0) + (m / 64 + 60) * U * d.abs().sum(0), bias_dtype or dtype, f"dbias {what}")
    for a, b in zip((dx, dw, db), kernels.gated_linear_backward(dh, x, w, pre, act, bias_dtype=bias_dtype)):
        assert torch.equal(a, b), "the same inputs, other bits"
    return dx, dw, db


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(1, 320, 2048), (2, 77, 512), (3, 129, 512), (17, 100, 136), (40, 65, 264), (300, 260, 1024)])
def test_forms(gpu, dtype, act, m, n, k):
    x, w, b, dh = _inputs(m, n, k, dtype)
    for bias in (None, b, b.float() + 1e-3):
        _, pre = _check_forward(x, w, bias, act, f"bias {bias is not None and bias.dtype}")
    _check_backward(dh, x, w, pre, act)
    _check_backward(dh, x, w, pre, act, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 2, 4, 5, 16, 17, 31, 32, 33, 48, 64, 65, 129, 257])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 5), (8, 8), (31, 1003), (50, 64), (192, 520), (515, 2312)])
def test_sizes(gpu, dtype, m, n, k):
    x, w, b, dh = _inputs(m, n, k, dtype)
    _, pre = _check_forward(x, w, b, "silu")
    _check_backward(dh, x, w, pre, "silu")


@pytest.mark.parametrize("m,n,k", [(1, 14336, 640), (16, 512, 8192), (5, 7168, 640), (33, 256, 14336), (64, 2048, 1024), (2048, 1024, 512), (700, 2000, 4096), (4096, 96, 96)])
def test_large(gpu, m, n, k):
    x, w, b, dh = _inputs(m, n, k, torch.bfloat16)
    _, pre = _check_forward(x, w, b, "gelu")
    _check_backward(dh, x, w, pre, "gelu")


@pytest.fixture
def tuned(monkeypatch):
    from neuropress_amd import _lib

    def force(tile, splits):
        monkeypatch.setenv("NPAMD_DENSE_TILE", str(tile))
        monkeypatch.setenv("NPAMD_DENSE_SPLITS", str(splits))
        _lib.load().npamd_diag_reload_tuning()

    yield force
    for name in ("NPAMD_DENSE_TILE", "NPAMD_DENSE_SPLITS"):
        monkeypatch.delenv(name, raising=False)
    _lib.load().npamd_diag_reload_tuning()


@pytest.mark.parametrize("tile", [2, 3, 4, 6, 7, 8, 9, 10, 12])  # the gated form's; turned operands: 2, 3, 4, 6, 12, others are planned
@pytest.mark.parametrize("dtype", DTYPES)
def test_every_tile(gpu, tuned, tile, dtype):
    bm, bn = cases.DENSE_TILES[tile]
    tuned(tile, 1)
    for m, n, k in ((65, bn // 2, 64), (bm - 1 + 64, bn // 2 - 1, 128), (bm + 65, bn // 2 + 1, 200), (2 * bm + 15, bn + 4, 320), (80, bn // 2 + 9, 584), (70, 36, 8 * bn + 8)):
        x, w, b, dh = _inputs(m, n, k, dtype)
        _, pre = _check_forward(x, w, b, "silu", (m, n, k))
        _check_backward(dh, x, w, pre, "silu", what=(m, n, k))
    for m in (1, 7, 9, 63, 64, 65, 130, 200, 321, 455):  # contracted rows that end anywhere in the first steps
        x, w, b, dh = _inputs(m, bm // 2 + 5, bn + 24, dtype)
        pre = torch.cat((dh, dh.flip(0)), -1)
        _check_backward(dh, x, w, pre, "gelu", what=m)


@pytest.mark.parametrize("tile", [2, 3, 4, 6, 7, 8, 9, 10, 12])
def test_parts_of_k(gpu, tuned, tile):
    tuned(tile, 3)
    for m, n, k in ((70, 66, 192), (70, 67, 704), (cases.DENSE_TILES[tile][0] + 65, 20, 1160), (100, 300, 584)):
        x, w, b, dh = _inputs(m, n, k, torch.bfloat16)
        for bias in (None, b):
            _, pre = _check_forward(x, w, bias, "silu", (m, n, k))
        _check_backward(dh, x, w, pre, "silu", what=(m, n, k))


@pytest.mark.parametrize("m", [1, 3, 20, 50, 200])
def test_rows_at_any_distance_and_address(gpu, m):
    from neuropress_amd import kernels

    x, w, b, dh = _inputs(m, 100, 264, torch.bfloat16)

    def spread(v, at, room):
        wide = torch.full((*v.shape[:-1], v.shape[-1] + room), float("inf"), device="cuda", dtype=v.dtype)
        wide[..., at : at + v.shape[-1]] = v
        return wide[..., at : at + v.shape[-1]]

    h, pre = kernels.gated_linear_pre(x, w, b)
    ref = kernels.gated_linear_backward(dh, x, w, pre)
    for at, room in ((0, 8), (1, 13), (8, 24), (3, 5)):
        xs, ws = spread(x, at, room), spread(w, at, room)
        got = kernels.gated_linear_pre(xs, ws, b)
        if m > 32 or (at, room) in ((0, 8), (8, 24)):  # few tokens at other addresses go another way, in another order of sums
            assert torch.equal(got[0], h) and torch.equal(got[1], pre)
        _check_forward(xs, ws, b, "silu")
        out = kernels.gated_linear_backward(spread(dh, at, room), xs, ws, spread(pre, at, room))
        assert all(torch.equal(i, j) for i, j in zip(out, ref))
    lead = kernels.gated_linear(x.view(1, m, 264).transpose(0, 1), w.t().contiguous().t(), b)
    assert lead.shape == (m, 1, 100)
    _within(lead[:, 0], h.double(), _half(h.double(), torch.bfloat16) + 1e-4, torch.bfloat16, "other strides")


def test_odd_rows_next_to_infinities(gpu):
    """What lies between rows, and rows and columns that only fill a tile, count for nothing."""
    from neuropress_amd import kernels

    for m, n, k in ((45, 33, 100), (70, 19, 203), (3, 9, 77)):
        x, w, b, dh = _inputs(m, n, k, torch.float16)
        x[0, 0] = float("inf")
        w[n, 0] = 0.0
        h, pre = kernels.gated_linear_pre(x, w, b)
        assert bool(h[1:].isfinite().all()) and bool(pre[1:].isfinite().all()) and bool(pre[0, n].isnan())
        pre[:] = 0.5
        dh[m - 1, n - 1] = float("nan")
        dx, dw, db = kernels.gated_linear_backward(dh, x, w, pre)
        assert bool(dx[:-1].isfinite().all()) and bool(dx[-1].isnan().all())
        bad = torch.zeros(2 * n, dtype=torch.bool, device="cuda")
        bad[[n - 1, 2 * n - 1]] = True
        assert torch.equal(db.isnan(), bad) and torch.equal(dw[:, 1:].isnan().any(1), bad) and not bool(dw[~bad, 0].isfinite().any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bias", [None, "same", "float32"])
def test_recorded(gpu, dtype, bias):
    from neuropress_amd import kernels

    x, w, b, dh = _inputs(42, 67, 136, dtype)
    b = None if bias is None else b.float() if bias == "float32" else b
    leaves = [None if t is None else t.clone().requires_grad_() for t in (x.view(2, 21, 136), w, b)]
    h = kernels.gated_linear(*leaves, "gelu")
    ref, pre = kernels.gated_linear_pre(x, w, b, "gelu")
    assert torch.equal(h.view(42, 67), ref)
    live = [t for t in leaves if t is not None]
    got = torch.autograd.grad(h, live, dh.view(2, 21, 67), retain_graph=True)
    want = kernels.gated_linear_backward(dh, x, w, pre, "gelu", bias_dtype=None if b is None else b.dtype)
    for a, e in zip(got, want):
        assert torch.equal(a.reshape(e.shape), e)
    for i, leaf in enumerate(live):
        only = kernels.gated_linear(*[t if t is leaf else None if t is None else t.detach() for t in leaves], "gelu")
        assert torch.equal(torch.autograd.grad(only, leaf, dh.view(2, 21, 67))[0], got[i])
    twice = torch.autograd.grad(h, live[0], dh.view(2, 21, 67), create_graph=True)[0]
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        twice.sum().backward()


@pytest.mark.parametrize("act", ACTS)
def test_gradients_against_differences(gpu, act):
    """Along random directions, by the central difference of the formula in 64 bits around the sums as they were rounded."""
    from neuropress_amd import kernels

    x, w, b, dh = _inputs(37, 41, 72, torch.float16)
    pre = kernels.gated_linear_pre(x, w, b, act)[1]
    pre[pre.abs() < 1e-2] = 0.5  # off the corner of relu
    dx, dw, db = _check_backward(dh, x, w, pre, act, torch.float32)
    d, e = _pointwise(dh, pre, act)
    er = e + _half(d, torch.float16)
    g = cases.gen(3)
    move = lambda t: torch.randn(t.shape, generator=g).double().cuda()
    vx, vw, vb = move(x), move(w), move(b)

    def loss(p):
        gate, up = p.chunk(2, -1)
        return (dh.double() * _act(act, gate) * up).sum()

    step = 1e-5
    for grad, v, along in ((dx, vx, vx @ w.double().T), (dw, vw, x.double() @ vw.T), (db, vb, vb[None])):
        diff = (loss(pre.double() + step * along) - loss(pre.double() - step * along)) / (2 * step)
        # the gradient's roundings (those of its terms, its own), all in the worst direction, and the difference's own step^2 and cancellation
        room = (er * along.abs()).sum() + (_half(grad.double(), grad.dtype) * v.abs()).sum() + 1e-4 * (d.abs() * along.abs()).sum()
        assert abs((grad.double() * v).sum() - diff) <= room


def test_followed_otherwise(gpu):
    from neuropress_amd import kernels

    x, w, b, _ = _inputs(6, 32, 64, torch.float16)
    y = kernels.gated_linear(x, w, b)
    out, tangent = torch.func.jvp(lambda t: kernels.gated_linear(t, w, b), (x,), (x,))
    assert torch.allclose(out, y, rtol=1e-2, atol=1e-2) and bool(tangent.isfinite().all())
    assert torch.allclose(torch.func.vmap(lambda t: kernels.gated_linear(t, w, b))(x), y, rtol=1e-2, atol=1e-2)
    with torch.autocast("cuda", torch.bfloat16):
        assert kernels.gated_linear(x, w, b).dtype == torch.bfloat16  # as torch's own products


def test_nothing_to_do(gpu):
    from neuropress_amd import kernels

    x, w, b, dh = _inputs(4, 16, 64, torch.float16)
    h, pre = kernels.gated_linear_pre(x[:0], w, b)
    assert h.shape == (0, 16) and pre.shape == (0, 32)
    dx, dw, db = kernels.gated_linear_backward(dh[:0], x[:0], w, pre)
    assert dx.shape == (0, 64) and not bool(dw.any()) and not bool(db.any()) and dw.shape == w.shape and db.shape == (32,)
    assert kernels.gated_linear(x, w[:0]).shape == (4, 0)
    leaves = [x[:0].clone().requires_grad_(), w.clone().requires_grad_()]
    kernels.gated_linear(*leaves).sum().backward()
    assert not bool(leaves[1].grad.any())
    h, pre = kernels.gated_linear_pre(x, w, b)
    assert all(t is None for t in kernels.gated_linear_backward(dh, x, w, pre, needs=(False, False, False)))
    whole = kernels.gated_linear_backward(dh, x, w, pre)
    for i in range(3):
        part = kernels.gated_linear_backward(dh, x, w, pre, needs=[i == j for j in range(3)])
        assert torch.equal(part[i], whole[i]) and sum(t is None for t in part) == 2


def test_refusals(gpu):
    from neuropress_amd import kernels

    x, w, b, dh = _inputs(4, 16, 64, torch.float16)
    for args, match in [((x.float(), w.float()), "float16 or bfloat16"), ((x, w.bfloat16()), "float16 or bfloat16"), ((x, w[:31]), "2 N"), ((x, w[:, :32]), "K"), ((x, w, b[:16]), "bias"),
                        ((x, w, b.bfloat16()), "bias"), ((x, w, b, "tanh"), "activation"), ((x, w.cpu()), "GPU"), ((x[:, :0], w[:, :0]), "at least 1")]:  # fmt: skip
        for call in (kernels.gated_linear, kernels.gated_linear_pre):
            with pytest.raises(RuntimeError, match=match):
                call(*args)
    pre = kernels.gated_linear_pre(x, w, b)[1]
    for args, match in [((dh[:, :8], x, w, pre), "dh and pre"), ((dh, x, w, pre[:2]), "dh and pre"), ((dh.float(), x, w, pre), "dh and pre"), ((dh, x, w, pre, "tanh"), "activation"),
                        ((dh, x.cpu(), w, pre), "GPU"), ((dh.cpu(), x, w, pre), "GPU"), ((dh, x, w, pre, "silu", (True,) * 3, torch.bfloat16), "bias_dtype")]:  # fmt: skip
        with pytest.raises(RuntimeError, match=match):
            kernels.gated_linear_backward(*args)


@pytest.mark.parametrize("m", [2, 12, 90])
def test_broadcast_gradients_and_inputs(gpu, m):
    """The gradient of a sum, one value for all, and inputs whose rows are one row or lie the other way round."""
    from neuropress_amd import kernels

    x, w, b, _ = _inputs(m, 40, 72, torch.bfloat16)
    one = torch.ones(m, 40, dtype=x.dtype, device="cuda")
    for xs, ws in ((x, w), (x[:1].expand(m, -1), w[:1].expand(80, -1)), (x.T.contiguous().T, w.T.contiguous().T)):
        h, pre = _check_forward(xs.contiguous(), ws.contiguous(), b, "gelu_tanh")
        leaves = [t.detach().requires_grad_() for t in (xs, ws, b)]
        out = kernels.gated_linear(*leaves, "gelu_tanh")
        assert torch.equal(out, h)
        got = torch.autograd.grad(out.sum(), leaves)
        want = kernels.gated_linear_backward(one, xs.contiguous(), ws.contiguous(), pre, "gelu_tanh")
        assert all(torch.equal(a, e) for a, e in zip(got, want))


def test_gradients_of_other_rows_are_refused(gpu):
    """As many rows in another shape: which belongs to which is not said."""
    from neuropress_amd import kernels

    x, w, b, dh = _inputs(6, 16, 64, torch.float16)
    x = x.view(2, 3, 64)
    pre = kernels.gated_linear_pre(x, w, b)[1]
    assert kernels.gated_linear_backward(dh.view(2, 3, 16), x, w, pre)[0].shape == x.shape
    for wrong in ((dh.view(3, 2, 16), pre), (dh, pre), (dh.view(2, 3, 16), pre.view(6, 32)), (dh.view(2, 3, 16), pre.view(3, 2, 32))):
        with pytest.raises(RuntimeError, match="dh and pre"):
            kernels.gated_linear_backward(wrong[0], x, w, wrong[1])


@pytest.fixture
def paired(tuned, monkeypatch):
    """Both products of the backward pass in one launch (1) or one after the other (-1)."""
    from neuropress_amd import _lib

    def force(pair, tile, splits):
        monkeypatch.setenv("NPAMD_DENSE_PAIR", str(pair))
        tuned(tile, splits)

    yield force
    monkeypatch.delenv("NPAMD_DENSE_PAIR", raising=False)
    _lib.load().npamd_diag_reload_tuning()


@pytest.mark.parametrize("tile", [2, 3, 4, 6, 12])
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("dtype", DTYPES)
def test_both_products_in_one_launch(gpu, paired, tile, splits, dtype):
    from neuropress_amd import kernels

    bm, bn = cases.DENSE_TILES[tile]
    shapes = [(bm + 65, bn // 2 + 1, 200), (70, 36, 8 * bn + 8), (1, 130, 9), (9, bm // 2 + 5, bn + 24), (455, 20, 40), (2 * bm + 15, bn + 4, 320), (1300, 40, 24), (6, 900, 330)]
    for m, n, k in shapes:
        x, w, b, dh = _inputs(m, n, k, dtype)
        pre = torch.cat((dh, dh.flip(0)), -1)
        paired(1, tile, splits)
        together = _check_backward(dh, x, w, pre, "silu", what=(m, n, k))
        paired(-1, tile, splits)
        for a, e in zip(together[:1], kernels.gated_linear_backward(dh, x, w, pre)):
            assert torch.equal(a, e), "of the same tile and parts"


def test_products_one_after_the_other(gpu, paired):
    """What is planned for both, or for one of them by itself, agrees with the formulas whichever way they go."""
    for m, n, k in ((3, 700, 520), (64, 512, 1024), (700, 300, 1160), (2500, 96, 264)):
        x, w, b, dh = _inputs(m, n, k, torch.float16)
        pre = torch.cat((dh, dh.flip(0)), -1)
        for pair in (-1, 0, 1):
            paired(pair, 0, 0)
            _check_backward(dh, x, w, pre, "gelu", what=(m, n, k, pair))


def _formula(x, w, b):
    """((h, its tolerance), (both sums, theirs)) with SiLU, as in _check_forward."""
    v, spread = x.double() @ w.double().T + b.double(), x.double().abs() @ w.double().abs().T + b.double().abs()
    e = (x.shape[-1] / 16 + 40) * U * spread
    (g, u), (eg, eu) = v.chunk(2, -1), e.chunk(2, -1)
    a, ea = _act("silu", g), 1.13 * eg + 2.0**-20 * g.abs()
    return (a * u, ea * u.abs() + (a.abs() + ea) * eu + 2 * U * (a * u).abs()), (v, e)


@pytest.mark.parametrize("m,n,k", [(20, 5504, 264), (32, 3000, 2992), (17, 6000, 72)])
def test_outputs_far_apart(gpu, m, n, k):
    """Rows of y and of the sums further apart than the tiles take, at sizes that go there otherwise."""
    from neuropress_amd import _lib

    x, w, b, _ = _inputs(m, n, k, torch.bfloat16)
    refs = _formula(x, w, b)
    far, bits = 1 << 22, dict(device="cuda", dtype=torch.int16)
    for ldy, ldp in ((far, 2 * n), (n, far), (far + 1, far + 3)):
        wide = [torch.full((m - 1, ld), 77, **bits) for ld in (ldy, ldp)]
        wide = [torch.cat((t.view(-1), torch.full((c,), 77, **bits))) for t, c in zip(wide, (n, 2 * n))]
        _lib.call("npamd_gated_linear", x.data_ptr(), k, w.data_ptr(), k, b.data_ptr(), _lib.BF16, 4, wide[0].data_ptr(), ldy, wide[1].data_ptr(), ldp, m, n, k, _lib.BF16, None, 0,
                  torch.cuda.current_stream().cuda_stream)  # fmt: skip
        for t, ld, (ref, tol) in zip(wide, (ldy, ldp), refs):
            got = t.view(torch.bfloat16).as_strided(ref.shape, (ld, 1))
            _within(got, ref, tol, torch.bfloat16, (ldy, ldp))
            got.view(torch.int16).fill_(77)
            assert bool((t == 77).all()), "between the rows"


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m,n,k", [(9, 5, 40), (70, 61, 72)])
def test_sums_that_are_not_numbers(gpu, act, m, n, k):
    """A NaN among the gate's sums or the other ones goes on into every gradient that the formula multiplies it into, and no other: the slope of an activation is NaN there."""
    from neuropress_amd import kernels

    for dtype in DTYPES:
        x, w, b, dh = _inputs(m, n, k, dtype)
        clean = kernels.gated_linear_pre(x, w, b, act)[1]
        assert bool(clean.isfinite().all())
        for row, column, bad in ((2, 1, {1, n + 1} if act else {n + 1}), (m - 1, n + 3, {3})):
            pre = clean.clone()
            pre[row, column] = float("nan")
            dx, dw, db = kernels.gated_linear_backward(dh, x, w, pre, act)
            rows, columns = torch.zeros(m, dtype=torch.bool, device="cuda"), torch.zeros(2 * n, dtype=torch.bool, device="cuda")
            rows[row] = True
            columns[list(bad)] = True
            assert torch.equal(dx.isnan(), rows[:, None].expand(m, k)) and torch.equal(dw.isnan(), columns[:, None].expand(2 * n, k)) and torch.equal(db.isnan(), columns)


@pytest.mark.parametrize("bias_dtype", [torch.float16, torch.float32])
def test_the_bias_may_change_between_the_passes(gpu, bias_dtype):
    """Its gradient needs none of its values."""
    from neuropress_amd import kernels

    x, w, b, dh = _inputs(12, 40, 72, torch.float16)
    leaves = [t.clone().requires_grad_() for t in (x, w, b.to(bias_dtype))]
    want = torch.autograd.grad(kernels.gated_linear(*leaves), leaves, dh)
    out = kernels.gated_linear(*leaves)
    with torch.no_grad():
        leaves[2].mul_(3.0)
    got = torch.autograd.grad(out, leaves, dh)
    assert got[2].dtype == bias_dtype and all(torch.equal(a, e) for a, e in zip(got, want))


@pytest.mark.parametrize("m,n,k", [(16, 512, 4096), (16, 512, 4104), (24, 3584, 3584), (32, 4096, 8192), (33, 2730, 3584), (48, 4096, 8192), (40, 4096, 8200), (17, 6912, 2048), (32, 9728, 2048), (3, 8200, 1024)])
def test_some_tokens_of_long_rows(gpu, m, n, k):
    """Both sides of the lines between the kernel for some tokens and the tiles."""
    x, w, b, _ = _inputs(m, n, k, torch.bfloat16)
    _check_forward(x, w, b, "silu")
