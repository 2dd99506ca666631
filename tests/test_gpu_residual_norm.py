"""The residual add with the norms around it, forward and backward, against the formulas in 64 bits.

Tolerances: half a step of the output type, plus what f32 adds, u = 2^-24 per operation.  A sum over a row is a chain of at most H / 64 additions, then those over lanes and waves: off by at most
n u of the sum of its terms' absolute values, n = H / 64 + 60.  A sum over M rows is a chain of at most M / 32 + 80 (blocks take at most M / 256 + 2 rows, their parts meet
in at most 16 + 16 + 8 additions).  Errors of an intermediate value go on by the formula's derivatives."""

import pytest
import torch

from tests import cases

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16, torch.float32]
U = 2.0**-24
EPS = 1e-6


def _make(shape, dtype, post=True, gate="channel", seed=0):
    g = cases.gen(seed + shape[-1] + 31 * len(shape) + 7 * shape[0])
    h = shape[-1]
    x, y = torch.randn(shape, generator=g) * 3, torch.randn(shape, generator=g) * 0.7
    x[..., :: max(1, h // 4)] *= 10
    w, p = torch.randn(h, generator=g) * 0.2 + 1, torch.randn(h, generator=g) * 0.2 + 1
    gs = {"none": None, "channel": (h,), "sequence": (shape[0], *[1] * (len(shape) - 2), h), "token": shape}[gate]
    t = [x, y, w, p if post else None, None if gs is None else torch.randn(gs, generator=g) * 0.5 + 0.5]
    return [None if v is None else v.to(dtype).cuda() for v in t]


def _half(ref, dtype):
    return ref.abs() * (torch.finfo(dtype).eps / 2) * 1.0001 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _within(got, ref, tol, dtype, what):
    assert got.dtype == dtype and got.shape == ref.shape, what
    err = (got.double() - ref).abs()
    bad = err / (tol + _half(ref, dtype))
    assert bool((bad <= 1).all()), f"{what}: {bad.max().item():.2f} of the tolerance"


def _forward(x, y, w, p, g, scale):
    """Outputs, statistics and tolerances in 64 bits."""
    x, y, w, p, g = (None if t is None else t.double() for t in (x, y, w, p, g))
    h = x.shape[-1]
    n = (h / 64 + 60) * U
    pr, b = None, y
    if p is not None:
        pr = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
        b = y * pr * p
    a = scale * b * (1 if g is None else g)
    r = x + a
    er = a.abs() * (n + 6 * U) + r.abs() * U
    rstd = torch.rsqrt(r.square().mean(-1, keepdim=True) + EPS)
    z = r * rstd * w
    ez = w.abs() * rstd * er + z.abs() * (n + er.square().mean(-1, keepdim=True).sqrt() * rstd + 4 * U)
    return r, z, pr, rstd, er, ez


def _backward(ds, dz, y, r, w, p, g, scale, pr, rstd):
    """(gradients, tolerances) of x, y, weight, post_weight, gate."""
    gate_shape = None if g is None else g.shape
    ds, dz, y, r, w, p, g = (None if t is None else t.double() for t in (ds, dz, y, r, w, p, g))
    ds = torch.zeros_like(y) if ds is None else ds
    dz = torch.zeros_like(y) if dz is None else dz
    h, m = y.shape[-1], y.numel() // y.shape[-1]
    n, k = (h / 64 + 60) * U, (m / 32 + 80) * U
    mean = lambda t: t.mean(-1, keepdim=True)
    rstd = rstd.double()[..., None]
    rh, v = r * rstd, dz * w
    c1 = mean(v * rh)
    dr = ds + rstd * (v - rh * c1)
    edr = 8 * U * (ds.abs() + rstd * (v.abs() + (rh * c1).abs())) + rstd * rh.abs() * n * mean((v * rh).abs())
    flat = lambda t: t.reshape(-1, h)
    down = lambda t, e: (flat(t).sum(0), flat(e).sum(0) + k * flat(t).abs().sum(0))
    dw = down(dz * rh, (dz * rh).abs() * 3 * U)
    one = torch.ones((), dtype=torch.float64, device=y.device)
    gg = one if g is None else g
    yh, pp = y, one
    if p is not None:
        yh, pp = y * pr.double()[..., None], p
    d, ed = scale * dr, abs(scale) * edr
    u, eu = d * gg, (ed + d.abs() * 2 * U) * gg.abs()
    b = yh * pp
    dgate = None
    if g is not None:
        t, e = d * b, (ed + d.abs() * 4 * U) * b.abs()
        lead = [i for i in range(t.dim() - 1) if len(gate_shape) < t.dim() or gate_shape[i] == 1]
        dgate = (t.sum(lead, keepdim=True).reshape(gate_shape), (e.sum(lead, keepdim=True) + k * t.abs().sum(lead, keepdim=True)).reshape(gate_shape)) if lead else (t, e)
    if p is None:
        return dr, edr, (u, eu), dw, None, dgate
    dp = down(u * yh, (eu + u.abs() * 3 * U) * yh.abs())
    c = scale * gg * b
    c2 = mean(u * pp * yh)
    ec2 = (n + 8 * U) * (mean(c.abs() * (ds.abs() + rstd * v.abs())) + rstd * mean((v * rh).abs()) * mean((c * rh).abs())) + rstd * n * mean((v * rh).abs()) * mean((c * rh).abs())
    s = pr.double()[..., None]
    dy = (s * (u * pp - yh * c2), s * (eu * pp.abs() + yh.abs() * ec2 + 6 * U * ((u * pp).abs() + (yh * c2).abs())))
    return dr, edr, dy, dw, dp, dgate


def _check_forward(t, scale, what=""):
    from neuropress_amd import kernels

    x, y, w, p, g = t
    r, z, pr, rstd, er, ez = _forward(*t, scale)
    out = kernels.residual_norm(x, y, w, p, g, scale, EPS)
    _within(out[0], r, er, x.dtype, f"stream {what}")
    _within(out[1], z, ez, x.dtype, f"normed {what}")
    stats = kernels.residual_norm_stats(x, y, w, p, g, scale, EPS)
    assert torch.equal(stats[0], out[0]) and torch.equal(stats[1], out[1])
    return stats


def _check_backward(t, scale, stats, ds, dz, what=""):
    from neuropress_amd import kernels

    x, y, w, p, g = t
    args = (ds, dz, y, stats[0], w, p, g, scale, stats[2], stats[3])
    out = kernels.residual_norm_backward(*args)
    dr, edr, dy, dw, dp, dg = _backward(*args)
    for name, got, ref in (("dx", out[0], (dr, edr)), ("dy", out[1], dy), ("dweight", out[2], dw), ("dpost", out[3], dp), ("dgate", out[4], dg)):
        if ref is None:
            assert got is None
            continue
        _within(got, *ref, x.dtype, f"{name} {what}")
    again = kernels.residual_norm_backward(*args)
    for a, b in zip(out, again):
        assert a is None and b is None or torch.equal(a, b), "the same inputs, other bits"


def _grads(shape, dtype, seed=5):
    g = cases.gen(seed)
    return [torch.randn(shape, generator=g).to(dtype).cuda() for _ in range(2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", ["none", "channel", "sequence", "token"])
@pytest.mark.parametrize("shape", [(1, 1, 64), (3, 5, 203), (2, 40, 1024), (5, 7, 4100)])
def test_forms(gpu, dtype, post, gate, shape):
    t = _make(shape, dtype, post, gate)
    stats = _check_forward(t, 0.35)
    _check_backward(t, 0.35, stats, *_grads(shape, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("h", [1, 2, 3, 4, 7, 8, 9, 63, 64, 513, 2048, 2056, 4096, 4104, 8192, 8200, 16384, 16392, 20001])
@pytest.mark.parametrize("rows", [1, 9])
def test_widths(gpu, dtype, h, rows):
    t = _make((rows, h), dtype)
    stats = _check_forward(t, -1.25)
    _check_backward(t, -1.25, stats, *_grads((rows, h), dtype))


@pytest.mark.parametrize("rows,h,gate", [(1, 300, "none"), (17, 96, "channel"), (300, 520, "channel"), (1500, 264, "sequence"), (2100, 2048, "channel"), (4099, 72, "token"), (700, 5000, "none")])
def test_rows(gpu, rows, h, gate):
    t = _make((rows, h) if gate != "sequence" else (3, rows // 3, h), torch.bfloat16, True, gate)
    stats = _check_forward(t, 0.5)
    _check_backward(t, 0.5, stats, *_grads(t[0].shape, torch.bfloat16))


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("seqs,tokens,h", [(600, 3, 128), (300, 2, 4096), (7, 1, 512), (1, 700, 256), (130, 9, 20), (3, 90, 5), (40, 3, 17000)])
def test_gates_of_many_sequences(gpu, post, seqs, tokens, h):
    t = _make((seqs, tokens, h), torch.float16, post, "sequence")
    stats = _check_forward(t, 1.0)
    _check_backward(t, 1.0, stats, *_grads((seqs, tokens, h), torch.float16))


def test_one_of_the_two_gradients(gpu):
    for gate in ("none", "channel"):
        t = _make((4, 6, 320), torch.float32, True, gate)
        stats = _check_forward(t, 1.0)
        ds, dz = _grads((4, 6, 320), torch.float32)
        _check_backward(t, 1.0, stats, ds, None)
        _check_backward(t, 1.0, stats, None, dz)


def test_needs(gpu):
    from neuropress_amd import kernels

    t = _make((4, 6, 320), torch.bfloat16, True, "sequence")
    x, y, w, p, g = t
    stats = kernels.residual_norm_stats(*t)
    ds, dz = _grads((4, 6, 320), torch.bfloat16)
    whole = kernels.residual_norm_backward(ds, dz, y, stats[0], w, p, g, 1.0, stats[2], stats[3])
    for i in range(5):
        out = kernels.residual_norm_backward(ds, dz, y, stats[0], w, p, g, 1.0, stats[2], stats[3], needs=[i == j for j in range(5)])
        assert all((o is None) == (i != j) for j, o in enumerate(out)) and torch.equal(out[i], whole[i])


def test_rows_at_any_distance_and_address(gpu):
    from neuropress_amd import kernels

    t = _make((6, 4, 333), torch.bfloat16, True, "token")
    ds, dz = _grads((6, 4, 333), torch.bfloat16)

    def spread(v, at):
        room = torch.full((*v.shape[:-1], v.shape[-1] + 13), 7.0, device="cuda", dtype=v.dtype)
        room[..., at : at + v.shape[-1]] = v
        return room[..., at : at + v.shape[-1]]

    x, y, w, p, g = t
    far = [spread(x, 1), spread(y, 5), w, p, spread(g, 3)]
    stats = kernels.residual_norm_stats(*t)
    for a, b in zip(stats, kernels.residual_norm_stats(*far)):
        assert torch.equal(a, b)
    a = kernels.residual_norm_backward(ds, dz, y, stats[0], w, p, g, 1.0, stats[2], stats[3])
    b = kernels.residual_norm_backward(spread(ds, 2), spread(dz, 7), far[1], spread(stats[0], 1), w, p, far[4], 1.0, stats[2], stats[3])
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    for a, b in zip(kernels.residual_norm(x, y, w, p, g[:1, :1]), kernels.residual_norm(x, y, w, p, g[0, 0])):  # one for all, with and without x's dimensions
        assert torch.equal(a, b)
    turned = [v.transpose(0, 1).contiguous().transpose(0, 1) for v in (x, y, g)]
    for a, b in zip(stats, kernels.residual_norm_stats(turned[0], turned[1], w, p, turned[2])):
        assert torch.equal(a, b)
    wide = g[:, :1].expand(6, 4, 333)  # one for each sequence, spelt out
    for a, b in zip(kernels.residual_norm(x, y, w, p, wide), kernels.residual_norm(x, y, w, p, g[:, :1])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("h", [64, 1037, 4096, 5, 17000])
def test_outputs_in_the_place_of_inputs(gpu, h):
    from neuropress_amd import _lib, kernels

    t = _make((50, h), torch.bfloat16, True, "channel")
    x, y, w, p, g = t
    r, z, pr, rstd = kernels.residual_norm_stats(*t)
    st = torch.cuda.current_stream().cuda_stream
    x2, y2 = x.clone(), y.clone()
    _lib.call("npamd_residual_norm", x2.data_ptr(), h, y2.data_ptr(), h, w.data_ptr(), p.data_ptr(), g.data_ptr(), h, 50, 1.0, x2.data_ptr(), h, y2.data_ptr(), h, None, None,
              50, h, EPS, _lib.BF16, st)  # fmt: skip
    assert torch.equal(x2, r) and torch.equal(y2, z)
    ds, dz = _grads((50, h), torch.bfloat16)
    ref = kernels.residual_norm_backward(ds, dz, y, r, w, p, g, 1.0, pr, rstd)
    need = _lib.load().npamd_residual_norm_workspace_bytes(50, h, 50, _lib.BF16)
    ws = torch.empty(max(4, need), dtype=torch.uint8, device="cuda")
    for into_y in (False, True):
        ds2, dz2, y2 = ds.clone(), dz.clone(), y.clone()
        dw, dp, dg = (torch.empty(h, device="cuda", dtype=torch.bfloat16) for _ in range(3))
        dy = y2 if into_y else dz2
        _lib.call("npamd_residual_norm_backward", ds2.data_ptr(), h, dz2.data_ptr(), h, y2.data_ptr(), h, r.data_ptr(), h, w.data_ptr(), p.data_ptr(), g.data_ptr(), h, 50, 1.0,
                  pr.data_ptr(), rstd.data_ptr(), ds2.data_ptr(), h, dy.data_ptr(), h, dw.data_ptr(), dp.data_ptr(), dg.data_ptr(), 50, h, _lib.BF16, ws.data_ptr(), need, st)  # fmt: skip
        for a, b in zip((ds2, dy, dw, dp, dg), ref):
            assert torch.equal(a, b)


def test_special_values_stay_in_their_rows(gpu):
    from neuropress_amd import kernels

    t = _make((4, 515), torch.float32, True, "none")
    ref = kernels.residual_norm(*t)
    t[1][1, 514] = float("nan")
    t[0][2, 3] = float("inf")
    t[0][3], t[1][3] = 0.0, 0.0
    r, z = kernels.residual_norm(*t)
    assert torch.equal(r[0], ref[0][0]) and torch.equal(z[0], ref[1][0])
    assert bool(r[1].isnan().all()) and bool(r[2, 3].isinf()) and bool(r[2, :3].isfinite().all()) and bool(z[2, 3].isnan())
    assert not bool(r[3].any()) and not bool(z[3].any())
    small = [torch.full((2, 64), v, device="cuda", dtype=torch.float32) for v in (0.0, 1e-22)]
    w = torch.ones(64, device="cuda")
    assert bool(kernels.residual_norm(*small, w, w)[1].isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gate", ["none", "sequence"])
def test_recorded(gpu, dtype, gate):
    """The node's gradients are the backward function's; r used twice, z unused and the other way round."""
    from neuropress_amd import kernels

    t = _make((3, 9, 260), dtype, gate != "none", gate)
    leaves = [None if v is None else v.clone().requires_grad_() for v in t]
    r, z = kernels.residual_norm(*leaves, scale=0.7)
    stats = kernels.residual_norm_stats(*t, scale=0.7)
    assert torch.equal(r, stats[0]) and torch.equal(z, stats[1])
    ds, dz = _grads((3, 9, 260), dtype)
    live = [v for v in leaves if v is not None]
    for use in ((ds, dz), (ds, None), (None, dz)):
        outs, grads = [o for o, d in zip((r, z), use) if d is not None], [d for d in use if d is not None]
        got = torch.autograd.grad(outs, live, grads, retain_graph=True, allow_unused=True)
        want = [v for v in kernels.residual_norm_backward(*use, t[1], stats[0], t[2], t[3], t[4], 0.7, stats[2], stats[3]) if v is not None]
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    only = kernels.residual_norm(t[0], leaves[1], *t[2:], scale=0.7)[1]
    assert only.requires_grad and torch.equal(torch.autograd.grad(only, leaves[1], dz)[0], kernels.residual_norm_backward(None, dz, t[1], stats[0], t[2], t[3], t[4], 0.7, stats[2], stats[3])[1])
    twice = torch.autograd.grad(kernels.residual_norm(*leaves)[1], leaves[0], dz, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="cannot be differentiated"):
        twice.sum().backward()


def test_gradients_against_differences(gpu):
    from neuropress_amd import kernels

    t = _make((2, 3, 48), torch.float32, True, "sequence")
    ds, dz = _grads((2, 3, 48), torch.float32)
    leaves = [v.clone().requires_grad_() for v in t]
    r, z = kernels.residual_norm(*leaves, scale=0.8)
    got = torch.autograd.grad((r, z), leaves, (ds, dz))

    def loss(v):
        r, z, *_ = _forward(*v, 0.8)
        return (r * ds.double() + z * dz.double()).sum()

    step = 1e-5
    for i, grad in enumerate(got):
        flat = t[i].double().reshape(-1)
        for at in range(0, flat.numel(), 5):
            move = torch.zeros_like(flat)
            move[at] = step
            move = move.reshape(t[i].shape)
            hi, lo = (loss([v.double() + s * move if j == i else v.double() for j, v in enumerate(t)]) for s in (1, -1))
            # a central difference of a smooth function of values around 30: step^2 and 1e-14 / step; the gradient's own f32
            assert abs(((hi - lo) / (2 * step)).item() - grad.reshape(-1)[at].item()) < 1e-4 * (1 + abs(grad.reshape(-1)[at].item()))


def test_followed_otherwise(gpu):
    """Forward mode and torch.func go through torch's own operations."""
    from neuropress_amd import kernels

    t = _make((3, 64), torch.float32, True, "channel")
    f = lambda y: kernels.residual_norm(t[0], y, *t[2:])[1]
    y, v = t[1], torch.randn_like(t[1])
    out, tangent = torch.func.jvp(f, (y,), (v,))
    assert torch.allclose(out, f(y), rtol=1e-5, atol=1e-5) and bool(tangent.isfinite().all())
    per_row = torch.func.vmap(lambda x, y: kernels.residual_norm(x, y, t[2], t[3], t[4])[0])(t[0], t[1])
    assert torch.allclose(per_row, kernels.residual_norm(*t)[0], rtol=1e-5, atol=1e-5)


def test_nothing_to_do(gpu):
    from neuropress_amd import kernels

    t = _make((2, 3, 64), torch.float32, True, "channel")
    empty = [t[0][:0], t[1][:0], *t[2:]]
    out = kernels.residual_norm_stats(*empty)
    assert [o.shape for o in out] == [(0, 3, 64), (0, 3, 64), (0, 3), (0, 3)]
    grads = kernels.residual_norm_backward(out[0], out[1], empty[1], out[0], t[2], t[3], t[4], 1.0, out[2], out[3])
    assert [g.shape for g in grads] == [(0, 3, 64), (0, 3, 64), (64,), (64,), (64,)] and not any(bool(g.any()) for g in grads)
    leaves = [v.clone().requires_grad_() for v in empty]
    kernels.residual_norm(*leaves)[1].sum().backward()
    assert leaves[2].grad.shape == (64,) and not bool(leaves[2].grad.any())


def test_refusals(gpu):
    from neuropress_amd import kernels

    x, y, w, p, g = _make((2, 3, 64), torch.float16, True, "sequence")
    for args, match in [((x, y[:, :2], w), "one shape"), ((x, y.float(), w), "one shape"), ((x, y, w[:63]), "1-D"), ((x, y, w.float()), "dtype"), ((x, y, w, p[None]), "1-D"),
                        ((x, y, w, p, g[..., :32]), "gate"), ((x, y, w, p, g.float()), "gate"), ((x, y, w, p, g[:, 0]), "gate"), ((x, y, w, p, x[:1]), "gate"), ((x, y, w.cpu()), "GPU"),
                        ((x.double(), y.double(), w.double()), "dtype"), ((x[..., :0], y[..., :0], w[:0]), "at least 1")]:  # fmt: skip
        for call in (kernels.residual_norm, kernels.residual_norm_stats):
            with pytest.raises(RuntimeError, match=match):
                call(*args)
    r, z, pr, rstd = kernels.residual_norm_stats(x, y, w, p, g)
    good = dict(dstream=x, dnormed=y, y=y, stream=r, weight=w, post_weight=p, gate=g, scale=1.0, post_rstd=pr, rstd=rstd)
    for change, match in [(dict(dstream=None, dnormed=None), "one of"), (dict(dstream=x[:1]), "shape"), (dict(dnormed=x.float()), "shape"), (dict(rstd=rstd[:1]), "rstd"),
                          (dict(rstd=rstd.half()), "rstd"), (dict(post_rstd=None), "rstd"), (dict(stream=r.cpu()), "GPU"), (dict(gate=g[:, 0]), "gate")]:  # fmt: skip
        with pytest.raises(RuntimeError, match=match):
            kernels.residual_norm_backward(**{**good, **change})


def test_each_input_by_itself(gpu):
    """One leaf that follows, the others not: its gradient is the one that all of them together give."""
    from neuropress_amd import kernels

    t = _make((2, 11, 136), torch.bfloat16, True, "sequence")
    grads = _grads((2, 11, 136), torch.bfloat16)
    all_leaves = [v.clone().requires_grad_() for v in t]
    want = torch.autograd.grad(kernels.residual_norm(*all_leaves, scale=0.6), all_leaves, grads)
    for i in range(5):
        leaves = [v.clone().requires_grad_(j == i) for j, v in enumerate(t)]
        got = torch.autograd.grad(kernels.residual_norm(*leaves, scale=0.6), leaves[i], grads)[0]
        assert torch.equal(got, want[i])


@pytest.mark.parametrize("dtype", DTYPES)
def test_broadcast_gradients_and_inputs(gpu, dtype):
    """The gradient of a sum, one value for all, and inputs whose rows are one row or lie the other way round."""
    from neuropress_amd import kernels

    t = _make((6, 10, 72), dtype, True, "channel")
    one = torch.ones((6, 10, 72), dtype=dtype, device="cuda")
    for x, y in ((t[0], t[1]), (t[0][:1].expand(6, -1, -1), t[1][:, :1].expand(-1, 10, -1)), (t[0].transpose(0, 1).contiguous().transpose(0, 1), t[1].permute(2, 0, 1).contiguous().permute(1, 2, 0))):
        same = [x.contiguous(), y.contiguous(), *t[2:]]
        stats = _check_forward(same, 0.9)
        leaves = [v.detach().requires_grad_() for v in (x, y, *t[2:])]
        r, z = kernels.residual_norm(*leaves, scale=0.9)
        assert torch.equal(r, stats[0]) and torch.equal(z, stats[1])
        got = torch.autograd.grad(r.sum() + z.sum(), leaves)
        want = kernels.residual_norm_backward(one, one, same[1], stats[0], *t[2:], 0.9, stats[2], stats[3])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_one_tensor_as_both_inputs(gpu):
    from neuropress_amd import kernels

    t = _make((7, 264), torch.float32, True, "none")
    stats = _check_forward([t[0], t[0], *t[2:]], 0.5)
    leaf = t[0].clone().requires_grad_()
    ds, dz = _grads((7, 264), torch.float32)
    got = torch.autograd.grad(kernels.residual_norm(leaf, leaf, t[2], t[3], scale=0.5), leaf, (ds, dz))[0]
    want = kernels.residual_norm_backward(ds, dz, t[0], stats[0], t[2], t[3], None, 0.5, stats[2], stats[3])
    assert torch.equal(got, want[0] + want[1])


@pytest.mark.parametrize("rows,every", [(1000, 1000), (1000, 37), (777, 300), (513, 512)])
def test_rows_of_a_part_lie_apart(gpu, rows, every):
    """Blocks take every so manieth row of a gate's: the last gate has fewer rows than there are parts."""
    from neuropress_amd import _lib, kernels

    t = _make((rows, 200), torch.float32, True, "none")
    gate = torch.randn((rows + every - 1) // every, 200, generator=cases.gen(rows)).cuda()
    wide = gate.repeat_interleave(every, 0)[:rows].contiguous()
    stats = kernels.residual_norm_stats(*t[:4], wide, 0.8)
    ds, dz = _grads((rows, 200), torch.float32)
    _check_backward([*t[:4], wide], 0.8, stats, ds, dz)
    whole = rows // every * every
    if whole:  # as sequences, with the rows of the last, shorter one left out
        seq = [v[:whole].view(-1, every, 200) for v in t[:2]]
        _check_backward([*seq, t[2], t[3], gate[: rows // every, None]], 0.8, [s[:whole].view(-1, every, *s.shape[1:]) for s in stats],
                        *(d[:whole].view(-1, every, 200) for d in (ds, dz)))  # fmt: skip
    # through the C interface, whose last gate may have fewer rows
    out = [torch.empty_like(t[0]), torch.empty_like(t[0]), torch.empty(200, device="cuda"), torch.empty(200, device="cuda"), torch.empty_like(gate)]
    lib = _lib.load()
    need = lib.npamd_residual_norm_workspace_bytes(rows, 200, every, 2)
    scratch = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
    p = lambda v: v.data_ptr()
    rc = lib.npamd_residual_norm_backward(p(ds), 200, p(dz), 200, p(t[1]), 200, p(stats[0]), 200, p(t[2]), p(t[3]), p(gate), 200, every, 0.8, p(stats[2]), p(stats[3]), p(out[0]), 200, p(out[1]),
                                          200, p(out[2]), p(out[3]), p(out[4]), rows, 200, 2, p(scratch), need, torch.cuda.current_stream().cuda_stream)  # fmt: skip
    assert rc == 0
    dr, edr, dy, dw, dp, dg = _backward(ds, dz, t[1], stats[0], t[2], t[3], wide, 0.8, stats[2], stats[3])
    seg = lambda v: torch.stack([v[i : i + every].sum(0) for i in range(0, rows, every)])
    k = (rows / 32 + 80) * U
    for got, ref in zip(out, ((dr, edr), dy, dw, dp, (seg(dg[0]), seg(dg[1]) + k * seg(dg[0].abs())))):
        _within(got, *ref, torch.float32, f"{rows} rows, a gate for {every}")


@pytest.mark.parametrize("dtype,h", [(torch.bfloat16, 513), (torch.bfloat16, 1025), (torch.float16, 4100), (torch.bfloat16, 8193), (torch.float32, 257), (torch.float32, 4099)])
@pytest.mark.parametrize("gate", ["none", "channel", "token"])
def test_gradients_in_the_place_of_inputs_without_the_norm_behind(gpu, dtype, h, gate):
    """The last two pieces of these rows overlap and are those of two waves: what one of them stores the other may not read any more."""
    from neuropress_amd import _lib, kernels

    rows, code = 300, {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}[dtype]
    x, y, w, _, g = _make((rows, h), dtype, False, gate)
    r, _, _, rstd = kernels.residual_norm_stats(x, y, w, None, g)
    ds, dz = _grads((rows, h), dtype)
    ref = kernels.residual_norm_backward(ds, dz, y, r, w, None, g, 1.0, None, rstd)
    every = 0 if g is None else 1 if gate == "token" else rows
    need = _lib.load().npamd_residual_norm_workspace_bytes(rows, h, every, code)
    ws = torch.empty(max(4, need), dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    for into_y in (False, True):
        ds2, dz2, y2, dw = ds.clone(), dz.clone(), y.clone(), torch.empty(h, device="cuda", dtype=dtype)
        dg = None if g is None else torch.empty_like(g)
        dy = y2 if into_y else dz2
        _lib.call("npamd_residual_norm_backward", ds2.data_ptr(), h, dz2.data_ptr(), h, y2.data_ptr(), h, r.data_ptr(), h, w.data_ptr(), None, None if g is None else g.data_ptr(), h,
                  max(1, every), 1.0, None, rstd.data_ptr(), ds2.data_ptr(), h, dy.data_ptr(), h, dw.data_ptr(), None, None if g is None else dg.data_ptr(), rows, h, code,
                  ws.data_ptr(), need, st)  # fmt: skip
        for a, b in zip((ds2, dy, dw, None, dg), ref):
            assert a is None and b is None or torch.equal(a, b)


@pytest.mark.parametrize("post", [False, True])
def test_the_stream_may_change_between_the_passes(gpu, post):
    """No gradient needs x's values: a leaf that an optimizer, say, has changed meanwhile is no error; y's values are needed, and torch says so."""
    from neuropress_amd import kernels

    t = _make((6, 515), torch.bfloat16, post, "none")
    ds, dz = _grads((6, 515), torch.bfloat16)
    x, y, w = (v.clone().requires_grad_() for v in t[:3])
    want = torch.autograd.grad(kernels.residual_norm(x, y, w, t[3]), (x, y, w), (ds, dz))
    out = kernels.residual_norm(x, y, w, t[3])
    with torch.no_grad():
        x.mul_(3.0)
    for a, b in zip(torch.autograd.grad(out, (x, y, w), (ds, dz)), want):
        assert torch.equal(a, b)
    out = kernels.residual_norm(x, y, w, t[3])
    with torch.no_grad():
        y.mul_(3.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, (x, y, w), (ds, dz))
