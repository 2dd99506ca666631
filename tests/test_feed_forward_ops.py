"""What the layer norm, the dense product with an epilogue and the experts' layer refuse before any GPU work, and (on a GPU) a run of them as a block makes it."""

import pytest
import torch

from neuropress_amd import _lib
from tests import cases

P = 4096  # an address that is aligned and never read: every call with it is refused, or has nothing to do
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are none: where nothing can be launched, a call that is not refused only fails")


def _refused(name, *args, match, code=-1):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == code
    assert match in lib.npamd_last_error().decode()


@no_gpu
def test_layer_norm_refuses():
    ok = dict(x=P, ldx=64, w=P, b=P, out=P, ldo=64, mean=None, rstd=None, m=2, h=64, eps=1e-5, dtype=1, st=None)
    for change, match in [(dict(h=0), "bad shape"), (dict(m=-1), "bad shape"), (dict(dtype=3), "dtype"), (dict(ldx=63), "stride"), (dict(ldo=1), "stride"), (dict(x=None), "null"),
                          (dict(out=None), "null")]:  # fmt: skip
        _refused("npamd_layer_norm", *{**ok, **change}.values(), match=match)
    assert _lib.load().npamd_layer_norm(*{**ok, "m": 0, "x": None}.values()) == 0
    need = _lib.load().npamd_layer_norm_workspace_bytes(100, 64)
    assert need > 0 and _lib.load().npamd_layer_norm_workspace_bytes(0, 64) == 0
    ok = dict(dy=P, lddy=64, x=P, ldx=64, w=P, mean=P, rstd=P, dx=P, lddx=64, dw=P, db=P, m=100, h=64, dtype=0, ws=P, n=need, st=None)
    for change, match in [(dict(h=0), "bad shape"), (dict(dtype=-1), "dtype"), (dict(lddy=8), "stride"), (dict(lddx=8), "stride"), (dict(mean=None), "null"), (dict(rstd=None), "null"),
                          (dict(dy=None), "null"), (dict(ws=None), "workspace"), (dict(n=need - 1), "workspace"), (dict(ws=P + 4), "workspace")]:  # fmt: skip
        _refused("npamd_layer_norm_backward", *{**ok, **change}.values(), match=match)


@no_gpu
def test_dense_gemm_act_refuses():
    ok = dict(x=P, ldx=64, w=P, ldw=64, b=P, bdt=2, act=1, r=P, ldr=32, y=P, ldy=32, m=40, n=32, k=64, dtype=0, ws=None, wsn=0, st=None)
    for change, match in [(dict(k=0), "bad shape"), (dict(m=-1), "bad shape"), (dict(dtype=2), "f16 or bf16"), (dict(bdt=1), "bias"), (dict(act=5), "activation"), (dict(act=-1), "activation"),
                          (dict(ldx=63), "stride"), (dict(ldw=63), "stride"), (dict(ldr=31), "stride"), (dict(ldy=31), "stride"), (dict(x=None), "null"), (dict(w=None), "null"),
                          (dict(y=None), "null")]:  # fmt: skip
        _refused("npamd_dense_gemm_act", *{**ok, **change}.values(), match=match)
    for m, n in ((0, 32), (40, 0)):
        assert _lib.load().npamd_dense_gemm_act(*{**ok, "m": m, "n": n, "x": None}.values()) == 0


@no_gpu
def test_moe_layer_refuses():
    need = _lib.load().npamd_moe_workspace_bytes(4, 8, 2, 128, 192)
    assert need > 0 and _lib.load().npamd_moe_workspace_bytes(0, 8, 2, 128, 192) == 0
    ok = dict(x=P, ldx=128, router=P, gu=P, gus=P, guz=None, d=P, ds=P, dz=None, y=P, ldy=128, m=4, e=8, k=2, h=128, i=192, nbits=4, gs=64, re=1, dtype=1, ws=P, wsn=need, st=None)
    for change, match in [(dict(dtype=2), "f16 or bf16"), (dict(nbits=2), "nbits"), (dict(k=0), "bad shape"), (dict(k=9), "bad shape"), (dict(m=-1), "bad shape"), (dict(gus=None), "scales"),
                          (dict(ds=None), "scales"), (dict(dz=P), "zero points"), (dict(ldx=120), "stride"), (dict(ldy=127), "stride"), (dict(router=None), "null"),
                          (dict(router=P + 2), "16-byte"), (dict(gus=P + 2), "4-byte"), (dict(gu=P + 8), "16-byte"), (dict(d=P + 8), "16-byte"), (dict(ws=None), "workspace"), (dict(wsn=need - 1), "workspace"),
                          (dict(ws=P + 8), "workspace")]:  # fmt: skip
        _refused("npamd_moe_layer", *{**ok, **change}.values(), match=match)
    for change, match in [(dict(m=33), "at most"), (dict(e=513), "at most"), (dict(e=64, k=17), "at most"), (dict(h=96), "multiples of 64"), (dict(i=160), "multiples of 64"),
                          (dict(gs=48), "group_size"), (dict(gs=16), "group_size"), (dict(gs=128), "group_size"), (dict(gs=0), "group_size")]:  # fmt: skip
        _refused("npamd_moe_layer", *{**ok, **change}.values(), match=match, code=-2)
    assert _lib.load().npamd_moe_layer(*{**ok, "m": 0, "x": None, "ws": None}.values()) == 0


@no_gpu
def test_sizes_past_the_kernels_are_refused():
    far = 1 << 31
    _refused("npamd_layer_norm", P, far, P, P, P, far, None, None, 2, 2**27 + 1, 1e-5, 1, None, match="bad shape")
    _refused("npamd_layer_norm_backward", P, far, P, far, P, P, P, P, far, None, None, 2, 2**27 + 1, 1, None, 0, None, match="bad shape")
    for n, k in ((2**25 + 1, 64), (32, 2**30 + 1)):
        _refused("npamd_dense_gemm_act", P, far, P, far, None, 2, 0, None, 0, P, far, 40, n, k, 0, None, 0, None, match="at most", code=-2)
    lib = _lib.load()
    assert lib.npamd_layer_norm_workspace_bytes(2, far - 1) == 0 == lib.npamd_moe_workspace_bytes(33, 8, 2, 128, 192)
    assert lib.npamd_moe_workspace_bytes(4, 8, 9, 128, 192) == 0 == lib.npamd_moe_workspace_bytes(4, 600, 2, 128, 192)
    assert lib.npamd_moe_workspace_bytes(1, 1, 1, 1, 1) > 0  # refused by the call, not here


def test_wrappers_refuse_what_is_not_on_a_gpu():
    from neuropress_amd import kernels

    x, w = torch.randn(2, 64).half(), torch.randn(64, 64).half()
    for call in (lambda: kernels.layer_norm(x), lambda: kernels.layer_norm_stats(x), lambda: kernels.layer_norm_backward(x, x, None, x, x), lambda: kernels.dense_linear_act(x, w),
                 lambda: kernels.MoEExperts(w, w, w)):  # fmt: skip
        with pytest.raises(RuntimeError, match="GPU"):
            call()


@pytest.mark.gpu
def test_wrappers_refuse_arguments_that_do_not_fit(gpu):
    from neuropress_amd import kernels

    x, w, v = torch.randn(2, 64, device=gpu).half(), torch.randn(32, 64, device=gpu).half(), torch.ones(64, device=gpu).half()
    with pytest.raises(RuntimeError, match="share dtype"):
        kernels.layer_norm(x, v.float())
    with pytest.raises(RuntimeError, match="matching"):
        kernels.layer_norm(x, v[:63])
    with pytest.raises(RuntimeError, match="dtype must be"):
        kernels.layer_norm(x.double())
    with pytest.raises(RuntimeError, match="at least 1"):
        kernels.layer_norm(x[:, :0])
    stat = torch.ones(2, device=gpu)
    for bad in ((x[:1], x, v, stat, stat), (x.float(), x, v, stat, stat)):
        with pytest.raises(RuntimeError, match="dy must"):
            kernels.layer_norm_backward(*bad)
    for bad in (stat[:1], stat.half()):
        with pytest.raises(RuntimeError, match="mean and rstd"):
            kernels.layer_norm_backward(x, x, v, bad, stat)
    for kwargs, match in [(dict(activation="tanh"), "activation"), (dict(bias=v[:31]), "bias"), (dict(bias=v[:32].double()), "bias"), (dict(residual=x), "residual"),
                          (dict(residual=x[:, :32].float()), "residual")]:  # fmt: skip
        with pytest.raises(RuntimeError, match=match):
            kernels.dense_linear_act(x, w, **kwargs)
    with pytest.raises(RuntimeError, match="x and w must"):
        kernels.dense_linear_act(x.float(), w.float())
    with pytest.raises(RuntimeError, match="x and w must"):
        kernels.dense_linear_act(x, w[:, :32])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 5, 32])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_feed_forward_half_of_a_block(gpu, tokens, dtype):
    """norm -> up with activation -> down added to the residual -> norm -> experts, eagerly, captured and replayed, against 64 bits."""
    from neuropress_amd import kernels
    from tests.test_gpu_moe import _experts, _layer

    h, i = 256, 640
    g = cases.gen(tokens)
    rand = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype)
    x, n1, b1, n2, b2 = rand(tokens, h), rand(h) + 1, rand(h, std=0.1), rand(h) + 1, rand(h, std=0.1)
    up, ub, down = rand(i, h, std=h**-0.5), rand(i, std=0.2), rand(h, i, std=i**-0.5)
    layer, dense = _layer(3, 8, h, 128, dtype, 4)
    experts = _experts(layer)
    on = [t.to(gpu) for t in (x, n1, b1, n2, b2, up, ub, down)]

    def block(x, n1, b1, n2, b2, up, ub, down):
        hidden = kernels.dense_linear_act(kernels.layer_norm(x, n1, b1), up, ub, "gelu")
        mid = kernels.dense_linear_act(hidden, down, residual=x)
        return mid, kernels.moe_layer(kernels.layer_norm(mid, n2, b2), experts, 2)

    mid, y = block(*on)
    f = torch.nn.functional
    d = [t.double() for t in (x, n1, b1, n2, b2, up, ub, down)]
    hidden = f.gelu(f.layer_norm(d[0], (h,), d[1], d[2]) @ d[5].T + d[6])
    ref = hidden @ d[7].T + d[0]
    # three roundings of up to a step each on values whose sums over K average them: a few steps of values of up to 8
    eps = torch.finfo(dtype).eps
    assert (mid.double().cpu() - ref).abs().max() < 16 * eps
    normed = f.layer_norm(mid.double().cpu(), (h,), d[3], d[4])
    logits = normed @ layer["router"].double().T
    p, ids = torch.softmax(logits, -1).sort(-1, descending=True)
    want = torch.zeros_like(ref)
    for m in range(tokens):
        for t in range(2):
            gate, u = (dense["gate_up"][ids[m, t]] @ normed[m]).chunk(2)
            want[m] += p[m, t] / p[m, :2].sum() * (dense["down"][ids[m, t]] @ (f.silu(gate) * u))
    clear = p[:, 1] - p[:, 2] > 0.02 * p[:, 1]  # where the rounded norm picks the same experts
    assert bool(clear.any()) and (y.double().cpu() - want)[clear].abs().max() < 24 * eps * max(1.0, want.abs().max().item())


class _Declining:
    """The native call path as it answers a call that it does not take."""

    def __init__(self, host):
        self._host, self.asked = host, []

    def __getattr__(self, name):
        if name not in ("layer_norm", "layer_norm_backward", "dense_linear_act", "moe_layer"):
            return getattr(self._host, name)
        return lambda *args: self.asked.append(name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 2, 9, 32])
def test_native_and_python_route_agree(gpu, monkeypatch, dtype, m):
    from neuropress_amd import _lib, kernels

    g = torch.Generator().manual_seed(5 + m)
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype).to("cuda")
    x, dy, w, b, res = rand(m, 192), rand(m, 192), rand(192), rand(192), rand(m, 200)
    xs = rand(2, 16, 256)[:, : (m + 1) // 2, :192]  # rows that no single distance joins
    lin, experts = rand(200, 192), kernels.MoEExperts(rand(6, 192), rand(6, 128, 192) / 14, rand(6, 192, 64) / 8)

    def calls():
        y, mean, rstd = kernels.layer_norm_stats(x, w, b, 1e-5)
        out = [y, mean, rstd, kernels.layer_norm(x, w, b), kernels.layer_norm(xs, None, b, 0), kernels.layer_norm(x[:0], w, b)]
        out += kernels.layer_norm_backward(dy, x, w, mean, rstd) + kernels.layer_norm_backward(dy.T.contiguous().T, x, None, mean, rstd, needs=(1, 0, 1))
        for args in [(x, lin), (x, lin, b.new_ones(200).float(), "silu"), (x, lin[:, ::2].repeat(1, 2), b.new_ones(200), "gelu", res), (xs, lin, None, "relu")]:
            out.append(kernels.dense_linear_act(*args))
        return out + [kernels.moe_layer(x, experts, 2), kernels.moe_layer(x, experts, 3, 0)] + ([kernels.moe_layer(xs, experts, 3, 1)] if xs.numel() <= 32 * 192 else [])

    with torch.no_grad():
        native = calls()
        host = _Declining(_lib.host())
        monkeypatch.setattr(_lib, "host", lambda: host)
        python = calls()
    assert set(host.asked) == {"layer_norm", "layer_norm_backward", "dense_linear_act", "moe_layer"}
    for a, c in zip(native, python, strict=True):
        assert (a is None) == (c is None) and (a is None or (a.dtype == c.dtype and torch.equal(a, c)))
