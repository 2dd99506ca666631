"""What the operators between a block's halves refuse before any GPU work."""

import pytest
import torch

from neuropress_amd import _lib

P = 4096  # an address that is aligned and never read: every call with it is refused, or has nothing to do
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that are none: where nothing can be launched, a call that is not refused only fails")


def _refused(name, *args, match, code=-1):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == code
    assert match in lib.npamd_last_error().decode()


@no_gpu
def test_residual_norm_refuses():
    ok = dict(x=P, ldx=64, y=P, ldy=64, w=P, wp=P, g=P, ldg=64, every=2, scale=1.0, out=P, lds=64, z=P, ldn=64, pr=None, r=None, m=4, h=64, eps=1e-6, dtype=1, st=None)
    for change, match in [(dict(h=0), "bad shape"), (dict(h=2**27 + 1), "bad shape"), (dict(m=-1), "bad shape"), (dict(dtype=3), "dtype"), (dict(ldx=63), "stride"), (dict(ldy=1), "stride"),
                          (dict(lds=63), "stride"), (dict(ldn=63), "stride"), (dict(ldg=63), "stride"), (dict(every=0), "gate_every"), (dict(x=None), "null"), (dict(y=None), "null"),
                          (dict(w=None), "null"), (dict(out=None), "null"), (dict(z=None), "null")]:  # fmt: skip
        _refused("npamd_residual_norm", *{**ok, **change}.values(), match=match)
    assert _lib.load().npamd_residual_norm(*{**ok, "m": 0, "x": None}.values()) == 0
    size = _lib.load().npamd_residual_norm_workspace_bytes
    need = size(100, 64, 100, 0)
    assert need > 0 and size(0, 64, 0, 0) == 0 == size(4, 2**27 + 1, 0, 0) == size(4, 64, 0, 5)
    ok = dict(ds=P, ldds=64, dz=P, lddz=64, y=P, ldy=64, r=P, ldr=64, w=P, wp=P, g=P, ldg=64, every=100, scale=1.0, pr=P, rstd=P, dx=P, lddx=64, dy=P, lddy=64, dw=P, dwp=P, dg=P,
              m=100, h=64, dtype=0, ws=P, n=need, st=None)  # fmt: skip
    for change, match in [(dict(h=0), "bad shape"), (dict(m=0), "bad shape"), (dict(dtype=-1), "dtype"), (dict(ldds=8), "stride"), (dict(lddz=8), "stride"), (dict(lddx=8), "stride"),
                          (dict(lddy=8), "stride"), (dict(ldg=8), "stride"), (dict(every=0), "gate_every"), (dict(ds=None, dz=None), "null"), (dict(y=None), "null"), (dict(r=None), "null"),
                          (dict(w=None), "null"), (dict(rstd=None), "null"), (dict(pr=None), "null"), (dict(ws=None), "workspace"), (dict(n=need - 1), "workspace"),
                          (dict(ws=P + 4), "workspace")]:  # fmt: skip
        _refused("npamd_residual_norm_backward", *{**ok, **change}.values(), match=match)


@no_gpu
def test_adapter_linear_refuses():
    size = _lib.load().npamd_adapter_linear_workspace_bytes
    for m in (1, 64, 65, 5000):
        need = size(m, 72, 64, 12, 4)
        ok = dict(x=P, ldx=64, ids=P, bits=32, a=P, b=P, scale=P, base=P, ldb=72, y=P, ldy=72, m=m, n=72, k=64, r=12, l=4, dtype=0, ws=P, wsn=need, st=None)
        for change, match in [(dict(m=-1), "bad shape"), (dict(n=-1), "bad shape"), (dict(k=0), "bad shape"), (dict(r=0), "bad shape"), (dict(l=0), "bad shape"), (dict(dtype=2), "f16 or bf16"),
                              (dict(bits=16), "32 or 64"), (dict(ldx=63), "stride"), (dict(ldy=71), "stride"), (dict(ldb=71), "stride"), (dict(x=None), "null"), (dict(ids=None), "null"),
                              (dict(a=None), "null"), (dict(b=None), "null"), (dict(y=None), "null"), (dict(b=P + 8), "16-byte"), (dict(a=P + 8), "16-byte"), (dict(ws=None), "workspace"), (dict(ws=P + 4), "workspace"),
                              (dict(wsn=need - 1), "workspace")]:  # fmt: skip
            _refused("npamd_adapter_linear", *{**ok, **change}.values(), match=match)
        for change in (dict(x=P + 2), dict(ldx=66), dict(k=63)):
            _refused("npamd_adapter_linear", *{**ok, **change}.values(), match="multiples of 8")
        for change in (dict(r=257), dict(l=8193), dict(m=2**22 + 1), dict(n=2**24 + 1, ldy=1 << 25, ldb=1 << 25)):
            _refused("npamd_adapter_linear", *{**ok, **change}.values(), match="at most", code=-2)
        for change in (dict(m=0), dict(n=0)):
            assert _lib.load().npamd_adapter_linear(*{**ok, **change, "x": None, "ws": None}.values()) == 0
    assert size(0, 72, 64, 12, 4) == 0 == size(4, 72, 64, 257, 4) == size(4, 72, 64, 12, 8193)


def test_workspace_of_the_residual_norm_grows_with_neither_rows_nor_sequences():
    size = _lib.load().npamd_residual_norm_workspace_bytes
    for dtype in (0, 1, 2):
        for h in (64, 1000, 4096, 8192):
            for every in (0, 1, 2, 100, 8192):
                assert size(8192, h, every, dtype) <= 3 * 256 * ((h + 7) // 8 * 8) * 4
        assert size(2**31 - 1, 64, 2, dtype) <= 3 * 256 * 64 * 4


@no_gpu
def test_gated_linear_refuses():
    far = 1 << 31
    ok = dict(x=P, ldx=64, w=P, ldw=64, b=P, bdt=2, act=4, y=P, ldy=32, pre=P, ldp=64, m=70, n=32, k=64, dtype=0, ws=None, wsn=0, st=None)
    for change, match in [(dict(k=0), "bad shape"), (dict(m=-1), "bad shape"), (dict(n=-1), "bad shape"), (dict(dtype=2), "f16 or bf16"), (dict(bdt=1), "bias"), (dict(act=5), "activation"),
                          (dict(act=-1), "activation"), (dict(ldx=63), "stride"), (dict(ldw=63), "stride"), (dict(ldp=63), "stride"), (dict(ldy=31), "stride"), (dict(x=None), "null"),
                          (dict(w=None), "null"), (dict(y=None), "null"), (dict(x=P + 2), "16-byte"), (dict(ldw=65), "16-byte"), (dict(k=63), "16-byte"), (dict(ldx=1 << 22), "16-byte"),
                          (dict(ws=P + 4), "16-byte")]:  # fmt: skip
        _refused("npamd_gated_linear", *{**ok, **change}.values(), match=match)
    for change, match in [(dict(n=2**24 + 1, ldy=far, ldp=far), "at most"), (dict(k=2**30 + 1, ldx=far, ldw=far), "at most"), (dict(ldy=1 << 22), "less than"), (dict(ldp=1 << 22), "less than")]:
        _refused("npamd_gated_linear", *{**ok, **change}.values(), match=match, code=-2)
    for m, n in ((0, 32), (70, 0)):
        assert _lib.load().npamd_gated_linear(*{**ok, "m": m, "n": n, "x": None}.values()) == 0
    size = _lib.load().npamd_gated_linear_workspace_bytes
    assert size(0, 32, 64) == 0 == size(70, 2**24 + 1, 64) == size(1, 32, 64) and size(70, 64, 8192) > 0


def test_gated_linear_of_some_tokens_goes_where_it_was_measured_to_be_faster():
    """The tiles split a long K over blocks and need workspace for it; the kernel for some tokens needs none."""
    size = _lib.load().npamd_gated_linear_workspace_bytes
    for m, n, k in ((16, 512, 14336), (24, 512, 8192), (24, 1024, 8192), (40, 512, 8192), (48, 2048, 8192)):
        assert size(m, n, k) > 0, (m, n, k)
    for m, n, k in ((16, 512, 2560), (16, 8192, 2048), (24, 3584, 3584), (32, 4096, 4096), (40, 4096, 4096), (24, 14336, 4096)):
        assert size(m, n, k) == 0, (m, n, k)


@no_gpu
def test_gated_linear_takes_outputs_far_apart_up_to_32_tokens():
    """Whatever the sizes would be best served by: outputs' rows may be any distance apart up to there."""
    far = 1 << 22
    for m in (3, 16, 17, 20, 32):
        for n, k in ((32, 64), (2048, 4096), (4864, 896), (5504, 2048), (8192, 2048)):
            for ldy, ldp in ((far, 2 * n), (n, far), (far + 1, far + 3)):
                code = _lib.load().npamd_gated_linear(P, k, P, k, P, 2, 4, P, ldy, P, ldp, m, n, k, 0, None, 0, None)
                assert code not in (0, -1, -2), (m, n, k, _lib.load().npamd_last_error())  # nothing here to launch on


@no_gpu
def test_gated_linear_backward_refuses():
    size = _lib.load().npamd_gated_linear_backward_workspace_bytes
    need = size(70, 32, 64, 1, 1, 1)
    assert need > 0 and size(0, 32, 64, 1, 1, 1) == 0
    ok = dict(dh=P, lddh=32, x=P, ldx=64, w=P, ldw=64, pre=P, ldp=64, act=4, dx=P, lddx=64, dw=P, lddw=64, db=P, bdt=2, m=70, n=32, k=64, dtype=0, ws=P, wsn=need, st=None)
    for change, match in [(dict(m=0), "bad shape"), (dict(n=0), "bad shape"), (dict(k=0), "bad shape"), (dict(dtype=2), "f16 or bf16"), (dict(bdt=1), "bias"), (dict(act=5), "activation"),
                          (dict(lddh=31), "stride"), (dict(ldp=63), "stride"), (dict(ldx=63), "stride"), (dict(ldw=63), "stride"), (dict(lddx=63), "stride"), (dict(lddw=63), "stride"),
                          (dict(dh=None), "null"), (dict(pre=None), "null"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(x=P + 2), "16-byte"), (dict(w=P + 8), "16-byte"),
                          (dict(ldx=66), "16-byte"), (dict(ldw=1 << 22), "16-byte"), (dict(ws=None), "workspace"), (dict(ws=P + 8), "workspace"), (dict(wsn=need - 1), "workspace")]:  # fmt: skip
        _refused("npamd_gated_linear_backward", *{**ok, **change}.values(), match=match)
    for change in (dict(lddx=1 << 22), dict(lddw=1 << 22)):
        _refused("npamd_gated_linear_backward", *{**ok, **change}.values(), match="less than", code=-2)


def test_wrappers_refuse_what_is_not_on_a_gpu():
    from neuropress_amd import kernels

    x, w = torch.randn(2, 64).half(), torch.randn(64).half()
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.LowRankAdapters(x[None], x[None])
    for call in (lambda: kernels.residual_norm(x, x, w), lambda: kernels.residual_norm_stats(x, x, w), lambda: kernels.residual_norm_backward(x, x, x, x, w, None, None, 1.0, None, w),
                 lambda: kernels.gated_linear(x, x), lambda: kernels.gated_linear_pre(x, x), lambda: kernels.gated_linear_backward(x[:, :1], x, x, x[:, :2])):  # fmt: skip
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_attaching_adapters_to_what_is_not_there():
    from neuropress_amd.nn import NPAdapterLinear, attach_adapters, set_adapter_ids

    model = torch.nn.Sequential(torch.nn.Linear(4, 4))
    for name in ("1", "0.weight", "a.b", ""):
        with pytest.raises(RuntimeError, match="no module|itself"):
            attach_adapters(model, {"0": None, name: None})
        assert isinstance(model[0], torch.nn.Linear)
    layer = NPAdapterLinear(model[0], None)  # without ids it is the projection
    set_adapter_ids(torch.nn.Sequential(layer), None)
    x = torch.randn(3, 4)
    assert torch.equal(layer(x), model[0](x)) and set(layer.state_dict()) == {"base.weight", "base.bias"}


def test_attaching_adapters_of_other_sizes():
    """Found when they are attached, not at the first call; nothing has been replaced then."""
    from types import SimpleNamespace

    from neuropress_amd.nn import NPAdapterLinear, attach_adapters

    model = torch.nn.Sequential(torch.nn.Linear(4, 8), torch.nn.Linear(8, 6, bias=False), torch.nn.ReLU())
    sizes = lambda k, n: SimpleNamespace(in_features=k, out_features=n)
    for wrong in (sizes(8, 4), sizes(4, 7), sizes(5, 8)):
        with pytest.raises(RuntimeError, match="0: .*_features"):
            attach_adapters(model, {"1": sizes(8, 6), "0": wrong})
        assert not any(isinstance(layer, NPAdapterLinear) for layer in model)
        with pytest.raises(RuntimeError, match="_features"):
            NPAdapterLinear(model[0], wrong)
    assert attach_adapters(model, {"0": sizes(4, 8), "1": sizes(8, 6), "2": sizes(1, 1)}) == 3  # a layer that says nothing of its sizes
    first = model[0].base
    assert attach_adapters(model, {"0": sizes(4, 8)}) == 1 and model[0].base is first
    with pytest.raises(RuntimeError, match="_features"):
        attach_adapters(model, {"0": sizes(8, 4)})


def test_attaching_adapters_leaves_modes_alone():
    from neuropress_amd.nn import NPAdapterLinear

    inner = torch.nn.Dropout().eval()
    base = torch.nn.Sequential(inner).train()
    inner.eval()
    assert NPAdapterLinear(base, None).training and base.training and not inner.training
    assert not NPAdapterLinear(base.eval(), None).training
