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


def test_workspace_of_the_residual_norm_grows_with_neither_rows_nor_sequences():
    size = _lib.load().npamd_residual_norm_workspace_bytes
    for dtype in (0, 1, 2):
        for h in (64, 1000, 4096, 8192):
            for every in (0, 1, 2, 100, 8192):
                assert size(8192, h, every, dtype) <= 3 * 256 * ((h + 7) // 8 * 8) * 4
        assert size(2**31 - 1, 64, 2, dtype) <= 3 * 256 * 64 * 4


def test_wrappers_refuse_what_is_not_on_a_gpu():
    from neuropress_amd import kernels

    x, w = torch.randn(2, 64).half(), torch.randn(64).half()
    for call in (lambda: kernels.residual_norm(x, x, w), lambda: kernels.residual_norm_stats(x, x, w), lambda: kernels.residual_norm_backward(x, x, x, x, w, None, None, 1.0, None, w)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
