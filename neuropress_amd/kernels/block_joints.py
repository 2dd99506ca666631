"""What joins the halves of a decoder block: the residual add with the norms around it, the gated product of a feed-forward half, and
low-rank adapters beside a projection.

Operators of the framework's own, next to ``layer_norm``, ``rms_norm`` and ``dense_linear_act``, whose rules they follow: torch's current stream, outputs of torch's
allocator, ``RuntimeError`` for what the kernels do not take.
"""

from __future__ import annotations

import torch

from .. import _lib
from . import ACTIVATIONS, _check_device, _dt, _on_device, _rows_of, tracked

__all__ = ["residual_norm", "residual_norm_stats", "residual_norm_backward", "gated_linear", "gated_linear_pre", "gated_linear_backward", "LowRankAdapters",
           "adapter_linear"]  # fmt: skip


def _residual_args(what, x, y, weight, post_weight, gate) -> int:
    """Checks the arguments that the forward and the backward pass share; returns the number of rows."""
    _check_device(what, x, y, weight, post_weight, gate)
    _dt(x.dtype, what)
    if x.dim() < 1 or x.shape[-1] < 1 or y.shape != x.shape or y.dtype != x.dtype:
        raise RuntimeError(f"{what}: x and y must be [..., H] of one shape and dtype with H of at least 1")
    h = x.shape[-1]
    for p in (weight, post_weight):
        if p is not None and (p.shape != (h,) or p.dtype != x.dtype):
            raise RuntimeError(f"{what}: the weights must be 1-D [H] in x's dtype")
    if gate is not None:
        shape, lead = list(gate.shape), list(x.shape[:-1])
        same = 0
        while same < len(lead) and len(shape) == x.dim() and shape[same] == lead[same]:
            same += 1
        if gate.dtype != x.dtype or (shape != [h] and shape != lead[:same] + [1] * (len(lead) - same) + [h]):
            raise RuntimeError(f"{what}: the gate must be [H], x's shape, or x's first dimensions, ones and H, in x's dtype; got {gate.dtype} {shape}")
    return _rows_of(what, x, h)


def _torch_residual_norm(x, y, weight, post_weight, gate, scale, eps):
    b, r = y.float(), x.float()
    if post_weight is not None:
        b = b * torch.rsqrt(b.square().mean(-1, keepdim=True) + eps) * post_weight.float()
    if gate is not None:
        b = b * gate.float()
    r = r + scale * b
    return r.to(x.dtype), (r * torch.rsqrt(r.square().mean(-1, keepdim=True) + eps) * weight.float()).to(x.dtype)


def _residual_norm(what, x, y, weight, post_weight, gate, scale, eps, stats):
    if _residual_args(what, x, y, weight, post_weight, gate) == 0:
        out = (torch.empty_like(x), torch.empty_like(x))
        rows = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
        return (*out, None if post_weight is None else rows, rows.clone()) if stats else out
    with torch.no_grad(), _on_device(x):
        x, y, weight, post_weight, gate = (None if t is None else t.detach().contiguous() for t in (x, y, weight, post_weight, gate))
        out = _lib.host().residual_norm(x, y, weight, post_weight, gate, float(scale), float(eps), stats)
    if out is None:
        raise RuntimeError(f"{what}: no kernel for these tensors")
    return out


def residual_norm(
    x: torch.Tensor,
    y: torch.Tensor,
    weight: torch.Tensor,
    post_weight: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    scale: float = 1.0,
    eps: float = 1e-6,
) -> tuple[torch.Tensor, torch.Tensor]:
    """``(r, z)`` of a residual stream *x* ``[..., H]`` and the output *y* of a half of a block (``npamd_residual_norm``): ``r = x + scale * gate * b`` with b the RMS norm of y
    with *post_weight*, or y where that is None, and ``z`` the RMS norm of r, before it is rounded, with *weight*: what the next half takes.

    *gate*: None, ``[H]``, x's shape, or x's first dimensions with ones behind them (``[B, 1, H]``: one for each sequence).  All in one of float16, bfloat16 and float32; any H.
    Where a gradient is recorded the backward pass is :func:`residual_norm_backward`'s kernels (first derivatives; captured under the terms of :func:`layer_norm`).  Calls that torch follows
    in other ways go through torch's own operations, in float32.
    """
    out = _lib.host().residual_norm(x, y, weight, post_weight, gate, scale, eps, False)
    if out is not None:
        return out
    what = "residual_norm"
    tensors = [t for t in (x, y, weight, post_weight, gate) if t is not None]
    if not any(tracked(t) for t in tensors):
        return _residual_norm(what, x, y, weight, post_weight, gate, scale, eps, False)
    rows = _residual_args(what, x, y, weight, post_weight, gate)
    with torch.no_grad():  # what is left of it when no gradient is recorded
        otherwise = any(tracked(t) for t in tensors)
    if otherwise or rows == 0:
        return _torch_residual_norm(x, y, weight, post_weight, gate, float(scale), float(eps))
    return _lib.host().residual_norm_recorded(x, y, weight, post_weight, gate, float(scale), float(eps))


def residual_norm_stats(
    x: torch.Tensor,
    y: torch.Tensor,
    weight: torch.Tensor,
    post_weight: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    scale: float = 1.0,
    eps: float = 1e-6,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None, torch.Tensor]:
    """:func:`residual_norm` without a recorded gradient, and the reciprocal root mean squares (float32 ``[...]``) of y (None without *post_weight*) and of r that
    :func:`residual_norm_backward` takes."""
    out = _lib.host().residual_norm(x, y, weight, post_weight, gate, scale, eps, True)
    return out if out is not None else _residual_norm("residual_norm_stats", x, y, weight, post_weight, gate, scale, eps, True)


def residual_norm_backward(
    dstream: torch.Tensor | None,
    dnormed: torch.Tensor | None,
    y: torch.Tensor,
    stream: torch.Tensor,
    weight: torch.Tensor,
    post_weight: torch.Tensor | None,
    gate: torch.Tensor | None,
    scale: float,
    post_rstd: torch.Tensor | None,
    rstd: torch.Tensor,
    needs: tuple[bool, bool, bool, bool, bool] = (True, True, True, True, True),
) -> tuple[torch.Tensor | None, ...]:
    """Gradients of x, y, weight, post_weight and gate (``npamd_residual_norm_backward``) from those of r and z (None for one of them: zero), in y's dtype; None where *needs* says
    no or there is no such input.  *stream*, *post_rstd*, *rstd*: r as it was rounded and the statistics of :func:`residual_norm_stats`.  The sums over rows are float32 from 8 to 16384 columns
    (float32 rows: 4 to 8192), float64 otherwise.  The same bits from run to run."""
    out = _lib.host().residual_norm_backward(dstream, dnormed, y, stream, weight, post_weight, gate, scale, post_rstd, rstd, *needs)
    if out is not None:
        return out
    what = "residual_norm_backward"
    rows = _residual_args(what, stream, y, weight, post_weight, gate)
    if dstream is None and dnormed is None:
        raise RuntimeError(f"{what}: one of dstream and dnormed has to be there")
    for t in (dstream, dnormed):
        if t is not None and (t.shape != y.shape or t.dtype != y.dtype):
            raise RuntimeError(f"{what}: dstream and dnormed must have y's shape and dtype")
    stats = [rstd] if post_weight is None else [rstd, post_rstd]
    for t in stats:
        if t is None or t.dtype != torch.float32 or t.numel() != rows:
            raise RuntimeError(f"{what}: rstd and, with post_weight, post_rstd must be float32, one for each row")
    _check_device(what, y, dstream, dnormed, *stats)
    if rows == 0:
        like = (y, y, weight, post_weight, gate)
        return tuple(torch.zeros_like(t) if need and t is not None else None for t, need in zip(like, needs))
    with torch.no_grad(), _on_device(y):
        tensors = [None if t is None else t.detach().contiguous() for t in (dstream, dnormed, y, stream, weight, post_weight, gate, post_rstd if post_weight is not None else None, rstd)]
        out = _lib.host().residual_norm_backward(*tensors[:7], float(scale), *tensors[7:], *(bool(n) for n in needs))
    if out is None:
        raise RuntimeError(f"{what}: no kernel for these tensors")
    return out


def _gated_args(what, x, gate_up, bias, activation) -> tuple[int, int]:
    """Checks the arguments that the forward and the backward pass share; returns the number of rows and of columns of the output."""
    _check_device(what, x, gate_up, bias)
    if x.dtype not in (torch.float16, torch.bfloat16) or gate_up.dtype != x.dtype or gate_up.dim() != 2 or x.dim() < 1 or gate_up.shape[1] != x.shape[-1] or gate_up.shape[0] % 2:
        raise RuntimeError(f"{what}: x and gate_up must be float16 or bfloat16 [..., K] and [2 N, K]")
    if activation not in ACTIVATIONS:
        raise RuntimeError(f"{what}: activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    if x.shape[-1] < 1:
        raise RuntimeError(f"{what}: K must be at least 1")
    if bias is not None and (bias.dtype not in (torch.float32, x.dtype) or bias.shape != gate_up.shape[:1]):
        raise RuntimeError(f"{what}: bias must be [2 N] in float32 or x's dtype")
    _rows_of(what, gate_up, x.shape[-1])
    return _rows_of(what, x, x.shape[-1]), gate_up.shape[0] // 2


def _torch_gated_linear(x, gate_up, bias, activation):
    f = torch.nn.functional
    gate, up = f.linear(x, gate_up, None if bias is None else bias.to(gate_up.dtype)).chunk(2, -1)
    if activation is not None:
        gate = f.gelu(gate, approximate="tanh") if activation == "gelu_tanh" else getattr(f, activation)(gate)
    return gate * up


def _gated_linear(what, x, gate_up, bias, activation, pre):
    rows, n = _gated_args(what, x, gate_up, bias, activation)
    if rows == 0 or n == 0:
        out = x.new_empty((*x.shape[:-1], n))
        return (out, x.new_empty((*x.shape[:-1], 2 * n))) if pre else out
    with torch.no_grad(), _on_device(x):
        x, gate_up, bias = (None if t is None else t.detach().contiguous() for t in (x, gate_up, bias))
        out = _lib.host().gated_linear(x, gate_up, bias, ACTIVATIONS[activation], pre)
    if out is None:
        raise RuntimeError(f"{what}: no kernel for these tensors")
    return out


def gated_linear(x: torch.Tensor, gate_up: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = "silu") -> torch.Tensor:
    """``act(x @ gate.T + bias) * (x @ up.T + bias)`` of an fp16 / bf16 *x* ``[..., K]`` and *gate_up* ``[2 N, K]`` of its dtype, N gate rows before N up rows (as
    :class:`MoEExperts` has them), rounded once (``npamd_gated_linear``): the first half of a gated feed-forward block in one kernel.

    *activation*: as for :func:`dense_linear_act`; *bias* ``[2 N]`` in float32 or x's dtype.  Any number of tokens, N below 2**21 and K below 2**22 (a few tokens: 2**24 and 2**30).  Where a gradient is recorded both sums are kept, rounded to x's dtype, and the
    backward pass is :func:`gated_linear_backward`'s kernels (first derivatives; captured under the terms of :func:`layer_norm`).  Calls that torch follows in other ways go through torch's
    own operations, which round in between.
    """
    code = ACTIVATIONS.get(activation)
    out = None if code is None else _lib.host().gated_linear(x, gate_up, bias, code, False)
    if out is not None:
        return out
    what = "gated_linear"
    tensors = [t for t in (x, gate_up, bias) if t is not None]
    if not any(tracked(t) for t in tensors):
        return _gated_linear(what, x, gate_up, bias, activation, False)
    rows, n = _gated_args(what, x, gate_up, bias, activation)
    with torch.no_grad():  # what is left of it when no gradient is recorded
        otherwise = any(tracked(t) for t in tensors)
    if otherwise or rows == 0 or n == 0:
        return _torch_gated_linear(x, gate_up, bias, activation)
    return _lib.host().gated_linear_recorded(x, gate_up, bias, code)


def gated_linear_pre(x: torch.Tensor, gate_up: torch.Tensor, bias: torch.Tensor | None = None, activation: str | None = "silu") -> tuple[torch.Tensor, torch.Tensor]:
    """:func:`gated_linear` without a recorded gradient, and both sums ``[..., 2 N]`` in x's dtype, which :func:`gated_linear_backward` takes."""
    code = ACTIVATIONS.get(activation)
    out = None if code is None else _lib.host().gated_linear(x, gate_up, bias, code, True)
    return out if out is not None else _gated_linear("gated_linear_pre", x, gate_up, bias, activation, True)


def gated_linear_backward(
    dh: torch.Tensor,
    x: torch.Tensor,
    gate_up: torch.Tensor,
    pre: torch.Tensor,
    activation: str | None = "silu",
    needs: tuple[bool, bool, bool] = (True, True, True),
    bias_dtype: torch.dtype | None = None,
) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """Gradients of x, gate_up and the bias (``npamd_gated_linear_backward``) from that of the output, in x's dtype (the bias's in *bias_dtype*, float32 or x's); None where *needs* says
    no.  *pre*: of :func:`gated_linear_pre`.  The gradients of both sums go into the products rounded to x's dtype (float16: infinite past 65504), the products' and the bias's sums are float32.  The same bits from run to
    run."""
    what = "gated_linear_backward"
    code = ACTIVATIONS.get(activation)
    wide = bias_dtype == torch.float32
    if bias_dtype not in (None, torch.float32, x.dtype):
        raise RuntimeError(f"{what}: bias_dtype must be float32 or x's dtype, got {bias_dtype}")
    out = None if code is None else _lib.host().gated_linear_backward(dh, x, gate_up, pre, code, wide, *needs)
    if out is not None:
        return out
    rows, n = _gated_args(what, x, gate_up, None, activation)
    _check_device(what, x, dh, pre)
    if dh.dtype != x.dtype or pre.dtype != x.dtype or dh.shape != (*x.shape[:-1], n) or pre.shape != (*x.shape[:-1], 2 * n):
        raise RuntimeError(f"{what}: dh and pre must be [..., N] and [..., 2 N] in x's dtype")
    if rows == 0 or n == 0:
        made = (lambda: torch.zeros_like(x), lambda: torch.zeros_like(gate_up), lambda: torch.zeros(2 * n, device=x.device, dtype=bias_dtype or x.dtype))
        return tuple(make() if need else None for make, need in zip(made, needs))
    with torch.no_grad(), _on_device(x):
        dh, x, gate_up, pre = (t.detach().contiguous() for t in (dh, x, gate_up, pre))
        out = _lib.host().gated_linear_backward(dh, x, gate_up, pre, code, wide, *(bool(need) for need in needs))
    if out is None:
        raise RuntimeError(f"{what}: no kernel for these tensors")
    return out


class LowRankAdapters:
    """The adapters of one projection, checked and laid out once, for :func:`adapter_linear`.

    *a* ``[L, r, K]`` and *b* ``[L, N, r]`` in float16 or bfloat16, *scale* float32 ``[L]`` or None (1): adapter i adds ``scale[i] * (x @ a[i].T) @ b[i].T``.  Ranks up to 256, up to
    8192 adapters.  Ranks and columns that are no multiples of eight are padded (a copy); otherwise the tensors are kept as they are.
    """

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scale: torch.Tensor | None = None):
        what = "LowRankAdapters"
        _check_device(what, a, b, scale)
        if a.dtype not in (torch.float16, torch.bfloat16) or b.dtype != a.dtype or a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise RuntimeError(f"{what}: a and b must be float16 or bfloat16 [L, r, K] and [L, N, r]")
        if min(*a.shape, *b.shape) < 1:
            raise RuntimeError(f"{what}: at least one adapter, rank, column and row, got {list(a.shape)} and {list(b.shape)}")
        if scale is not None and (scale.dtype != torch.float32 or scale.shape != a.shape[:1]):
            raise RuntimeError(f"{what}: scale must be float32 [L]")
        self.adapters, self.rank, self.in_features = a.shape
        self.out_features = b.shape[1]
        if self.rank > 256 or self.adapters > 8192:
            raise RuntimeError(f"{what}: ranks up to 256 and up to 8192 adapters, got {self.rank} and {self.adapters}")
        a, b = a.detach(), b.detach()
        if self.rank % 8:
            b = torch.nn.functional.pad(b, (0, -self.rank % 8))
        if self.in_features % 8:
            a = torch.nn.functional.pad(a, (0, -self.in_features % 8))
        a, b = a.contiguous(), b.contiguous()
        self.a, self.b = (t if t.data_ptr() % 16 == 0 else t.clone() for t in (a, b))
        self.scale = None if scale is None else scale.detach().contiguous()


def adapter_linear(x: torch.Tensor, adapters: LowRankAdapters, ids: torch.Tensor, base: torch.Tensor | None = None) -> torch.Tensor:
    """``base + scale[i] * (x @ a[i].T) @ b[i].T`` with i each token's adapter (``npamd_adapter_linear``): the adapters of many requests at once, next to a projection of *x*
    ``[..., K]`` that they share, whose output is *base* ``[..., N]`` (None: zero).

    *ids*: int32 or int64, one for each token (x's dimensions but the last) or for each of the first of x's dimensions (``[B]`` for x ``[B, T, K]``); a number that is no adapter's, such as
    -1, leaves its tokens' base as it is.  Tokens may come in any order; an adapter's weights are read once for up to 16 of its tokens in a decode step, in a prompt *a* for up to 32 or 64 and *b* for up to 32 to 128.  For inference: calls that torch
    follows (:func:`tracked`) are refused.
    """
    y = _lib.host().adapter_linear(x, ids, adapters.a, adapters.b, adapters.scale, base, adapters.in_features, adapters.out_features)
    if y is not None:
        return y
    what = "adapter_linear"
    _check_device(what, x, ids, base, adapters.a)
    k, n = adapters.in_features, adapters.out_features
    if x.dtype != adapters.a.dtype or x.dim() < 1 or x.shape[-1] != k:
        raise RuntimeError(f"{what}: x must be {adapters.a.dtype} [..., {k}], got {x.dtype} {list(x.shape)}")
    lead = x.shape[:-1]
    if ids.dtype not in (torch.int32, torch.int64) or ids.shape != lead[: ids.dim()]:
        raise RuntimeError(f"{what}: ids must be int32 or int64, one for each token or for each of the first of x's dimensions, got {ids.dtype} {list(ids.shape)}")
    if base is not None and (base.dtype != x.dtype or base.shape != (*lead, n)):
        raise RuntimeError(f"{what}: base must be {[*lead, n]} in x's dtype")
    if tracked(x) or (base is not None and tracked(base)):
        raise RuntimeError(f"{what}: for inference only: no gradient, trace or transform of torch can follow it")
    rows = _rows_of(what, x, k)
    if rows > 1 << 22 or n > 1 << 24:
        raise RuntimeError(f"{what}: at most 2**22 tokens and 2**24 columns, got {rows} and {n}")
    if rows == 0:
        return x.new_empty((*lead, n))
    with torch.no_grad(), _on_device(x):
        ids = ids.reshape(*ids.shape, *[1] * (len(lead) - ids.dim())).expand(lead).contiguous()
        x = x.detach().contiguous()
        y = _lib.host().adapter_linear(x, ids, adapters.a, adapters.b, adapters.scale, None if base is None else base.detach().contiguous(), k, n)
    if y is None:
        raise RuntimeError(f"{what}: no kernel for these tensors")
    return y
