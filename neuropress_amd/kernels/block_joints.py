"""Between the halves of a decoder block: the residual add with the norms around it.

Operators of the framework's own, next to ``layer_norm``, ``rms_norm`` and ``dense_linear_act``, whose rules they follow: torch's current stream, outputs of torch's
allocator, ``RuntimeError`` for what the kernels do not take.
"""

from __future__ import annotations

import torch

from .. import _lib
from . import _check_device, _dt, _on_device, _rows_of, tracked

__all__ = ["residual_norm", "residual_norm_stats", "residual_norm_backward"]


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
    no or there is no such input.  *stream*, *post_rstd*, *rstd*: r and the statistics of :func:`residual_norm_stats`.  The same bits from run to run."""
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
