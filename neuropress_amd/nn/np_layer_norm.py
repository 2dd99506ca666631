"""NPLayerNorm: layer norm as one HIP kernel, its backward pass as one or two, and the pass that installs it.

A neighbour of :mod:`.np_rms_norm` for models that norm with mean and variance.  It replaces ``nn.LayerNorm`` over the last dimension on a GPU; the
parameters stay the module's own objects, so optimizers and ``state_dict`` keys go on as before.  ``AutoKernelLowering`` runs the pass with
``norm_backend="all"``.
"""

from __future__ import annotations

import logging

import torch
from torch import nn

__all__ = ["NPLayerNorm", "linearize_layer_norms"]

log = logging.getLogger(__name__)

_HOOKS = ("_forward_hooks", "_forward_pre_hooks", "_backward_hooks", "_backward_pre_hooks", "_state_dict_hooks", "_state_dict_pre_hooks",
          "_load_state_dict_pre_hooks", "_load_state_dict_post_hooks")  # fmt: skip
_DTYPES = (torch.float16, torch.bfloat16, torch.float32)  # of the kernels


class NPLayerNorm(nn.Module):
    """``(x - mean) * rstd * weight + bias`` over the last dimension in f32 arithmetic, rounded once to x's dtype; differentiable.  Types, and what autocast makes of
    them, are those of ``nn.LayerNorm``."""

    def __init__(self, weight: nn.Parameter | None, bias: nn.Parameter | None, width: int, eps: float = 1e-5, source: nn.Module | None = None) -> None:
        super().__init__()
        self.register_parameter("weight", weight)
        self.register_parameter("bias", bias)
        self.width = width
        self.eps = eps
        self.__dict__["_source"] = source  # outside the module tree: no state_dict entries

    def to_source_module(self) -> nn.Module | None:
        """The module this one replaced, with this one's parameters."""
        source = self.__dict__.get("_source")
        if source is not None:
            source.weight, source.bias = self.weight, self.bias
            source.train(self.training)
        return source

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        w, b = self.weight, self.bias
        # Types that the kernels do not have, and parameters of another type, are torch's to decide on, as they were the replaced module's: under autocast it norms in float32 with the
        # parameters as they are, without it refuses.
        if x.is_cuda and x.dtype in _DTYPES and all(p is None or p.dtype == x.dtype for p in (w, b)):
            from .. import kernels

            if x.shape[-1:] != (self.width,):
                raise RuntimeError(f"NPLayerNorm: x must be [..., {self.width}], got {list(x.shape)}")
            return kernels.layer_norm(x, w, b, self.eps)
        return nn.functional.layer_norm(x, (self.width,), w, b, self.eps)

    def extra_repr(self) -> str:
        return f"H={self.width}, eps={self.eps}, weight={self.weight is not None}, bias={self.bias is not None}"


def _fits(module: nn.Module) -> bool:
    """Whether the kernels can norm what *module* norms: one dimension, with a weight on a GPU, of a type that they have."""
    w = module.weight
    return len(module.normalized_shape) == 1 and w is not None and w.device.type == "cuda" and w.dtype in _DTYPES


def _as_made(module: nn.Module) -> bool:
    """Whether nothing was hung on *module* that its replacement would not have: a hook, a forward of its own, another parameter, buffer or child."""
    own = vars(module)
    return not any(own.get(name) for name in _HOOKS) and "forward" not in own and set(own["_parameters"]) <= {"weight", "bias"} and not own["_buffers"] and not own["_modules"]


def linearize_layer_norms(model: nn.Module) -> int:
    """Replace every ``nn.LayerNorm`` inside *model* that has a weight on a GPU, of a type that the kernels have, and norms one dimension; returns how many.
    Subclasses are left alone: what they override is theirs; so are modules with hooks, which would be lost."""
    from .backends import is_hip_backend_available

    if not is_hip_backend_available():
        log.debug("linearize_layer_norms: HIP kernel library unavailable - skipping")
        return 0
    fused: dict[int, NPLayerNorm] = {}  # a module that stands in several places is replaced by one
    for name, mod in list(model.named_modules(remove_duplicate=False)):
        if not name or type(mod) is not nn.LayerNorm or not _fits(mod) or not _as_made(mod):
            continue
        if id(mod) not in fused:
            fused[id(mod)] = NPLayerNorm(mod.weight, mod.bias, mod.normalized_shape[0], mod.eps, source=mod).train(mod.training)
        parent_name, _, attr = name.rpartition(".")
        setattr(model.get_submodule(parent_name) if parent_name else model, attr, fused[id(mod)])
    return len(fused)
