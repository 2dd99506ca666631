"""NPAdapterLinear: a projection, quantized or dense, with the low-rank adapters of many requests beside it.

The projection stays the module it was (``NPLinear``, ``NPVQLinear``, ``nn.Linear``); what it gives is the base that the adapters add to, two launches for a decode step
whatever the number of requests and adapters.
"""

from __future__ import annotations

import torch
from torch import nn

from ..kernels import LowRankAdapters, adapter_linear

__all__ = ["NPAdapterLinear", "attach_adapters", "set_adapter_ids"]


class NPAdapterLinear(nn.Module):
    """``base(x)`` plus each token's adapter (:func:`neuropress_amd.kernels.adapter_linear`).

    *ids*: which adapter each token or each sequence of x has, -1 for none; given with the call, or left on the module by :func:`set_adapter_ids`.  Without either the module is
    ``base``.  The adapters are no parameters: ``state_dict`` and moves leave them where they are; the projection's own entries lie under ``base.``.
    """

    def __init__(self, base: nn.Module, adapters: LowRankAdapters) -> None:
        super().__init__()
        for side in ("in_features", "out_features"):
            theirs, ours = getattr(base, side, None), getattr(adapters, side, None)
            if isinstance(theirs, int) and isinstance(ours, int) and theirs != ours:
                raise RuntimeError(f"NPAdapterLinear: the adapters have {side} of {ours}, the projection of {theirs}")
        self.base = base
        self.training = base.training  # without a word to what is inside it
        self.adapters = adapters
        self.ids: torch.Tensor | None = None

    def forward(self, x: torch.Tensor, ids: torch.Tensor | None = None) -> torch.Tensor:
        ids = self.ids if ids is None else ids
        y = self.base(x)
        return y if ids is None else adapter_linear(x, self.adapters, ids, y)

    def extra_repr(self) -> str:
        a = self.adapters
        return f"adapters={a.adapters}, rank={a.rank}, in_features={a.in_features}, out_features={a.out_features}"


def attach_adapters(model: nn.Module, adapters: dict[str, LowRankAdapters]) -> int:
    """Put an :class:`NPAdapterLinear` in the place of every module of *model* that *adapters* names; returns how many.  Names that *model* does not have, and adapters
    of other sizes than the layer's, are an error, and nothing is replaced."""
    places = []
    for name, those in adapters.items():
        parent_name, _, attr = name.rpartition(".")
        try:
            parent = model.get_submodule(parent_name) if parent_name else model
            base = parent.get_submodule(attr)
        except AttributeError:
            raise RuntimeError(f"attach_adapters: the model has no module {name!r}") from None
        if not attr:
            raise RuntimeError("attach_adapters: the model itself cannot be replaced: wrap it in an NPAdapterLinear")
        base = base.base if isinstance(base, NPAdapterLinear) else base
        try:
            places.append((parent, attr, NPAdapterLinear(base, those)))
        except RuntimeError as e:
            raise RuntimeError(f"attach_adapters: {name}: {e}") from None
    for parent, attr, layer in places:
        setattr(parent, attr, layer)
    return len(places)


def set_adapter_ids(model: nn.Module, ids: torch.Tensor | None) -> None:
    """Which adapter each token or sequence of the next calls has, for every :class:`NPAdapterLinear` of *model*; None: none of them."""
    for module in model.modules():
        if isinstance(module, NPAdapterLinear):
            module.ids = ids
