"""The layer norms of a module tree on this package's kernels (the reference leaves them to torch; they are part of the model it
wraps at basedxl/unet.py:65-87)."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from ..layer_norm import add_layer_norm, layer_norm


class BasedXLLayerNorm(nn.Module):
    """Wraps an ``nn.LayerNorm`` over the last axis, whose parameters it keeps (the same objects: they train as before).
    ``forward(x)`` is the norm; ``forward(x, residual)`` returns the norm of ``x + residual`` and the sum itself, in one kernel.
    Traced by torch.compile it is one opaque op without gradients."""

    def __init__(self, submodule: nn.LayerNorm):
        super().__init__()
        if len(submodule.normalized_shape) != 1:
            raise ValueError(f"only norms over the last axis have a kernel, got normalized_shape {tuple(submodule.normalized_shape)}")
        self.normalized_shape, self.eps = submodule.normalized_shape, submodule.eps
        self.weight, self.bias = submodule.weight, submodule.bias

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        if x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"the norm is over {self.normalized_shape[0]} columns, got {x.shape[-1]}")
        if torch.compiler.is_compiling():
            # traced by torch.compile: one opaque op
            from ..compiled import add_layer_norm_op, layer_norm_op
            if residual is None:
                return layer_norm_op(x, self.weight, self.bias, self.eps)
            return add_layer_norm_op(x, residual, self.weight, self.bias, self.eps)
        if residual is None:
            return layer_norm(x, self.weight, self.bias, eps=self.eps)
        return add_layer_norm(x, residual, self.weight, self.bias, eps=self.eps)


def _hooked(module: nn.Module) -> bool:
    return any(getattr(module, hooks, None) for hooks in ("_forward_pre_hooks", "_forward_hooks", "_backward_pre_hooks", "_backward_hooks"))


def patch_layer_norms(model: nn.Module) -> nn.Module:
    """Replace every ``nn.LayerNorm`` child over the last axis with :class:`BasedXLLayerNorm`.  Subclasses, which may compute something else, stay, and so
    do norms with hooks, which would see other calls (a block may hand a norm the residual add in front of it)."""
    for module in list(model.modules()):
        for name, child in list(module.named_children()):
            if type(child) is nn.LayerNorm and len(child.normalized_shape) == 1 and not _hooked(child):
                setattr(module, name, BasedXLLayerNorm(child))
    return model
