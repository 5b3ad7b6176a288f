"""Gradients that pass through modules whose weights are constants (the reference's modules, basedxl/modules/lowp_linear.py:11-20, cut them:
its kernel is no autograd function)."""
from __future__ import annotations

from typing import Callable

import torch
from torch.autograd.function import once_differentiable


class _ConstantWeights(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, module):
        ctx.module = module
        ctx.save_for_backward(x if module.gradient_reads_input else None, *module.constants())   # (constants: so that torch notices if they are written to)
        return module.forward(x)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return ctx.module.input_gradient(dy, ctx.saved_tensors[0]), None


def with_gradient(module: torch.nn.Module, x: torch.Tensor) -> torch.Tensor:
    """``module.forward(x)`` as it is without gradients, kernel for kernel, with ``module.input_gradient(dy, x)`` as its way back."""
    return _ConstantWeights.apply(x, module)


def gradient_of(function: Callable[[torch.Tensor], torch.Tensor], x: torch.Tensor, dy: torch.Tensor) -> torch.Tensor:
    """The gradient of ``function`` at ``x``, computed once more: nothing between was kept."""
    with torch.enable_grad():
        leaf = x.detach().requires_grad_()
        y = function(leaf)
        return torch.autograd.grad(y, leaf, dy.to(y.dtype))[0]
