"""The module wrappers' GEMM as a ``torch.library`` custom op, so that a model holding them can be
traced by ``torch.compile`` (the reference compiles its UNet, basedxl/unet.py:76-78, and its Triton
kernel is traced natively; a ctypes call is opaque to the tracer).  The op has a shape-only ("fake")
implementation for tracing and runs the ordinary wrapper when executed.  The modules go through it
only while ``torch.compiler.is_compiling()``: in eager mode they call the wrapper directly, which
saves the dispatcher's per-call overhead.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .cascaded_lowp_matmul import PreparedWeight, cascaded_lowp_matmul, raw_is_faster
from .layer_norm import add_layer_norm, layer_norm
from .matmul_epilogue import cascaded_lowp_matmul_epilogue


@torch.library.custom_op("basedxl_amd::cascade_linear", mutates_args=(), device_types="cuda")
def cascade_linear(x: torch.Tensor, weight: torch.Tensor, slots: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                   lowp: str, terms: int, products: str, glu: bool, b_exp: Optional[torch.Tensor]) -> torch.Tensor:
    """``x @ weight (+ bias)`` through the cascade; with ``slots`` (the operand slots of a
    PreparedWeight of ``weight``) the prepared kernels run when they take ``x``.  ``glu``: the
    gated projection, ``slots`` required, result ``[..., weight.shape[1] // 2]``."""
    K, N = int(weight.shape[0]), int(weight.shape[1])
    if slots is not None:
        pw = PreparedWeight.from_slots(slots, K, N, weight.dtype, lowp, terms, glu, b_exp)
        x2 = x.reshape(-1, K)
        few_rows = raw_is_faster(x2.shape[0], K, N, x2.dtype, lowp, terms, products)
        if glu or (not few_rows and pw.usable_with(x2 if x2.stride(-1) == 1 else x2.contiguous(), products)):
            return cascaded_lowp_matmul(x, pw, bias=bias, products=products)
    return cascaded_lowp_matmul(x, weight, bias=bias, lowp=lowp, terms=terms, products=products, b_exp=b_exp)


@cascade_linear.register_fake
def _(x, weight, slots, bias, lowp, terms, products, glu, b_exp):
    n = weight.shape[1] // 2 if glu else weight.shape[1]
    return x.new_empty((*x.shape[:-1], n))


@torch.library.custom_op("basedxl_amd::cascade_linear_epilogue", mutates_args=(), device_types="cuda")
def cascade_linear_epilogue(x: torch.Tensor, weight: torch.Tensor, slots: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                            residual: Optional[torch.Tensor], activation: Optional[str], lowp: str, terms: int, products: str,
                            b_exp: Optional[torch.Tensor]) -> torch.Tensor:
    """``activation(x @ weight + bias) + residual`` through the cascade, ``slots`` as for :func:`cascade_linear`."""
    K, N = int(weight.shape[0]), int(weight.shape[1])
    if slots is not None and x.dtype == weight.dtype:
        pw = PreparedWeight.from_slots(slots, K, N, weight.dtype, lowp, terms, False, b_exp)
        x2 = x.reshape(-1, K)
        few_rows = raw_is_faster(x2.shape[0], K, N, x2.dtype, lowp, terms, products)
        if not few_rows and pw.usable_with(x2 if x2.stride(-1) == 1 else x2.contiguous(), products):
            return cascaded_lowp_matmul_epilogue(x, pw, bias=bias, activation=activation, residual=residual, products=products)
    return cascaded_lowp_matmul_epilogue(x, weight, bias=bias, activation=activation, residual=residual, lowp=lowp, terms=terms, products=products, b_exp=b_exp)


@cascade_linear_epilogue.register_fake
def _(x, weight, slots, bias, residual, activation, lowp, terms, products, b_exp):
    return x.new_empty((*x.shape[:-1], weight.shape[1]))


@torch.library.custom_op("basedxl_amd::layer_norm", mutates_args=(), device_types="cuda")
def layer_norm_op(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float) -> torch.Tensor:
    return layer_norm(x, weight, bias, eps=eps)


@layer_norm_op.register_fake
def _(x, weight, bias, eps):
    return x.new_empty(x.shape)


@torch.library.custom_op("basedxl_amd::add_layer_norm", mutates_args=(), device_types="cuda")
def add_layer_norm_op(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor],
                      eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    return add_layer_norm(x, residual, weight, bias, eps=eps)


@add_layer_norm_op.register_fake
def _(x, residual, weight, bias, eps):
    return x.new_empty(x.shape), x.new_empty(x.shape)
