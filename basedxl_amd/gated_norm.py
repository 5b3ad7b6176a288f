"""The norms on both sides of a block's residual add in one kernel, with the add, its gate and the residual's scale, and their gradients: what :func:`add_layer_norm` is
for a block that ends in a norm of its own, a layer scale or a gate that its conditioning gives.  (The model that the reference wraps at
basedxl/unet.py:65-87 runs such steps in torch.)  Kernels: csrc/cascmm_gated_kernel.h.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .cascaded_lowp_matmul import _DTYPES
from .layer_norm import _flat, _ld, _ptr, refuse_tangents

_NORMS = {"layer": 0, "rms": 1}


def _parameter(t: Optional[torch.Tensor], name: str, x: torch.Tensor, grouped: bool) -> Optional[torch.Tensor]:
    """``t`` as [cols], or, where groups of rows (the first axis of ``x``) may have one each, [groups, cols]."""
    if t is None:
        return None
    cols = x.shape[-1]
    if t.device != x.device:
        raise ValueError(f"gated_add_norm: {name} is on {t.device} but x on {x.device}")
    if t.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"gated_add_norm: {name} must be {x.dtype} or float32, got {t.dtype}")
    if t.dim() >= 1 and t.shape[-1] == cols:
        if t.dim() == 1:
            return t
        if t.dim() <= x.dim() and t.numel() == cols:
            return t.reshape(cols)
        if grouped and t.dim() == x.dim() and t.shape[0] == x.shape[0] and t.shape[1:-1].numel() == 1:
            return t.reshape(t.shape[0], cols)
    shapes = f"({cols},)" + (f" or {(x.shape[0],) + (1,) * (x.dim() - 2) + (cols,)}" if grouped and x.dim() > 1 else "")
    raise ValueError(f"gated_add_norm: {name} must have shape {shapes}, got {tuple(t.shape)}")


def _leading(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None or t.dim() == 1 else t.stride(0)


def _rows(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """``t`` itself where the kernels can read its rows as they lie, at any distance from each other."""
    if t is None or (t.shape[-1] == 1 or t.stride(-1) == 1) and (t.dim() == 1 or t.stride(0) >= t.shape[1]):
        return t
    return t.contiguous()


def _arguments(x2, r2, s2, parameters, rows, cols, group_rows, how, weight_dtype):
    weight, bias, gate, scale, post_weight, post_bias = parameters
    post, norm, eps, alpha = how
    a = _lib.GatedNorm()
    a.x, a.residual, a.sum = _ptr(x2), _ptr(r2), s2.data_ptr()
    a.weight, a.bias, a.gate, a.scale, a.post_weight, a.post_bias = map(_ptr, parameters)
    a.rows, a.cols, a.group_rows = rows, cols, group_rows
    a.ldx, a.ldr, a.lds = 0 if x2 is None else _ld(x2), 0 if r2 is None else _ld(r2), _ld(s2)
    a.gate_ld, a.scale_ld, a.weight_ld, a.bias_ld = _leading(gate), _leading(scale), _leading(weight), _leading(bias)
    a.residual_scale, a.eps, a.norm, a.post, a.dtype, a.weight_dtype = alpha, eps, norm, int(post), _DTYPES[s2.dtype], _DTYPES[weight_dtype]
    return a


def _sizes(x: torch.Tensor, parameters) -> Tuple[int, int, int]:
    """rows, columns, and the rows that share a parameter's row."""
    cols = x.shape[-1]
    rows = x.shape[:-1].numel()
    grouped = any(t is not None and t.dim() == 2 for t in parameters)
    return rows, cols, x.shape[1:-1].numel() if grouped else rows


def _weight_dtype(x, parameters) -> torch.dtype:
    return next((t.dtype for t in parameters if t is not None), x.dtype)


def _forward(x, residual, parameters, how, keep):
    """(y, s, statistics or None)."""
    y, s = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for _ in range(2))
    rows, cols, group_rows = _sizes(x, parameters)
    stats = torch.empty(4, rows, dtype=torch.float32, device=x.device) if keep else None
    if rows == 0 or cols == 0:
        return y, s, stats
    x2, r2, parameters = _flat(x), _flat(residual), [_rows(t) for t in parameters]
    with torch.cuda.device(x.device):
        a = _arguments(x2, r2, s.view(rows, cols), parameters, rows, cols, group_rows, how, _weight_dtype(x, parameters))
        a.y, a.ldy, a.stats = y.data_ptr(), cols, _ptr(stats)
        _lib.check(_lib.lib().cascmm_gated_norm_forward(ctypes.byref(a), torch.cuda.current_stream(x.device).cuda_stream), "cascmm_gated_norm_forward")
    return y, s, stats


class _GatedAddNorm(torch.autograd.Function):
    """``weight`` to ``post_bias``: [cols] or [groups, cols], all of one dtype."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, gate, scale, post_weight, post_bias, post, norm, eps, alpha):
        parameters, how = (weight, bias, gate, scale, post_weight, post_bias), (post, norm, eps, alpha)
        y, s, stats = _forward(x, residual, parameters, how, True)
        ctx.save_for_backward(x if post or gate is not None else None, None if scale is None else residual, s, stats, *parameters)
        ctx.set_materialize_grads(False)
        ctx.how = how
        return y, s

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds):
        x, residual, s, stats, *parameters = ctx.saved_tensors
        want, (post, _, _, alpha) = ctx.needs_input_grad[:8], ctx.how
        none = (None,) * 12
        if dy is None and ds is None:
            return none
        dev, dtype = s.device, s.dtype
        if dy is None:
            dy = torch.zeros_like(s)
        rows, cols, group_rows = _sizes(s, parameters)
        new = lambda: torch.empty(s.shape, dtype=dtype, device=dev)   # noqa: E731
        # (neither gate, scale nor norm in front of the sum: its gradient is that of both)
        same = not post and parameters[2] is None and parameters[3] is None and alpha == 1.0
        dx = new() if want[0] and not same else None
        dr = new() if want[1] or (want[0] and same) else None
        fresh = torch.empty_like if rows > 0 else torch.zeros_like
        grads = [fresh(t, memory_format=torch.contiguous_format) if w else None for t, w in zip(parameters, want[2:])]
        if rows > 0 and cols > 0:
            parameters = [_rows(t) for t in parameters]
            l = _lib.lib()
            with torch.cuda.device(dev):
                # (names of their own until the launch: a copy that is given back before the workspace is allocated is where the workspace may come to lie)
                dy2, s2, (ds2, x2, r2) = _flat(dy), _flat(s), (None if t is None else _flat(t) for t in (ds, x, residual))
                a = _arguments(x2, r2, s2, parameters, rows, cols, group_rows, ctx.how, _weight_dtype(s, parameters))
                a.dy, a.ds, a.stats, a.dx, a.dresidual = dy2.data_ptr(), _ptr(ds2), stats.data_ptr(), _ptr(dx), _ptr(dr)
                a.dweight, a.dbias, a.dgate, a.dscale, a.dpost_weight, a.dpost_bias = map(_ptr, grads)
                a.lddy, a.ldds, a.lddx, a.lddr = _ld(dy2), 0 if ds2 is None else _ld(ds2), cols, cols
                ws = torch.empty(l.cascmm_gated_norm_backward_bytes(ctypes.byref(a)), dtype=torch.uint8, device=dev)   # (a temporary of the call)
                _lib.check(l.cascmm_gated_norm_backward(ctypes.byref(a), ws.data_ptr(), ws.numel(), torch.cuda.current_stream(dev).cuda_stream),
                           "cascmm_gated_norm_backward")
        return (dr if same and want[0] else dx, dr if want[1] else None, *grads, None, None, None, None)


def gated_add_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                   gate: Optional[torch.Tensor] = None, residual_scale: Union[float, torch.Tensor] = 1.0, post_norm: bool = False,
                   post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None, norm: str = "layer",
                   eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """``s = residual_scale * residual + gate * p; return norm(s) * weight + bias, s`` in one kernel, with ``p = norm(x) * post_weight + post_bias`` where ``post_norm``
    is set, else ``x``: a block's result ``x``, its own norm, its gate, the residual stream and the next block's norm.  ``norm``: "layer" (``(v - mean) / sqrt(var + eps)``)
    or "rms" (``v / sqrt(mean(v * v) + eps)``), over the last axis, for both.

    ``x`` and ``residual``: fp32, fp16 or bf16, alike, with any leading dimensions.  ``gate``, ``residual_scale`` (a number or a tensor), ``weight`` and ``bias`` are
    [C], or one row for each entry of the first axis of ``x``, ``(B, 1, .., C)``, as a conditioning gives them to its samples (made for many rows to a sample: the backward
    pass holds three to five fp32 rows of sums for each while it runs, if any of their gradients is wanted); gate and scale may be scalars too; ``post_weight`` and ``post_bias`` are [C].  All of the dtype of ``x`` or fp32; None: ones, for a bias
    zeros.  The norm is of ``s`` as it is returned, rounded to the tensors' dtype; statistics and arithmetic are fp32, each result is rounded once.
    Differentiable once in all tensors, through both results; sums over rows are added in a fixed order, so the same call gives the same bits."""
    # the ordinary eager call in one native function; None: whatever is not ordinary about it is decided below
    both = _lib.short_cut().gated_add_norm(x, residual, weight, bias, gate, residual_scale, post_weight, post_bias, post_norm, _NORMS.get(norm, -1) if type(norm) is str else -1, eps)
    if both is not None:
        return both
    if not x.is_cuda:
        raise RuntimeError(f"gated_add_norm: x is on {x.device}; the operator only runs on an AMD GPU (there is no CPU fallback)")
    if x.dtype not in _DTYPES:
        raise TypeError(f"gated_add_norm: unsupported dtype {x.dtype}")
    if x.dim() < 1:
        raise ValueError("gated_add_norm: x needs at least one dimension")
    if residual.device != x.device or residual.dtype != x.dtype or residual.shape != x.shape:
        raise ValueError(f"gated_add_norm: residual must be like x, {tuple(x.shape)} {x.dtype} on {x.device}, got {tuple(residual.shape)} {residual.dtype} on {residual.device}")
    if norm not in _NORMS:
        raise ValueError(f"gated_add_norm: norm must be one of {list(_NORMS)}, got {norm!r}")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"gated_add_norm: eps must be a number from 0 on, got {eps}")
    if not post_norm and (post_weight is not None or post_bias is not None):
        raise ValueError("gated_add_norm: post_weight and post_bias belong to post_norm=True")
    cols, scale, alpha = x.shape[-1], None, 1.0
    if isinstance(residual_scale, torch.Tensor):
        scale = residual_scale.expand(cols) if residual_scale.dim() == 0 else residual_scale
    else:
        alpha = float(residual_scale)
        if not math.isfinite(alpha):
            raise ValueError(f"gated_add_norm: residual_scale must be finite, got {residual_scale}")
    if gate is not None and gate.dim() == 0:
        gate = gate.expand(cols)
    named = (("weight", weight, True), ("bias", bias, True), ("gate", gate, True), ("residual_scale", scale, True), ("post_weight", post_weight, False), ("post_bias", post_bias, False))
    parameters = [_parameter(t, name, x, grouped) for name, t, grouped in named]
    if len({t.dtype for t in parameters if t is not None}) > 1:
        parameters = [None if t is None else t.float() for t in parameters]
    refuse_tangents("gated_add_norm", x, residual, *parameters)
    how = (bool(post_norm), _NORMS[norm], float(eps), alpha)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual, *parameters)):
        return _GatedAddNorm.apply(x, residual, *parameters, *how)
    y, s, _ = _forward(x, residual, parameters, how, False)
    return y, s
