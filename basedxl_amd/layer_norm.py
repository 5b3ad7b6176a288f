"""Layer norm and residual add with layer norm on the GPU, with their gradients: what stands between the projections of a
transformer block (diffusers' ``BasicTransformerBlock``, part of the model that the reference wraps at basedxl/unet.py:65-87,
runs it in torch).  Kernels: csrc/cascmm_norm_kernel.h.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .cascaded_lowp_matmul import _DTYPES, _rows


def refuse_tangents(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Forward-mode differentiation (dual tensors) would lose its tangents here."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} is differentiable in reverse mode only")


def _check(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"layer_norm: x is on {x.device}; the operator only runs on an AMD GPU (there is no CPU fallback)")
    if x.dtype not in _DTYPES:
        raise TypeError(f"layer_norm: unsupported dtype {x.dtype}")
    if x.dim() < 1:
        raise ValueError("layer_norm: x needs at least one dimension")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"layer_norm: eps must be a number from 0 on, got {eps}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.device != x.device:
            raise ValueError(f"layer_norm: {name} is on {t.device} but x on {x.device}")
        if t.dim() != 1 or t.shape[0] != x.shape[-1]:
            raise ValueError(f"layer_norm: {name} must have shape ({x.shape[-1]},), got {tuple(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"layer_norm: {name} must be {x.dtype} or float32, got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"layer_norm: weight is {weight.dtype} but bias is {bias.dtype}")


def _check_residual(x: torch.Tensor, residual: torch.Tensor) -> None:
    if residual.device != x.device:
        raise ValueError(f"add_layer_norm: residual is on {residual.device} but x on {x.device}")
    if residual.dtype != x.dtype or residual.shape != x.shape:
        raise ValueError(f"add_layer_norm: residual must be like x, {tuple(x.shape)} {x.dtype}, got {tuple(residual.shape)} {residual.dtype}")


def _flat(t: torch.Tensor) -> torch.Tensor:
    """``t`` as rows of its last axis, a view where its strides allow one."""
    return _rows(t.reshape(t.shape[:-1].numel(), t.shape[-1]))


def _ld(t2: torch.Tensor) -> int:
    return t2.stride(0) if t2.shape[0] > 1 else t2.shape[1]


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _forward(x, residual, weight, bias, eps, keep_statistics):
    """(y, s, mean, rstd): s is x where there is no residual, the statistics None unless kept."""
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    s = x if residual is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    mean = rstd = None
    if keep_statistics:
        mean, rstd = torch.empty(2, rows, dtype=torch.float32, device=x.device)
    if rows == 0:
        return y, s, mean, rstd
    x2, r2 = _flat(x), None if residual is None else _flat(residual)
    weight, bias = None if weight is None else weight.contiguous(), None if bias is None else bias.contiguous()
    like = weight if weight is not None else bias if bias is not None else x
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().cascmm_layer_norm(
            x2.data_ptr(), _ptr(r2), _ptr(weight), _ptr(bias), y.data_ptr(), None if r2 is None else s.data_ptr(), _ptr(mean), _ptr(rstd),
            rows, cols, _ld(x2), 0 if r2 is None else _ld(r2), cols, cols, eps, _DTYPES[x.dtype], _DTYPES[like.dtype],
            torch.cuda.current_stream(x.device).cuda_stream), "cascmm_layer_norm")
    return y, s, mean, rstd


def _backward(dy, ds, s, weight, bias, mean, rstd, want_x, want_weight, want_bias):
    """(dx, dweight, dbias), each None where it is not wanted."""
    cols = s.shape[-1]
    rows = s.numel() // cols if cols else 0
    dx = torch.empty(s.shape, dtype=s.dtype, device=s.device) if want_x else None
    dweight = torch.empty_like(weight, memory_format=torch.contiguous_format) if want_weight else None
    dbias = torch.empty_like(bias, memory_format=torch.contiguous_format) if want_bias else None
    if cols == 0 or not (want_x or want_weight or want_bias):
        return dx, dweight, dbias
    dy2, s2, ds2 = _flat(dy), _flat(s), None if ds is None else _flat(ds)
    like = weight if weight is not None else bias if bias is not None else s
    weight = None if weight is None else weight.contiguous()
    l = _lib.lib()
    with torch.cuda.device(s.device):
        ws = None
        if want_weight or want_bias:   # (a temporary of the call, as any operator's: of a recorded call in the graph's own memory)
            ws = torch.empty(l.cascmm_layer_norm_workspace_bytes(rows, cols, _DTYPES[s.dtype]), dtype=torch.uint8, device=s.device)
        _lib.check(l.cascmm_layer_norm_backward(
            dy2.data_ptr(), _ptr(ds2), s2.data_ptr(), _ptr(weight), mean.data_ptr(), rstd.data_ptr(), _ptr(dx), _ptr(dweight), _ptr(dbias),
            rows, cols, _ld(dy2), 0 if ds2 is None else _ld(ds2), _ld(s2), cols, _DTYPES[s.dtype], _DTYPES[like.dtype],
            _ptr(ws), 0 if ws is None else ws.numel(), torch.cuda.current_stream(s.device).cuda_stream), "cascmm_layer_norm_backward")
    return dx, dweight, dbias


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, _, mean, rstd = _forward(x, None, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        want = ctx.needs_input_grad
        dx, dweight, dbias = _backward(dy, None, x, weight, bias, mean, rstd, want[0], want[1], want[2])
        return dx, dweight, dbias, None


class _AddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        y, s, mean, rstd = _forward(x, residual, weight, bias, eps, True)
        ctx.save_for_backward(s, weight, bias, mean, rstd)
        ctx.set_materialize_grads(False)
        return y, s

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, ds):
        s, weight, bias, mean, rstd = ctx.saved_tensors
        want = ctx.needs_input_grad
        if dy is None:      # (the norm's result was not used: the sum's gradient passes through)
            return ds if want[0] else None, ds if want[1] else None, None, None, None
        dx, dweight, dbias = _backward(dy, ds, s, weight, bias, mean, rstd, want[0] or want[1], want[2], want[3])
        return dx if want[0] else None, dx if want[1] else None, dweight, dbias, None


def _differentiated(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last axis, in one kernel; ``x`` fp32, fp16 or bf16 with any leading
    dimensions, ``weight`` / ``bias`` 1-D of the dtype of ``x`` or fp32 (None: ones, zeros).  Statistics and arithmetic are fp32, the
    result is rounded once.  Differentiable once in ``x``, ``weight`` and ``bias``; the sums over rows behind the last two are
    added in a fixed order, so the same call gives the same bits."""
    y = _lib.short_cut().layer_norm(x, weight, bias, eps)   # the ordinary eager call in one native function; None: it is decided below
    if y is not None:
        return y
    _check(x, weight, bias, eps)
    refuse_tangents("layer_norm", x, weight, bias)
    if _differentiated(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _forward(x, None, weight, bias, float(eps), False)[0]


def add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                   eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor]:
    """``s = x + residual; return layer_norm(s, weight, bias), s`` in one kernel: ``s`` is written but not read back.  The norm is of ``s``
    as it is returned, rounded to the tensors' dtype.  Differentiable like :func:`layer_norm`, through both results; ``x`` and
    ``residual`` get the same tensor as their gradient."""
    both = _lib.short_cut().add_layer_norm(x, residual, weight, bias, eps)
    if both is not None:
        return both
    _check(x, weight, bias, eps)
    _check_residual(x, residual)
    refuse_tangents("add_layer_norm", x, residual, weight, bias)
    if _differentiated(x, residual, weight, bias):
        return _AddLayerNorm.apply(x, residual, weight, bias, float(eps))
    y, s, _, _ = _forward(x, residual, weight, bias, float(eps), False)
    return y, s
