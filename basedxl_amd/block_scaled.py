"""A product in 8-bit floating point with a power of two as the scale of every block of 128, and its gradients, which are products of the same kind.

The cascades of :func:`cascaded_lowp_matmul` hold a tensor under one scale and make up for the format's three bits with more terms; here every block has
the scale that its own elements ask for and there is one term: half the bytes of a 16-bit product and twice its rate, at the format's precision.
(The reference's counterpart of the layer is basedxl/modules/lowp_linear.py:7-20.)  Kernels: csrc/cascmm_block_kernel.h.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .cascaded_lowp_matmul import _DTYPES, _check_bias, _rows
from .layer_norm import _flat, refuse_tangents

_MOST_K = 2 ** 22


def _check_operand(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"block_scaled_matmul: {name} is on {t.device}; the operator only runs on an AMD GPU (there is no CPU fallback)")
    if t.dtype not in _DTYPES:
        raise TypeError(f"block_scaled_matmul: unsupported dtype {t.dtype} of {name}")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _ld(t2: torch.Tensor) -> int:
    return t2.stride(0) if t2.shape[0] > 1 else t2.shape[1]


Held = Tuple[torch.Tensor, torch.Tensor]   # values [rows, k padded], scales [blocks / 4, rows, 4], as bytes


def _space(rows: int, k: int, device: torch.device) -> Held:
    blocks = -(-k // 128)
    return (torch.empty((rows, blocks * 128), dtype=torch.uint8, device=device), torch.empty((-(-blocks // 4), rows, 4), dtype=torch.uint8, device=device))


def _round(x2: torch.Tensor, square: bool, along: bool, across: bool, sums: bool = False):
    """(held, held transposed, sums over rows) of the rows ``x2``, each None unless wanted: blocks along its rows, across them, or 128 x 128 (``square``)."""
    rows, cols = x2.shape
    dev, l = x2.device, _lib.lib()
    with torch.cuda.device(dev):
        q = _space(rows, cols, dev) if along else None
        qt = _space(cols, rows, dev) if across else None
        total = torch.empty(cols, dtype=x2.dtype, device=dev) if sums else None
        ws = torch.empty(l.cascmm_block_round_workspace_bytes(rows, cols), dtype=torch.uint8, device=dev) if sums else None   # (a temporary of the call)
        _lib.check(l.cascmm_block_round(x2.data_ptr(), rows, cols, _ld(x2), _DTYPES[x2.dtype], int(square), _ptr(q and q[0]), _ptr(q and q[1]), _ptr(qt and qt[0]),
                                        _ptr(qt and qt[1]), _ptr(total), _ptr(ws), 0 if ws is None else ws.numel(), torch.cuda.current_stream(dev).cuda_stream),
                   "cascmm_block_round")
    return q, qt, total


def _round_weight(b: torch.Tensor, forward: bool, backward: bool) -> Tuple[Optional[Held], Optional[Held]]:
    """A right operand [K, N] as the forward product ([N, K padded]) and the gradient of the left one ([K, N padded]) want it, read in the order it lies in."""
    if b.stride(0) == 1 and b.stride(1) >= max(b.shape[0], 1) and b.stride(1) != 1:
        q, qt, _ = _round(b.t(), True, forward, backward)
        return q, qt
    q, qt, _ = _round(_rows(b), True, backward, forward)
    return qt, q


def _multiply(a: Held, b: Held, out2: torch.Tensor, bias: Optional[torch.Tensor], K: int) -> None:
    (M, N), dev = out2.shape, out2.device
    with torch.cuda.device(dev):
        _lib.check(_lib.lib().cascmm_block_gemm(a[0].data_ptr(), a[1].data_ptr(), b[0].data_ptr(), b[1].data_ptr(), out2.data_ptr(), _ptr(bias), M, N, K, N, _DTYPES[out2.dtype],
                                                torch.cuda.current_stream(dev).cuda_stream), "cascmm_block_gemm")


class BlockScaledWeight:
    """A constant right operand ``w`` ([K, N], in either order of its elements) rounded once to 8 bits with a scale for each 128 x 128, as
    :func:`block_scaled_matmul` rounds a tensor in every call: K N bytes and a 128th of that."""

    def __init__(self, w: torch.Tensor):
        _check_operand(w, "w")
        if w.dim() != 2:
            raise ValueError(f"BlockScaledWeight needs a 2-D tensor, got {tuple(w.shape)}")
        self.K, self.N = int(w.shape[0]), int(w.shape[1])
        self.shape, self.dtype, self.device = (self.K, self.N), w.dtype, w.device
        if self.K > _MOST_K:
            raise ValueError(f"BlockScaledWeight: K is at most {_MOST_K}, got {self.K}")
        with torch.no_grad():
            held = _round_weight(w.detach(), True, False)[0]
        #: uint8 [N, K rounded up to 128] (e4m3) and [blocks / 4, N, 4] (E8M0: 2^(byte - 127)), blocks of 128 along K
        self.values, self.scales = held

    def dequantized(self) -> torch.Tensor:
        """The fp32 [K, N] values that the product uses (for inspection)."""
        scales = self.scales.permute(1, 0, 2).reshape(self.N, -1)[:, :self.values.shape[1] // 128].int()
        scales = torch.ldexp(torch.ones_like(scales, dtype=torch.float64), scales - 127)
        wide = self.values.view(torch.float8_e4m3fn).double() * scales.repeat_interleave(128, 1)
        return wide[:, :self.K].t().float()


class _BlockScaled(torch.autograd.Function):
    @staticmethod
    def forward(ctx, a, b, bias):
        want_a, want_b, _ = ctx.needs_input_grad
        a2, (K, N) = _flat(a), b.shape
        left, left_t, _ = _round(a2, False, True, want_b)
        right, right_t = _round_weight(b, True, want_a)
        out = torch.empty(*a.shape[:-1], N, dtype=a.dtype, device=a.device)
        _multiply(left, right, out.view(a2.shape[0], N), bias, K)
        # (what the way back multiplies is in 8 bits already: neither a nor b is kept)
        ctx.save_for_backward(*(left_t or (None, None)), *(right_t or (None, None)))
        ctx.of = (a.shape, K, N)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        at, at_scales, bt, bt_scales = ctx.saved_tensors
        want_a, want_b, want_bias = ctx.needs_input_grad
        shape, K, N = ctx.of
        dy2 = _flat(dy)
        M = dy2.shape[0]
        rows, columns, dbias = _round(dy2, False, want_a, want_b, want_bias)
        da = db = None
        if want_a:
            da = torch.empty(shape, dtype=dy.dtype, device=dy.device)
            _multiply(rows, (bt, bt_scales), da.view(M, K), None, N)
        if want_b:
            db = torch.empty(K, N, dtype=dy.dtype, device=dy.device)
            _multiply((at, at_scales), columns, db, None, M)
        return da, db, dbias


def block_scaled_matmul(a: torch.Tensor, b, *, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``a @ b (+ bias)`` of operands rounded to 8-bit floating point (e4m3): ``a`` [..., K] fp32, fp16 or bf16, ``b`` [K, N] of the same type, in either
    order of its elements (a Linear layer's ``weight.t()``), or a :class:`BlockScaledWeight`.  Each 128 consecutive k of a row of ``a`` and each 128 x 128 elements of ``b``
    have as their scale the smallest power of two, from 2^-127 on, with max|x| <= 448 * 2^e over the finite elements; infinities and NaN become NaN.  Sums are fp32, the
    result (of the dtype of ``a``) is rounded once.  16-bit results come from the 8-bit matrix instruction, which cuts products at about 2^-15 of the largest of their neighbours: of ordinary
    data 1.5e-5 of a result's usual size (rms; less than its rounding, but results far below the usual size show it), and at worst 2^-10 of the largest product of every sixteen
    neighbouring k, to which alone what large products that cancel leave is good.
    fp32 results have products and sums to fp32's accuracy (at about half the rate, 1272 against 2798 TFLOP/s at 8192 x 8192 x 8192; rounded elements below 2^-126 count as zeros there, and
    those that round to 2^128, from 1.9375 * 2^127 on, as infinite).  K and the rows of ``a`` up to 2^22.

    Differentiable once in ``a``, ``b`` (a tensor: a held weight is a constant that no gradient passes through) and ``bias``, by products of the same kind, with the
    rounding passed over: ``dy`` in blocks of 128 along N times the same rounded ``b``; ``a`` and ``dy`` both in blocks of 128 rows; ``dbias`` from ``dy`` itself."""
    held = isinstance(b, BlockScaledWeight)
    # the ordinary eager call in one native function; None: whatever is not ordinary about it is decided below
    if not held:
        y = _lib.short_cut().block_scaled(a, b, None, 0, 0, 0, bias)
    else:
        y = _lib.short_cut().block_scaled(a, b.values, b.scales, b.K, b.N, _DTYPES[b.dtype], bias)
    if y is not None:
        return y
    _check_operand(a, "a")
    if a.dim() < 1:
        raise ValueError("block_scaled_matmul: a needs at least one dimension")
    if not held:
        _check_operand(b, "b")
        if b.dim() != 2:
            raise ValueError(f"block_scaled_matmul: b must be 2-D, got {tuple(b.shape)}")
    if b.device != a.device:
        raise ValueError(f"block_scaled_matmul: b is on {b.device} but a on {a.device}")
    if b.dtype != a.dtype:
        raise TypeError(f"block_scaled_matmul: a is {a.dtype} but b is {b.dtype}")
    K, N = b.shape
    if a.shape[-1] != K:
        raise ValueError(f"block_scaled_matmul: a has {a.shape[-1]} columns but b {K} rows")
    if K > _MOST_K:
        raise ValueError(f"block_scaled_matmul: K is at most {_MOST_K}, got {K}")
    bias = _check_bias(bias, a, N)
    operands = [t for t in (a, None if held else b, bias) if t is not None]
    refuse_tangents("block_scaled_matmul", *operands)
    if torch.is_grad_enabled() and any(t.requires_grad for t in operands):
        if held:
            raise RuntimeError("block_scaled_matmul: a gradient needs the weight itself, not a BlockScaledWeight")
        if a.shape[:-1].numel() > _MOST_K or N > _MOST_K:
            raise ValueError(f"block_scaled_matmul: with gradients, rows of a and columns of b are at most {_MOST_K}")
        return _BlockScaled.apply(a, b, bias)
    a2 = _flat(a)
    out = torch.empty(*a.shape[:-1], N, dtype=a.dtype, device=a.device)
    if out.numel() == 0:
        return out
    (M, _), dev, l = a2.shape, a2.device, _lib.lib()
    right = (b.values, b.scales) if held else _round_weight(b, True, False)[0]
    with torch.cuda.device(dev):
        need = l.cascmm_block_linear_workspace_bytes(M, K, _DTYPES[a.dtype])
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None      # (a temporary of the call)
        _lib.check(l.cascmm_block_linear(a2.data_ptr(), right[0].data_ptr(), right[1].data_ptr(), out.data_ptr(), _ptr(bias), M, N, K, _ld(a2), N, _DTYPES[a.dtype], _ptr(ws), need,
                                         torch.cuda.current_stream(dev).cuda_stream), "cascmm_block_linear")
    return out
