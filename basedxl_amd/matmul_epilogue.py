"""A product with what follows it in a Linear layer, ``activation(a @ b + bias) + residual``, and its gradients.

The reference runs the layer (basedxl/modules/lowp_linear.py:15-20) and what its model does with the result (a transformer
block's residual adds, an embedding's SiLU) as separate kernels.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .cascaded_lowp_matmul import (_DTYPES, PreparedWeight, _activation_exps, _check_bias, _check_device_tensor, _rows, _workspace, _workspace_bytes,
                                   cascaded_lowp_matmul, default_cascade)
from .layer_norm import refuse_tangents


def _ld(t2: torch.Tensor) -> int:
    return t2.stride(0) if t2.shape[0] > 1 else max(t2.shape[1], 1)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _overlap(p: torch.Tensor, q: torch.Tensor) -> bool:
    """Whether two tensors may share an element: their memory does, and they are not columns of their own of the same rows."""
    if p.numel() == 0 or q.numel() == 0 or p.device != q.device:
        return False
    ends = [t.data_ptr() + t.element_size() * (1 + sum((n - 1) * st for n, st in zip(t.shape, t.stride()))) for t in (p, q)]
    if p.data_ptr() >= ends[1] or q.data_ptr() >= ends[0]:
        return False
    if p.dim() == q.dim() == 2 and min(p.shape[0], q.shape[0]) > 1 and p.stride() == q.stride() and p.stride(1) == 1 and p.element_size() == q.element_size():
        apart = (q.data_ptr() - p.data_ptr()) % (p.stride(0) * p.element_size())
        if apart % p.element_size() == 0:
            first = apart // p.element_size()
            return not (first >= p.shape[1] and first + q.shape[1] <= p.stride(0))
    return True


_COPIES_END = 2 ** 31 - 1     # (the library's copies of operands stay below 2 GiB)


def _off_dwords(t2: torch.Tensor, unit: int) -> bool:
    """16-bit rows that start between dwords and whose length, a multiple of ``unit``, would not have the library count a copy of them anyway."""
    return t2.element_size() == 2 and t2.shape[1] % unit == 0 and (t2.data_ptr() % 4 != 0 or (t2.shape[0] > 1 and t2.stride(0) % 2 != 0))


def _copied_bytes(a2: torch.Tensor, b: Optional[torch.Tensor]) -> int:
    """What the library copies of 16-bit operands off dwords: cascmm_workspace_bytes, which sees no addresses, does not count it, and without room for it the
    kernels that read element by element would run, or not, as the stream's workspace has grown."""
    (M, K), need = a2.shape, 0
    if _off_dwords(a2, 8):
        need += M * (-(-2 * K // 128) * 128) + 256
    if b is not None and _off_dwords(b, 2):
        need += -(-K // 32) * 64 * b.shape[1] + 256
    return need


def _kernel_rows(t2: torch.Tensor, copy: bool) -> torch.Tensor:
    """``t2``, or a copy: if ``copy``, and of rows 2^21 16-bit (2^20 fp32) elements apart and more, which the offsets of the kernels do not span."""
    far = t2.shape[0] > 1 and t2.stride(0) != t2.shape[1] and t2.stride(0) * t2.element_size() * 512 >= 2 ** 31 - 1
    return t2.clone(memory_format=torch.contiguous_format) if copy or far else t2


def _residual_rows(residual: torch.Tensor, M: int, N: int) -> Tuple[torch.Tensor, int]:
    """The residual (of the result's shape, expanded perhaps) as rows and their distance; 0: the same row for all."""
    if M > 1 and all(st == 0 or n == 1 for n, st in zip(residual.shape[:-1], residual.stride()[:-1])):
        row = residual[(0,) * (residual.dim() - 1)]
        return (row if row.stride(0) == 1 or N == 1 else row.contiguous()), 0
    r2 = _rows(residual.reshape(M, N))
    return r2, _ld(r2)


def _product(a2, b, bias, residual, preact, out2, activation, lowp, terms, products, b_exp):
    """One cascmm_gemm_epilogue: everything checked, ``a2`` [M, K] rows, ``residual`` of the shape of the result or None."""
    prepared = isinstance(b, PreparedWeight)
    M, K = a2.shape
    N = b.N if prepared else b.shape[1]
    if M == 0 or N == 0:
        return
    if a2.element_size() == 2 or prepared:
        a2 = _kernel_rows(a2, _copied_bytes(a2, None) > _COPIES_END)
    if not prepared and _off_dwords(b, 2) and _copied_bytes(a2, b) - _copied_bytes(a2, None) > _COPIES_END:
        b = b.clone()
    dt, fmt, prod = _DTYPES[a2.dtype], _lib.FMT_BY_NAME[lowp], _lib.PROD_BY_NAME[products]
    dev, l = a2.device, _lib.lib()
    with torch.cuda.device(dev):
        stream = torch.cuda.current_stream(dev).cuda_stream
        r2, ldr = (None, 0) if residual is None else _residual_rows(residual, M, N)
        ws = _workspace(dev, stream, _workspace_bytes(M, N, K, dt, fmt, terms, prod) + _copied_bytes(a2, None if prepared else b))
        exps = None
        if fmt == _lib.FMT_FP8:
            exps = torch.empty(2, dtype=torch.int32, device=dev)
            kept = b.exp if prepared else b_exp
            _activation_exps(a2, _ld(a2), kept, exps.data_ptr(), stream)
            if kept is None:
                _activation_exps(b, _ld(b), None, exps.data_ptr() + 4, stream)
        _lib.check(l.cascmm_gemm_epilogue(
            a2.data_ptr(), b.slots.data_ptr() if prepared else b.data_ptr(), 1 if prepared else 0, out2.data_ptr(), _ptr(bias), _ptr(r2), _ptr(preact), M, N, K,
            _ld(a2), N if prepared else _ld(b), _ld(out2), ldr, N, dt, fmt, terms, prod, _lib.ACT_BY_NAME[activation], _ptr(exps), _ptr(ws),
            0 if ws is None else ws.numel(), stream), "cascmm_gemm_epilogue")


def _flat(t: torch.Tensor) -> torch.Tensor:
    """``t`` as rows of its last axis, a view where its strides allow one."""
    return _rows(t.reshape(t.shape[:-1].numel(), t.shape[-1]))


class _EpilogueProduct(torch.autograd.Function):
    """Tensors only: ``a`` [..., K], ``b`` [K, N], ``residual`` of the result's shape."""

    @staticmethod
    def forward(ctx, a, b, bias, residual, activation, lowp, terms, products, b_exp):
        K, N = b.shape
        a2 = _flat(a)
        out = torch.empty(*a.shape[:-1], N, dtype=a.dtype, device=a.device)
        preact = torch.empty(a2.shape[0], N, dtype=a.dtype, device=a.device) if activation is not None else None
        _product(a2, b, bias, residual, preact, out.view(a2.shape[0], N), activation, lowp, terms, products, b_exp)
        ctx.save_for_backward(a, b, preact)
        ctx.how = (activation, lowp, terms, products, b_exp)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        a, b, preact = ctx.saved_tensors
        activation, lowp, terms, products, _ = ctx.how
        want_a, want_b, want_bias, want_residual = ctx.needs_input_grad[:4]
        K, N = b.shape
        dev, dt = a.device, _DTYPES[a.dtype]
        da = db = None
        with torch.cuda.device(dev):
            dy2 = _flat(dy)
            M = dy2.shape[0]
            # dz, dbias and the products' other operands in one launch
            a2, slope = _flat(a), activation is not None and (want_a or want_b)
            new = lambda *shape: torch.empty(shape, dtype=a.dtype, device=dev)   # noqa: E731
            dz, dbias = new(M, N) if slope else dy2, new(N) if want_bias else None
            at, bt = new(K, M) if want_b else None, new(N, K) if want_a else None
            l, ws = _lib.lib(), None
            if want_bias:
                ws = torch.empty(l.cascmm_epilogue_workspace_bytes(M, N, dt), dtype=torch.uint8, device=dev)
            _lib.check(l.cascmm_epilogue_backward_operands(
                dy2.data_ptr(), _ptr(preact), dz.data_ptr() if slope else None, _ptr(dbias), a2.data_ptr(), _ptr(at), b.data_ptr(), _ptr(bt), M, N, K, _ld(dy2), N, N,
                _ld(a2), M, N, K, _lib.ACT_BY_NAME[activation], dt, _ptr(ws), 0 if ws is None else ws.numel(), torch.cuda.current_stream(dev).cuda_stream),
                "cascmm_epilogue_backward_operands")
            if (want_a or want_b) and dz.element_size() == 2:
                dz = _kernel_rows(dz, _off_dwords(dz, 2))
            if want_a:
                da = cascaded_lowp_matmul(dz, bt, lowp=lowp, terms=terms, products=products).reshape(a.shape)
            if want_b:
                db = cascaded_lowp_matmul(at, dz.contiguous(), lowp=lowp, terms=terms, products=products)
        return da, db, dbias, dy if want_residual else None, None, None, None, None, None


def cascaded_lowp_matmul_epilogue(a: torch.Tensor, b, *, bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                                  residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, lowp: Optional[str] = None,
                                  terms: Optional[int] = None, products: str = "tri", b_exp: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``activation(a @ b + bias) + residual``: :func:`cascaded_lowp_matmul` of ``a`` [..., K] and a 2-D ``b`` [K, N] (or a plain
    :class:`PreparedWeight`; of fp32 one whose K and N its kernels take, see ``usable_with``) with what follows a Linear layer.  ``activation``: None, "relu", "gelu" (erf), "gelu_tanh" or "silu", in fp32.
    ``residual``: of the result's dtype and of a shape that broadcasts to the result's.  ``lowp`` / ``terms`` / ``products`` / ``b_exp`` as there.
    ``out``: [M, N] rows or the result's shape; it overlaps no operand.  The result is rounded once; 16-bit tensors in another cascade than one term of
    their own format, or with a raw weight beyond 2 GiB, have ``a @ b + bias`` rounded to their dtype on the way.

    Differentiable once in ``a``, ``b`` (a tensor: a prepared weight is a constant that no gradient passes through), ``bias`` and
    ``residual``; the gradients' products run with the cascade of the product itself, and sums over rows in a fixed order.  With an
    activation, ``z = a @ b + bias`` and ``dz``, its gradient, are held in the tensors' dtype between the kernels, as 16-bit modules of torch hold them: the
    slope is taken at the rounded ``z``, and the gradients of ``a`` and ``b`` are products of the rounded ``dz`` (that of ``bias`` is the sum of ``dz``
    before it is rounded).  Against gradients from fp32 ``z`` and ``dz`` their mean error is 1.45 times as large (bf16 2.4e-3 for 1.7e-3, fp16 3.0e-4 for 2.1e-4)."""
    act = _lib.ACT_BY_NAME.get(activation) if activation is None or type(activation) is str else None
    if out is None and act is not None and b_exp is None:
        # the ordinary eager call in one native function; None: whatever is not ordinary about it is decided below
        if type(b) is not PreparedWeight:
            y = _lib.short_cut().epilogue(a, b, bias, residual, act, lowp, terms, products)
        elif not b.glu and (lowp is None or lowp == b.lowp) and (terms is None or terms == b.terms):
            y = _lib.short_cut().epilogue_prepared(a, b.slots, bias, residual, act, b.K, b.N, b.fmt, b.terms, products, b.dt)
        else:
            y = None
        if y is not None:
            return y
    prepared = isinstance(b, PreparedWeight)
    _check_device_tensor(a, "a")
    if a.dtype not in _DTYPES:
        raise TypeError(f"cascaded_lowp_matmul_epilogue: unsupported dtype {a.dtype}")
    if a.dim() < 1:
        raise ValueError("cascaded_lowp_matmul_epilogue: a needs at least one dimension")
    if act is None:
        raise ValueError(f"activation must be one of {list(_lib.ACT_BY_NAME)}, got {activation!r}")
    if products not in _lib.PROD_BY_NAME:
        raise ValueError(f"products must be 'tri' or 'full', got {products!r}")
    if prepared:
        if b.glu:
            raise ValueError("a gated weight has an epilogue of its own: cascaded_lowp_matmul applies it")
        if (lowp, terms) != (None, None) and (lowp or b.lowp, terms or b.terms) != (b.lowp, b.terms):
            raise ValueError(f"the weight was prepared as {b.terms} {b.lowp} terms")
        if b.device != a.device:
            raise ValueError(f"the prepared weight is on {b.device} but a on {a.device}")
        if b.dtype != a.dtype:
            raise TypeError(f"cascaded_lowp_matmul_epilogue: a is {a.dtype} but the weight was {b.dtype}")
        if b.fmt == _lib.FMT_FP8 and b.exp is None:
            raise ValueError("an fp8 PreparedWeight needs its tensor-scale exponent (exp)")
        b.check_slots()
        lowp, terms, K, N = b.lowp, b.terms, b.K, b.N
    else:
        _check_device_tensor(b, "b")
        if b.dim() != 2:
            raise ValueError(f"cascaded_lowp_matmul_epilogue: b must be 2-D, got {tuple(b.shape)}")
        if b.device != a.device:
            raise ValueError(f"b is on {b.device} but a on {a.device}")
        if b.dtype != a.dtype:
            raise TypeError(f"cascaded_lowp_matmul_epilogue: a is {a.dtype} but b is {b.dtype}")
        if not b.is_contiguous():
            raise ValueError("cascaded_lowp_matmul_epilogue: b must be contiguous")
        K, N = b.shape
    d_lowp, d_terms = default_cascade(a.dtype)
    lowp, terms = d_lowp if lowp is None else lowp, d_terms if terms is None else terms
    if lowp not in _lib.FMT_BY_NAME:
        raise ValueError(f"lowp must be one of {sorted(_lib.FMT_BY_NAME)}, got {lowp!r}")
    if a.shape[-1] != K:
        raise ValueError(f"a has {a.shape[-1]} columns but b {K} rows")
    shape = (*a.shape[:-1], N)
    M = a.shape[:-1].numel()
    bias = _check_bias(bias, a, N)
    if residual is not None:
        if residual.device != a.device or residual.dtype != a.dtype:
            raise ValueError(f"residual must be like a, {a.dtype} on {a.device}, got {residual.dtype} on {residual.device}")
        try:
            residual = residual.expand(shape)
        except RuntimeError:
            raise ValueError(f"residual of shape {tuple(residual.shape)} does not broadcast to the result's {shape}") from None
    operands = [t for t in (a, None if prepared else b, bias, residual) if t is not None]
    refuse_tangents("cascaded_lowp_matmul_epilogue", *operands)
    if torch.is_grad_enabled() and any(t.requires_grad for t in operands):
        if prepared and a.requires_grad:
            raise RuntimeError("cascaded_lowp_matmul_epilogue: a gradient with respect to a needs the weight itself, not a PreparedWeight")
        if out is not None:
            raise RuntimeError("cascaded_lowp_matmul_epilogue: out= has no gradient")
        if prepared:
            raise RuntimeError("cascaded_lowp_matmul_epilogue: a PreparedWeight is for calls without gradients")
        return _EpilogueProduct.apply(a, b, bias, residual, activation, lowp, terms, products, b_exp)
    a2 = _flat(a)
    if prepared and not b.usable_with(a2, products) and (a.dtype == torch.float32 or K % 8 == 0):     # (16-bit rows of other lengths are copied by the library)
        a2 = a2.contiguous().clone() if a2.is_contiguous() else a2.contiguous()     # (rows off the boundaries that the prepared kernels want)
    if out is None:
        out = torch.empty(shape, dtype=a.dtype, device=a.device)
        out2 = out.view(M, N)
    else:
        _check_device_tensor(out, "out")
        if out.device != a.device or out.dtype != a.dtype:
            raise ValueError(f"out must be like a, {a.dtype} on {a.device}")
        if out.shape != shape and tuple(out.shape) != (M, N):
            raise ValueError(f"out must have shape {shape} or {(M, N)}, got {tuple(out.shape)}")
        try:
            out2 = out.view(M, N)
        except RuntimeError:
            raise ValueError("out must be rows of one distance") from None
        if (N > 1 and out2.stride(1) != 1) or (M > 1 and out2.stride(0) < N):
            raise ValueError("out must have unit stride along N and rows that do not overlap")
        held = [t for t in (a2, b.slots if prepared else b, bias, residual) if t is not None]
        if any(_overlap(out2, t) for t in held):
            raise ValueError("out overlaps an operand")
    _product(a2, b, bias, residual, None, out2, activation, lowp, terms, products, b_exp)
    return out.view(shape) if out.shape != shape else out
