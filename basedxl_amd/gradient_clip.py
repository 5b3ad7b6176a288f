"""The norm of a model's gradients taken together, and their clipping by it: what stands between the backward pass of the operators here and
the step that uses their gradients.  (The reference, basedxl/unet.py:65-87, runs its model without gradients.)  Kernels:
csrc/cascmm_gradients_kernel.h.
"""
from __future__ import annotations

import math
from array import array
from typing import Iterable, List, Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .cascaded_lowp_matmul import _DTYPES

_NORM_TYPES = {1.0: 1, 2.0: 2, math.inf: 0}


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements of ``t``, in whatever order, fill a range of memory once."""
    if t.is_contiguous():
        return True
    span = 1
    for stride, size in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n != 1):
        if stride != span:
            return False
        span *= size
    return True


def _reach(terms: Sequence[Tuple[int, int, int]], low: int, high: int) -> bool:
    """Whether some sum of c * stride, least <= c <= most for each of ``terms`` (stride, least, most), largest strides first, lies in [low, high]."""
    if not terms:
        return low <= 0 <= high
    (stride, least, most), rest = terms[0], terms[1:]
    down, up = sum(s * c for s, c, _ in rest), sum(s * c for s, _, c in rest)
    return any(_reach(rest, low - c * stride, high - c * stride) for c in range(max(least, -((up - low) // stride)), min(most, (high - down) // stride) + 1))


def _steps(t: torch.Tensor) -> List[Tuple[int, int]]:
    """(distance in bytes, indices behind the first) of the axes that move."""
    size = t.element_size()
    return sorted(((st * size, n - 1) for n, st in zip(t.shape, t.stride()) if n > 1), reverse=True)


def _overlap(p: torch.Tensor, q: torch.Tensor) -> bool:
    """Whether two tensors, of any strides, share a byte."""
    if p.numel() == 0 or q.numel() == 0:
        return False
    terms = {}
    for t, sign in ((p, -1), (q, 1)):
        for stride, most in _steps(t):
            if stride:
                least, up = terms.get(stride, (0, 0))
                terms[stride] = (least - most, up) if sign < 0 else (least, up + most)
    apart = q.data_ptr() - p.data_ptr()
    return _reach([(s, *terms[s]) for s in sorted(terms, reverse=True)], 1 - q.element_size() - apart, p.element_size() - 1 - apart)


def _overlaps_itself(t: torch.Tensor) -> bool:
    """Whether two elements of a tensor share memory."""
    if t.numel() == 0:
        return False
    steps = _steps(t)
    if any(stride == 0 for stride, _ in steps):
        return True
    # (two elements whose first index that differs is the k-th)
    return any(_reach([(steps[k][0], 1, steps[k][1])] + [(s, -n, n) for s, n in steps[k + 1:]], 0, 0) for k in range(len(steps)))


def _direct(g: torch.Tensor, o: torch.Tensor) -> bool:
    """Whether the kernels read ``g`` and write ``o`` as they lie (else the elements are copied)."""
    return _dense(g) and (o is g or (_dense(o) and o.stride() == g.stride()))


def _refuse_shared_memory(gradients: Sequence[torch.Tensor], results: Sequence[torch.Tensor]) -> None:
    """Refuses a result that shares memory with another, with a gradient that is not its own or with itself, where one of the two is copied (the C entry point
    sees copies in their places; of the others it sees all)."""
    spans = []
    for i, (g, o) in enumerate(zip(gradients, results)):
        copied = not _direct(g, o)
        if copied and _overlaps_itself(o):
            raise ValueError(f"clip_gradients: elements of result {i} share memory")
        for t, written in ((o, True),) if o is g else ((o, True), (g, False)):
            if t.numel():
                spans.append((t.data_ptr(), t.data_ptr() + sum(s * n for s, n in _steps(t)) + t.element_size(), i, written, copied, t))
    spans.sort(key=lambda s: s[0])
    behind = []      # those that reach beyond where the next one begins
    for span in spans:
        begin, _, i, written, copied, t = span
        behind = [s for s in behind if s[1] > begin]
        for _, _, k, w, c, other in behind:
            if k != i and (written or w) and (copied or c) and _overlap(t, other):
                which = "another" if written and w else f"gradient {k if written else i}"
                raise ValueError(f"clip_gradients: result {i if written else k} shares memory with {which}")
        behind.append(span)


def _check(gradients: Sequence[torch.Tensor], norm_type: float, name: str) -> int:
    kind = _NORM_TYPES.get(float(norm_type))
    if kind is None:
        raise ValueError(f"{name}: norm_type must be 1, 2 or inf, got {norm_type}")
    if not gradients:
        raise ValueError(f"{name}: there are no gradients")
    device = gradients[0].device
    for i, g in enumerate(gradients):
        if not g.is_cuda:
            raise RuntimeError(f"{name}: gradient {i} is on {g.device}; the operator only runs on an AMD GPU (there is no CPU fallback)")
        if g.device != device:
            raise ValueError(f"{name}: gradient {i} is on {g.device} but the first on {device}")
        if g.layout != torch.strided or g.dtype not in _DTYPES:
            raise TypeError(f"{name}: gradient {i} must be a dense fp32, fp16 or bf16 tensor, got {g.layout} {g.dtype}")
    return kind


def _run(gradients, outs, kind: int, max_norm: float) -> torch.Tensor:
    """One cascmm_clip_gradients over tensors that are dense, each like its result in shape and strides (``outs`` None: the norm alone)."""
    device = gradients[0].device
    table = array("q")
    for i, g in enumerate(gradients):
        code, out = _DTYPES[g.dtype], 0
        if outs is not None:
            out, code = outs[i].data_ptr(), code | _DTYPES[outs[i].dtype] << 32
        table.extend((g.data_ptr(), out, g.numel(), code))
    at, count, l = table.buffer_info()[0], len(gradients), _lib.lib()
    with torch.cuda.device(device):
        norm = torch.empty((), dtype=torch.float32, device=device)
        ws = torch.empty(l.cascmm_gradients_workspace_bytes(count, at), dtype=torch.uint8, device=device)   # (a temporary of the call)
        _lib.check(l.cascmm_clip_gradients(count, at, kind, max_norm, norm.data_ptr(), ws.data_ptr(), ws.numel(),
                                           torch.cuda.current_stream(device).cuda_stream), "cascmm_clip_gradients")
    return norm


@torch.no_grad()
def gradient_norm(gradients: Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """The norm (1, 2 or inf) of all elements of all ``gradients`` taken together, a device scalar in fp32; nothing waits for it.  fp32, fp16 and bf16
    tensors of any strides on one GPU, the types mixed at will.  Squares and sums are fp64 in a fixed order: the same call gives the same bits."""
    gradients = list(gradients)
    norm = _lib.short_cut().clip_gradients(gradients, None, _NORM_TYPES.get(norm_type, -1), 0.0)   # the ordinary call in one native function; None: it is decided below
    if norm is not None:
        return norm
    kind = _check(gradients, norm_type, "gradient_norm")
    return _run([g if _dense(g) else g.contiguous() for g in gradients], None, kind, 0.0)


@torch.no_grad()
def clip_gradients(gradients: Iterable[torch.Tensor], max_norm: float, *, norm_type: float = 2.0,
                   out: Optional[Iterable[torch.Tensor]] = None) -> torch.Tensor:
    """``g * min(1, max_norm / (norm + 1e-6))`` for every gradient, in place or into ``out`` (a tensor for each, of its shape and of its type or
    fp32), and the norm of all of them together as :func:`gradient_norm` returns it.  Nothing waits for the GPU: the factor stays there, and gradients
    in place that need no clipping are not written.  A NaN among the gradients makes all of them NaN; an infinity makes the factor 0 and itself NaN.  A result shares memory
    with no other result and no gradient but its own (CascmmError, ValueError where the elements of one of the two are copied: strides with gaps, or other than those of its
    gradient): a tensor that is listed twice would be scaled twice.  Parts of a buffer whose elements lie between each other do not share memory."""
    gradients = list(gradients)
    results = gradients if out is None else list(out)
    norm = _lib.short_cut().clip_gradients(gradients, results, _NORM_TYPES.get(norm_type, -1), max_norm)
    if norm is not None:
        return norm
    kind = _check(gradients, norm_type, "clip_gradients")
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"clip_gradients: max_norm must be a number from 0 on, got {max_norm}")
    if len(results) != len(gradients):
        raise ValueError(f"clip_gradients: {len(gradients)} gradients but {len(results)} results")
    sources, targets, copied = [], [], []
    for i, (g, o) in enumerate(zip(gradients, results)):
        if o is not g:
            if o.device != g.device or o.shape != g.shape or o.layout != torch.strided or o.dtype not in (g.dtype, torch.float32):
                raise ValueError(f"clip_gradients: out[{i}] must be {tuple(g.shape)}, {g.dtype} or float32, on {g.device}, got {tuple(o.shape)} {o.dtype} on {o.device}")
            if o.requires_grad and o.is_leaf:
                raise ValueError(f"clip_gradients: out[{i}] is a leaf that requires a gradient")
    direct = [_direct(g, o) for g, o in zip(gradients, results)]
    if not all(direct):
        _refuse_shared_memory(gradients, results)
    for g, o, whole in zip(gradients, results, direct):
        if whole:
            sources.append(g)
            targets.append(o)
        else:   # (orders of elements that differ, or gaps between them: the scaled elements are put in place behind the call)
            sources.append(g.contiguous())
            targets.append(torch.empty(g.shape, dtype=o.dtype, device=g.device))
            copied.append((o, targets[-1]))
    norm = _run(sources, targets, kind, max_norm)
    for o, t in copied:
        o.copy_(t)
    torch.autograd.graph.increment_version([o for o in results if not o.is_inference()])   # (written behind autograd's back)
    return norm


@torch.no_grad()
def clip_grad_norm_(parameters: Union[torch.Tensor, Iterable[torch.Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> torch.Tensor:
    """The form of ``torch.nn.utils.clip_grad_norm_`` on this package's kernels: clips the ``grad`` of ``parameters`` in place and returns their norm.  Narrower than torch's: gradients in
    fp32, fp16 or bf16 on one GPU, norms 1, 2 and inf, no ``foreach``, and a gradient that is there twice is refused (CascmmError).  Without gradients the norm is a zero on the host.
    ``error_if_nonfinite`` waits for the norm and raises before any gradient is touched."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    gradients = [p.grad for p in parameters if p.grad is not None]
    if not gradients:
        return torch.tensor(0.0)
    if error_if_nonfinite:
        norm = gradient_norm(gradients, norm_type)
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"The total norm of order {norm_type} for gradients is non-finite, so it cannot be clipped: disable this error with error_if_nonfinite=False")
    return clip_gradients(gradients, max_norm, norm_type=norm_type)
