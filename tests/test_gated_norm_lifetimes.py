"""What the norms around a residual add hand to the library, without a GPU: every copy that a call makes of its operands lives until the call's last launch.

The library is replaced by one that looks, at the time of a launch, at what the pointers in its arguments point to.  (Memory that is given back before the launch may be
handed to whatever is allocated in between, on the GPU from the same stream's pool: the backward pass allocates its workspace there.)
"""
import contextlib
import ctypes
import types
import weakref

import pytest
import torch

from basedxl_amd import _lib, gated_norm

SAMPLES, TOKENS, COLS = 3, 5, 8


class Library:
    """Stands for libcascmm.so: keeps what was wrong when a launch was asked for."""

    def __init__(self):
        self.copies, self.launches, self.wrong = {}, 0, []

    def copied(self, name, t):
        self.copies[t.data_ptr()] = (name, weakref.ref(t))

    def launch(self, args, names):
        a = ctypes.cast(args, ctypes.POINTER(_lib.GatedNorm)).contents
        self.launches += 1
        for name in names:
            at = getattr(a, name)
            if at in self.copies and self.copies[at][1]() is None:
                self.wrong.append(f"{name}: the copy is gone")
        self.seen = {name: (getattr(a, name), int(getattr(a, ld)) if ld else 0) for name, ld in
                     (("x", "ldx"), ("residual", "ldr"), ("sum", "lds"), ("dy", "lddy"), ("ds", "ldds"))}

    def cascmm_gated_norm_forward(self, args, stream):
        self.launch(args, ("x", "residual"))
        a = ctypes.cast(args, ctypes.POINTER(_lib.GatedNorm)).contents
        for at, n in ((a.y, 4 * SAMPLES * TOKENS * COLS), (a.sum, 4 * SAMPLES * TOKENS * COLS)):
            ctypes.memset(at, 0, n)
        return 0

    def cascmm_gated_norm_backward(self, args, workspace, nbytes, stream):
        self.launch(args, ("x", "residual", "sum", "dy", "ds", "weight", "bias", "gate", "scale", "post_weight", "post_bias"))
        return 0

    def __getattr__(self, name):
        if name.endswith("_bytes"):
            return lambda *_: 4096
        raise AttributeError(name)


@pytest.fixture
def library(monkeypatch):
    made = Library()
    monkeypatch.setattr(gated_norm._lib, "lib", lambda: made)
    monkeypatch.setattr(torch.cuda, "device", lambda _: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda _=None: types.SimpleNamespace(cuda_stream=0))
    for name in ("_flat", "_rows"):
        def watched(t, inner=getattr(gated_norm, name), name=name):
            out = inner(t)
            if out is not None and out.data_ptr() != t.data_ptr():
                made.copied(name, out)
            return out
        monkeypatch.setattr(gated_norm, name, watched)
    return made


def operands():
    gen = torch.Generator().manual_seed(1)
    draw = lambda *shape: torch.randn(*shape, generator=gen)   # noqa: E731
    plain, turned = draw(SAMPLES, TOKENS, COLS), draw(TOKENS, SAMPLES, COLS).transpose(0, 1)
    columns, expanded = draw(SAMPLES, COLS, TOKENS).transpose(1, 2), draw(SAMPLES, 1, COLS).expand(SAMPLES, TOKENS, COLS)
    return {"plain": plain, "turned": turned, "columns": columns, "expanded": expanded}


@pytest.mark.parametrize("of_gradients", ["plain", "turned", "expanded"])
@pytest.mark.parametrize("of_residual", ["plain", "turned", "columns", "expanded"])
@pytest.mark.parametrize("of_x", ["plain", "turned", "columns", "expanded"])
def test_copies_live_until_the_launch(library, of_x, of_residual, of_gradients):
    forms = operands()
    x, residual, spread = (t.detach().requires_grad_() for t in (forms[of_x], forms[of_residual], torch.ones(SAMPLES, 1).expand(SAMPLES, COLS)))
    parameters = [torch.ones(COLS, requires_grad=True), None, spread, torch.ones(COLS, requires_grad=True), torch.ones(2 * COLS)[::2].requires_grad_(), None]
    y, s = gated_norm._GatedAddNorm.apply(x, residual, *parameters, True, 0, 1e-5, 1.0)
    torch.autograd.grad((y, s), (x, residual), (forms[of_gradients], forms[of_gradients]), allow_unused=True)
    assert library.launches == 2 and not library.wrong, library.wrong
    # (and the rows are described as they lie)
    assert all(ld >= COLS for _, ld in library.seen.values())
