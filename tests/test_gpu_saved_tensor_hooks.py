"""The differentiable operators under hooks of saved tensors: activation checkpointing, which ends its second run by an exception in such a hook, saving on the host, and hooks that raise."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from basedxl_amd import _lib, add_layer_norm, block_scaled_matmul, cascaded_lowp_matmul_epilogue, gated_add_norm, layer_norm

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"], autouse=True)
def path(request, monkeypatch):
    """Ordinary eager calls by the host extension, and everything by the Python code."""
    if request.param == "python":
        monkeypatch.setattr(_lib, "_short_cut", _lib._NoShortCut)
    else:
        assert _lib.short_cut() is _lib.native()
    return request.param


# (x [3, 5, 64], a weight [64, 64], a row [64])
OPERATORS = {
    "layer_norm": lambda x, w, b: layer_norm(x, b, b),
    "add_layer_norm": lambda x, w, b: add_layer_norm(x, 2 * x, b, b),
    "epilogue": lambda x, w, b: cascaded_lowp_matmul_epilogue(x, w, bias=b, activation="gelu", residual=x),
    "block_scaled": lambda x, w, b: block_scaled_matmul(x, w, bias=b),
    "block_scaled_turned": lambda x, w, b: block_scaled_matmul(x, w.t(), bias=b),
    "gated": lambda x, w, b: gated_add_norm(x, 2 * x, b, b, gate=b, post_norm=True),
    "several": lambda x, w, b: block_scaled_matmul(gated_add_norm(layer_norm(x, b, b), x, b, gate=b)[0], w, bias=b),
}


def inputs(device):
    gen = torch.Generator().manual_seed(2)
    return [torch.randn(s, generator=gen).to(device) for s in ((3, 5, 64), (64, 64), (64,))]


def gradients(f, operands):
    leaves = [t.detach().clone().requires_grad_() for t in operands]
    out = f(*leaves)
    out = out if isinstance(out, tuple) else (out,)
    torch.autograd.backward(out, [torch.full_like(o, 0.5) for o in out])
    return [o.detach() for o in out] + [t.grad for t in leaves if t.grad is not None]


@pytest.mark.parametrize("name", OPERATORS)
def test_checkpointing(gpu_device, name):
    f, operands = OPERATORS[name], inputs(gpu_device)
    want = gradients(f, operands)
    for how in (dict(use_reentrant=False), dict(use_reentrant=False, early_stop=False), dict(use_reentrant=True)):
        got = gradients(lambda *a: checkpoint(f, *a, **how), operands)
        assert len(got) == len(want) and all(torch.equal(p, q) for p, q in zip(got, want)), how
    # (a call in front of the one that ends the second run, and one behind it)
    g = lambda *a: torch.cat([t.flatten() for t in gradients_of_all(f, *a)])   # noqa: E731
    assert all(torch.equal(p, q) for p, q in zip(gradients(lambda *a: checkpoint(g, *a, use_reentrant=False), operands), gradients(g, operands)))


def gradients_of_all(f, x, w, b):
    first = f(x, w, b)
    first = first if isinstance(first, tuple) else (first,)
    second = f(first[0], w, b)
    return (*first, *(second if isinstance(second, tuple) else (second,)))


@pytest.mark.parametrize("name", OPERATORS)
def test_saved_on_the_host(gpu_device, name):
    f, operands = OPERATORS[name], inputs(gpu_device)

    def saving(*a):
        with torch.autograd.graph.save_on_cpu():
            return f(*a)
    assert all(torch.equal(p, q) for p, q in zip(gradients(saving, operands), gradients(f, operands)))


@pytest.mark.parametrize("name", OPERATORS)
def test_a_hook_that_raises_is_called_once(gpu_device, name):
    f, calls = OPERATORS[name], []
    operands = [t.requires_grad_() for t in inputs(gpu_device)]

    def pack(t):
        calls.append(t)
        raise KeyError("of the hook")
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        with pytest.raises(KeyError, match="of the hook"):
            f(*operands)
    assert len(calls) == 1
    assert all(torch.isfinite(t).all() for t in gradients(f, operands))      # (and nothing is left behind)
