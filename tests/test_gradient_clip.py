"""The gradients' norm and clipping without a GPU: what the C entry point and the Python functions refuse, before anything is launched."""
import math
from array import array

import pytest
import torch

from basedxl_amd import _lib, clip_grad_norm_, clip_gradients, gradient_norm

F32, F16, BF16 = _lib.DT_F32, _lib.DT_F16, _lib.DT_BF16
P = 1 << 20   # (stands for a device pointer: the checks come before any launch)


def call(*entries, count=None, listed=True, norm_type=2, max_norm=1.0, norm=P, workspace=P, nbytes=1 << 20):
    table = array("q")
    for data, out, elements, dtype, out_dtype in entries:
        table.extend((data, out, elements, dtype | out_dtype << 32))
    return _lib.lib().cascmm_clip_gradients(len(entries) if count is None else count, table.buffer_info()[0] if listed and entries else None, norm_type, max_norm, norm,
                                            workspace, nbytes, None)


G = (P, P, 8, F32, F32)


@pytest.mark.parametrize("entries, how, status", [
    ([G], dict(count=-1), -2), ([G], dict(listed=False), -1), ([G], dict(norm_type=3), -4), ([G], dict(norm_type=-1), -4), ([G], dict(max_norm=-1.0), -2),
    ([G], dict(max_norm=math.nan), -2), ([G], dict(norm=None), -1), ([G], dict(norm=P + 2), -6), ([G], dict(workspace=None), -5), ([G], dict(nbytes=23), -5),
    ([G], dict(workspace=P + 8), -6), ([(P, P, -1, F32, F32)], {}, -2), ([(P, P, 2 ** 50, F32, F32)], {}, -9), ([(P, P, 8, 3, F32)], {}, -3),
    ([(P, P, 8, F32, F16)], {}, -3), ([(P, P, 8, F16, BF16)], {}, -3), ([(P + 2, P + 2, 8, F32, F32)], {}, -6), ([(P + 1, P + 1, 8, F16, F16)], {}, -6),
    ([(P, P + 64 + 2, 8, F16, F32)], {}, -6), ([(0, P, 8, F32, F32)], {}, -1), ([G, (P + 64, 0, 8, F32, F32)], {}, -1)])
def test_arguments(entries, how, status):
    assert call(*entries, **how) == status


@pytest.mark.parametrize("entries, shared", [
    ([G, G], True),                                                                     # the same one twice
    ([(P, P, 8, F32, F32), (P + 28, P + 28, 8, F32, F32)], True),                       # one element shared
    ([(P, P + 256, 8, F32, F32), (P + 64, P + 256 + 16, 8, F32, F32)], True),           # results over each other
    ([(P, P + 64, 8, F32, F32), (P + 64, P + 256, 8, F32, F32)], True),                 # a result over another's gradient
    ([(P, P + 4, 8, F32, F32)], True),                                                  # shifted onto itself
    ([(P, P, 8, F16, F32)], True)])                                                     # in place, but wider
def test_results_that_share_memory(entries, shared):
    assert call(*entries) == (-11 if shared else 0)
    assert _lib.lib().cascmm_strerror(-11) not in (None, b"unknown status")


def test_workspace():
    size = _lib.lib().cascmm_gradients_workspace_bytes
    table = array("q", [P, 0, 1, F32] * 200)
    at = table.buffer_info()[0]
    assert size(200, at) == 16 + 200 * 8 and size(0, None) == 16 and size(-1, at) == 0 and size(1, None) == 0
    for total in (1, 4096, 4097, 1 << 25, (1 << 25) + 1, 1 << 40):
        table[2] = total
        assert 16 < size(1, at) <= 16 + 8 * 8192


def test_what_the_functions_refuse():
    g = torch.zeros(4)
    for f in (gradient_norm, lambda t: clip_gradients(t, 1.0)):
        with pytest.raises(RuntimeError, match="only runs on an AMD GPU"):
            f([g])
        with pytest.raises(ValueError, match="no gradients"):
            f([])
    with pytest.raises(ValueError, match="norm_type"):
        gradient_norm([g], 3.0)
    with pytest.raises(ValueError, match="norm_type"):
        clip_gradients([g], 1.0, norm_type=0.5)
    p = torch.nn.Parameter(torch.zeros(3))
    assert clip_grad_norm_([p], 1.0).item() == 0.0 and clip_grad_norm_(p, 1.0).item() == 0.0
    p.grad = torch.zeros(3)
    with pytest.raises(RuntimeError, match="only runs on an AMD GPU"):
        clip_grad_norm_([p], 1.0)
