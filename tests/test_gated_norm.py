"""The norms around a residual add without a GPU: what the C entry points and the Python function refuse, before anything is launched."""
import ctypes
import math

import pytest
import torch

from basedxl_amd import _lib, gated_add_norm

F32, F16, BF16 = _lib.DT_F32, _lib.DT_F16, _lib.DT_BF16
P = 1 << 20   # (stands for a device pointer: the checks come before any launch)


def arguments(**change):
    a = _lib.GatedNorm()
    values = dict(x=P, residual=P, gate=P, scale=P, post_weight=P, post_bias=P, weight=P, bias=P, y=P, sum=P, stats=P, dy=P, ds=P, dx=P, dresidual=P, rows=6, cols=8, group_rows=3,
                  ldx=8, ldr=8, ldy=8, lds=8, lddy=8, ldds=8, lddx=8, lddr=8, gate_ld=8, scale_ld=0, weight_ld=8, bias_ld=0, residual_scale=1.0, eps=1e-5, norm=0, post=1,
                  dtype=F32, weight_dtype=F32)
    values.update(change)
    for name, v in values.items():
        setattr(a, name, v)
    return a


BOTH = [(dict(dtype=5), -3), (dict(weight_dtype=F16), -3), (dict(norm=2), -4), (dict(rows=-6), -2), (dict(cols=-1), -2), (dict(rows=7), -2), (dict(group_rows=0), -2),
        (dict(group_rows=-3), -2), (dict(eps=-1.0), -2), (dict(eps=math.nan), -2), (dict(gate_ld=7), -2), (dict(weight_ld=-8), -2), (dict(scale_ld=1), -2), (dict(bias_ld=7), -2),
        (dict(rows=3 * 2 ** 30), -9), (dict(cols=2 ** 26 + 1, gate_ld=0, weight_ld=0), -9), (dict(rows=2 ** 26, group_rows=1), -9), (dict(lds=7), -2), (dict(ldx=7), -2), (dict(ldr=7), -2),
        (dict(sum=None), -1), (dict(x=None), -1), (dict(residual=None), -1), (dict(x=P + 2), -6), (dict(sum=P + 2), -6), (dict(gate=P + 1), -6), (dict(post_bias=P + 2), -6),
        (dict(stats=P + 2), -6), (dict(cols=0, x=None, sum=None, dy=None, y=None, stats=None), 0)]


@pytest.mark.parametrize("change, status", BOTH + [(dict(ldy=7), -2), (dict(y=None), -1), (dict(y=P + 2), -6), (dict(rows=0, x=None, y=None), 0)])
def test_forward_arguments(change, status):
    a = arguments(**change)
    assert _lib.lib().cascmm_gated_norm_forward(ctypes.byref(a), None) == status


@pytest.mark.parametrize("change, status", BOTH + [
    (dict(lddy=7), -2), (dict(ldds=7), -2), (dict(lddx=7), -2), (dict(lddr=7), -2), (dict(dy=None), -1), (dict(stats=None), -1), (dict(dx=P + 2), -6), (dict(dgate=P + 2), -6),
    (dict(dgate=P, gate=None), -1), (dict(dscale=P, scale=None), -1), (dict(dpost_weight=P, post=0), -1), (dict(dpost_bias=P, post_bias=None), -1), (dict(dweight=P, weight=None), -1),
    (dict(dbias=P, bias=None), -1), (dict(dx=None, dresidual=None, dy=None), 0), (dict(rows=0, dy=None, x=None), 0)])
def test_backward_arguments(change, status):
    a = arguments(**change)
    assert _lib.lib().cascmm_gated_norm_backward(ctypes.byref(a), P, 1 << 30, None) == status


def test_workspace():
    a, l = arguments(dweight=P), _lib.lib()
    need = l.cascmm_gated_norm_workspace_bytes(ctypes.byref(a))
    assert need >= 2 * 5 * 8 * 4
    for workspace, nbytes, status in ((None, need, -5), (P, need - 1, -5), (P + 4, need, -6)):
        assert l.cascmm_gated_norm_backward(ctypes.byref(a), workspace, nbytes, None) == status
    for rows, group_rows, cols in ((1, 1, 1), (1 << 20, 1 << 20, 640), (1 << 20, 1 << 10, 640), (40, 10, 20000), (0, 0, 8)):
        a = arguments(rows=rows, group_rows=group_rows, cols=cols, **{k: 0 for k in ("gate_ld", "weight_ld")}, **{k: cols for k in ("ldx", "ldr", "lds", "lddy", "ldds", "lddx", "lddr")})
        groups = rows // group_rows if group_rows else 0
        assert l.cascmm_gated_norm_workspace_bytes(ctypes.byref(a)) >= groups * 20 * cols
    assert l.cascmm_gated_norm_workspace_bytes(None) == 0 and l.cascmm_gated_norm_workspace_bytes(ctypes.byref(arguments(rows=7))) == 0
    assert l.cascmm_gated_norm_forward(None, None) == -1 and l.cascmm_gated_norm_backward(None, None, 0, None) == -1


@pytest.mark.parametrize("dtype, cols", [(F32, 3), (BF16, 7), (F32, 6145), (F16, 9000)])
@pytest.mark.parametrize("rows, group_rows", [(65536, 1), (70000, 1), (1 << 21, 16)])
def test_the_backward_pass_takes_the_groups_that_the_forward_pass_takes(dtype, cols, rows, group_rows):
    """Rows that no registers hold, with parameters for more groups than a grid's second axis has places."""
    lds = {k: cols for k in ("ldx", "ldr", "ldy", "lds", "lddy", "ldds", "lddx", "lddr", "gate_ld", "weight_ld")}
    a, l = arguments(rows=rows, group_rows=group_rows, cols=cols, dtype=dtype, weight_dtype=dtype, dgate=P, dweight=P, dpost_weight=P, **lds), _lib.lib()
    need = l.cascmm_gated_norm_workspace_bytes(ctypes.byref(a))
    assert need >= rows // group_rows * 5 * cols * 4
    assert l.cascmm_gated_norm_backward(ctypes.byref(a), P, need - 1, None) == -5      # (nothing but the workspace is wrong)


@pytest.mark.parametrize("cols, rich", [(8, False), (8, True), (1280, False), (1280, True), (3, False), (9000, True)])
def test_a_backward_pass_asks_for_what_it_writes(cols, rich):
    """No more than 16 bytes where no sum over rows is wanted; three rows of sums, or five, for each group of one row."""
    lds = {k: cols for k in ("ldx", "ldr", "ldy", "lds", "lddy", "ldds", "lddx", "lddr", "gate_ld", "weight_ld")}
    how = dict(rows=32768, group_rows=1, cols=cols, **lds, **({} if rich else dict(scale=None, post_bias=None)))
    l, sums = _lib.lib(), 5 if rich or cols in (3, 9000) else 3
    means = 2 * 32768 * 4 if cols in (3, 9000) else 0
    for wanted, want in ((dict(), 16), (dict(dweight=P), 16 + 32768 * sums * cols * 4 + means), (dict(dgate=P, dbias=P), 16 + 32768 * sums * cols * 4 + means)):
        a = arguments(**how, **wanted)
        assert l.cascmm_gated_norm_backward_bytes(ctypes.byref(a)) == want <= l.cascmm_gated_norm_workspace_bytes(ctypes.byref(a))
        assert l.cascmm_gated_norm_backward(ctypes.byref(a), P, want - 1, None) == -5 and l.cascmm_gated_norm_backward(ctypes.byref(a), None, want, None) == -5
    assert l.cascmm_gated_norm_backward_bytes(None) == 0 and l.cascmm_gated_norm_backward_bytes(ctypes.byref(arguments(rows=7))) == 0


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="only runs on an AMD GPU"):
        gated_add_norm(x, x)
