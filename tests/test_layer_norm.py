"""Layer norm without a GPU: what the C entry points and the Python functions refuse, before anything is launched."""
import pytest
import torch

from basedxl_amd import _lib, add_layer_norm, layer_norm

F32, F16, BF16 = _lib.DT_F32, _lib.DT_F16, _lib.DT_BF16
P = 1 << 20   # (stands for a device pointer: the checks come before any launch)


def forward(x=P, residual=None, weight=P, bias=P, y=P, total=None, mean=None, rstd=None, rows=4, cols=8, ldx=8, ldr=8, ldy=8, lds=8, eps=1e-5,
            dtype=F32, weight_dtype=F32):
    return _lib.lib().cascmm_layer_norm(x, residual, weight, bias, y, total, mean, rstd, rows, cols, ldx, ldr, ldy, lds, eps, dtype, weight_dtype, None)


def backward(dy=P, ds=None, x=P, weight=P, mean=P, rstd=P, dx=P, dweight=P, dbias=P, rows=4, cols=8, lddy=8, ldds=8, ldx=8, lddx=8, dtype=F32,
             weight_dtype=F32, workspace=P, nbytes=1 << 20):
    return _lib.lib().cascmm_layer_norm_backward(dy, ds, x, weight, mean, rstd, dx, dweight, dbias, rows, cols, lddy, ldds, ldx, lddx, dtype, weight_dtype,
                                                 workspace, nbytes, None)


@pytest.mark.parametrize("change, status", [
    (dict(dtype=7), -3), (dict(weight_dtype=F16), -3), (dict(dtype=F16, weight_dtype=BF16), -3), (dict(rows=-1), -2), (dict(cols=-1), -2), (dict(ldx=7), -2),
    (dict(ldy=7), -2), (dict(residual=P, total=P, ldr=7), -2), (dict(residual=P, total=P, lds=7), -2), (dict(eps=-1.0), -2), (dict(eps=float("nan")), -2),
    (dict(x=None), -1), (dict(y=None), -1), (dict(residual=P), -1), (dict(total=P), -1), (dict(mean=P), -1), (dict(rstd=P), -1), (dict(x=P + 2), -6),
    (dict(y=P + 1), -6), (dict(weight=P + 2), -6), (dict(bias=P + 2), -6), (dict(rows=2 ** 31), -9), (dict(cols=2 ** 31, ldx=2 ** 31, ldy=2 ** 31), -9),
    (dict(rows=0, x=None, y=None), 0), (dict(cols=0, ldx=0, ldy=0, x=None, y=None), 0)])
def test_forward_arguments(change, status):
    assert forward(**change) == status


@pytest.mark.parametrize("change, status", [
    (dict(dtype=7), -3), (dict(weight_dtype=F16), -3), (dict(rows=-1), -2), (dict(lddy=7), -2), (dict(ldx=7), -2), (dict(lddx=7), -2), (dict(ds=P, ldds=7), -2),
    (dict(dy=None), -1), (dict(x=None), -1), (dict(mean=None), -1), (dict(rstd=None), -1), (dict(workspace=None), -5), (dict(nbytes=8), -5),
    (dict(workspace=P + 4), -6), (dict(dx=P + 2), -6), (dict(dweight=P + 1), -6), (dict(ds=P + 1), -6), (dict(rows=2 ** 31), -9),
    (dict(dx=None, dweight=None, dbias=None, workspace=None), 0), (dict(rows=0, dy=None, x=None, dweight=None, dbias=None), 0)])
def test_backward_arguments(change, status):
    assert backward(**change) == status


def test_workspace_of_the_sums():
    size = _lib.lib().cascmm_layer_norm_workspace_bytes
    assert size(-1, 8, F32) == size(8, -1, F32) == size(8, 2 ** 31, F32) == size(8, 8, 7) == 0
    for rows, cols in ((0, 5), (1, 1280), (65536, 1280), (3, 20000)):
        for dtype in (F32, F16, BF16):
            assert size(rows, cols, dtype) >= 8 * cols and size(rows, cols, dtype) % (8 * cols) == 0


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="only runs on an AMD GPU"):
        layer_norm(x)
    with pytest.raises(RuntimeError, match="only runs on an AMD GPU"):
        add_layer_norm(x, x)


def test_rows_longer_than_a_launch_can_sum():
    long = 2 ** 26 + 1
    assert forward(cols=long, ldx=long, ldy=long) == -9 and backward(cols=long, lddy=long, ldx=long, lddx=long, nbytes=2 ** 62) == -9
    assert _lib.lib().cascmm_layer_norm_workspace_bytes(4, long, F32) == 0
