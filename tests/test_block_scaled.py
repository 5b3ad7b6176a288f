"""Block-scaled products without a GPU: what the C entry points and the Python functions refuse, before anything is launched."""
import pytest
import torch

from basedxl_amd import BlockScaledWeight, _lib, block_scaled_matmul

F32, F16, BF16 = _lib.DT_F32, _lib.DT_F16, _lib.DT_BF16
P = 1 << 20   # (stands for a device pointer: the checks come before any launch)


def rounding(x=P, rows=4, cols=8, ldx=8, dtype=F32, square=0, values=P, scales=P, values_t=P, scales_t=P, sums=None, workspace=None, nbytes=0):
    return _lib.lib().cascmm_block_round(x, rows, cols, ldx, dtype, square, values, scales, values_t, scales_t, sums, workspace, nbytes, None)


def product(a=P, sa=P, b=P, sb=P, c=P, bias=None, M=4, N=8, K=16, ldc=8, dtype=F32):
    return _lib.lib().cascmm_block_gemm(a, sa, b, sb, c, bias, M, N, K, ldc, dtype, None)


@pytest.mark.parametrize("change, status", [
    (dict(dtype=3), -3), (dict(rows=-1), -2), (dict(cols=-1), -2), (dict(ldx=7), -2), (dict(rows=2 ** 31), -9), (dict(cols=2 ** 26 + 1, ldx=2 ** 27), -9),
    (dict(rows=2 ** 30, cols=2 ** 20, ldx=2 ** 20), -9), (dict(values=None), -1), (dict(scales=None), -1), (dict(values_t=None), -1), (dict(scales_t=None), -1),
    (dict(x=None), -1), (dict(x=P + 2), -6), (dict(values=P + 8), -6), (dict(values_t=P + 4), -6), (dict(scales=P + 1), -6), (dict(scales_t=P + 2), -6),
    (dict(sums=P), -5), (dict(sums=P, workspace=P, nbytes=31), -5), (dict(sums=P, workspace=P + 4, nbytes=64), -6), (dict(sums=P + 2, workspace=P, nbytes=64), -6),
    (dict(rows=0, x=None), 0), (dict(cols=0, ldx=0, x=None), 0), (dict(values=None, scales=None, values_t=None, scales_t=None, x=None), 0)])
def test_rounding_arguments(change, status):
    assert rounding(**change) == status


@pytest.mark.parametrize("change, status", [
    (dict(dtype=-1), -3), (dict(M=-1), -2), (dict(N=-1), -2), (dict(K=-1), -2), (dict(ldc=7), -2), (dict(M=2 ** 31), -9), (dict(N=2 ** 31, ldc=2 ** 31), -9),
    (dict(K=2 ** 22 + 1), -9), (dict(M=2 ** 20, N=2 ** 20, ldc=2 ** 20), -9), (dict(M=2 ** 17, K=2 ** 21), -9), (dict(N=2 ** 17, ldc=2 ** 17, K=2 ** 21), -9), (dict(a=None), -1), (dict(sa=None), -1), (dict(b=None), -1), (dict(sb=None), -1),
    (dict(c=None), -1), (dict(a=P + 8), -6), (dict(b=P + 1), -6), (dict(sa=P + 2), -6), (dict(sb=P + 1), -6), (dict(c=P + 2), -6), (dict(bias=P + 2), -6),
    (dict(M=0, a=None, c=None), 0), (dict(N=0, ldc=0, b=None, c=None), 0)])
def test_product_arguments(change, status):
    assert product(**change) == status


def linear(x=P, b=P, sb=P, c=P, bias=None, M=4, N=8, K=16, ldx=16, ldc=8, dtype=F16, workspace=P, nbytes=1 << 20):
    return _lib.lib().cascmm_block_linear(x, b, sb, c, bias, M, N, K, ldx, ldc, dtype, workspace, nbytes, None)


@pytest.mark.parametrize("rows", [4, 20])     # (one launch, and two with a workspace)
@pytest.mark.parametrize("change, status", [
    (dict(dtype=4), -3), (dict(M=-1), -2), (dict(N=-1), -2), (dict(K=-1), -2), (dict(ldx=15), -2), (dict(ldc=7), -2), (dict(M=2 ** 31), -9), (dict(N=2 ** 31, ldc=2 ** 31), -9),
    (dict(K=2 ** 22 + 1, ldx=2 ** 23), -9), (dict(x=None), -1), (dict(b=None), -1), (dict(sb=None), -1), (dict(c=None), -1), (dict(x=P + 1), -6), (dict(b=P + 8), -6),
    (dict(sb=P + 2), -6), (dict(c=P + 1), -6), (dict(bias=P + 1), -6), (dict(M=0, x=None, c=None), 0), (dict(N=0, ldc=0, c=None), 0)])
def test_linear_arguments(rows, change, status):
    assert linear(**{"M": rows, **change}) == status


def test_linear_workspace():
    need = _lib.lib().cascmm_block_linear_workspace_bytes
    assert need(16, 5120, F16) == 0 and need(17, 300, BF16) >= 17 * 384 + 17 * 4 and need(1, 300, F32) >= 384 + 4 and need(-1, 5, F16) == 0 and need(20, 2 ** 22 + 1, F16) == 0
    for workspace, nbytes, status in ((None, 1 << 20, -5), (P, need(20, 16, F16) - 1, -5), (P + 8, 1 << 20, -6)):
        assert linear(M=20, workspace=workspace, nbytes=nbytes) == status


def test_sizes():
    values, scales, ws = (getattr(_lib.lib(), f"cascmm_block_{n}_bytes") for n in ("values", "scales", "round_workspace"))
    assert values(3, 1) == 3 * 128 and values(3, 128) == 3 * 128 and values(3, 129) == 3 * 256 and values(0, 5) == 0 and values(5, 0) == 0 and values(-1, 5) == 0
    assert scales(3, 1) == 12 and scales(3, 512) == 12 and scales(3, 513) == 24 and scales(3, 0) == 0 and scales(3, -1) == 0
    assert ws(1, 7) == 28 and ws(129, 7) == 56 and ws(0, 7) == 0 and ws(5, 2 ** 26 + 1) == 0
    assert values(2 ** 31 - 1, 2 ** 31 - 1) == (2 ** 31 - 1) * 2 ** 31


def test_tensors_off_the_gpu_are_refused():
    x = torch.zeros(8, 8)
    with pytest.raises(RuntimeError, match="only runs on an AMD GPU"):
        block_scaled_matmul(x, x)
    with pytest.raises(RuntimeError, match="only runs on an AMD GPU"):
        BlockScaledWeight(x)
