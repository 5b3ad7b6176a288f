"""Products with an epilogue without a GPU: what the C entry points and the Python function refuse, before anything is launched."""
import pytest
import torch

from basedxl_amd import _lib, cascaded_lowp_matmul_epilogue
from basedxl_amd.matmul_epilogue import _overlap, _residual_rows

F32, F16, BF16 = _lib.DT_F32, _lib.DT_F16, _lib.DT_BF16
P = 1 << 20   # (stands for a device pointer: the checks come before any launch)


def product(A=P, B=P, prepared=0, C=P, bias=None, residual=None, preact=None, M=4, N=8, K=16, lda=16, ldb=8, ldc=8, ldr=8, ldp=8, dtype=F32, fmt=0, terms=2,
            products=0, activation=2, ws=None, nbytes=0):
    return _lib.lib().cascmm_gemm_epilogue(A, B, prepared, C, bias, residual, preact, M, N, K, lda, ldb, ldc, ldr, ldp, dtype, fmt, terms, products, activation,
                                           None, ws, nbytes, None)


def backward(dy=P, z=P, dz=P, dbias=P, rows=4, cols=8, lddy=8, ldz=8, lddz=8, activation=2, dtype=F32, ws=P, nbytes=1 << 20):
    return _lib.lib().cascmm_epilogue_backward(dy, z, dz, dbias, rows, cols, lddy, ldz, lddz, activation, dtype, ws, nbytes, None)


def transpose(x=P, out=P, rows=4, cols=8, ldx=8, ldo=4, dtype=F32):
    return _lib.lib().cascmm_transpose(x, out, rows, cols, ldx, ldo, dtype, None)


@pytest.mark.parametrize("change, status", [
    (dict(dtype=9), -3), (dict(fmt=9), -4), (dict(terms=4), -4), (dict(products=2), -4), (dict(activation=-1), -4), (dict(activation=5), -4), (dict(M=-1), -2),
    (dict(lda=15), -2), (dict(ldb=7), -2), (dict(ldc=7), -2), (dict(residual=P, ldr=7), -2), (dict(residual=P, ldr=-8), -2), (dict(preact=P, ldp=7), -2),
    (dict(C=None), -1), (dict(A=None), -1), (dict(B=None), -1), (dict(C=P + 2), -6), (dict(residual=P + 2), -6), (dict(preact=P + 1), -6), (dict(A=P + 2), -6),
    (dict(bias=P + 2), -6), (dict(M=2 ** 31), -9), (dict(M=0, A=None), 0), (dict(N=0, ldb=0, ldc=0, B=None), 0)])
def test_product_arguments(change, status):
    assert product(**change) == status


@pytest.mark.parametrize("change, status", [
    (dict(dtype=9), -3), (dict(activation=5), -4), (dict(rows=-1), -2), (dict(lddy=7), -2), (dict(ldz=7), -2), (dict(lddz=7), -2), (dict(dy=None), -1),
    (dict(z=None), -1), (dict(dy=P + 2), -6), (dict(dz=P + 2), -6), (dict(dbias=P + 2), -6), (dict(ws=None), -5), (dict(nbytes=4), -5), (dict(ws=P + 4), -6),
    (dict(rows=2 ** 31), -9), (dict(dz=None, dbias=None), 0), (dict(rows=0, dbias=None, dy=None, z=None), 0), (dict(cols=0, lddy=0, ldz=0, lddz=0, dy=None), 0)])
def test_backward_arguments(change, status):
    assert backward(**change) == status


@pytest.mark.parametrize("change, status", [
    (dict(dtype=9), -3), (dict(rows=-1), -2), (dict(ldx=7), -2), (dict(ldo=3), -2), (dict(x=None), -1), (dict(out=None), -1), (dict(x=P + 2), -6), (dict(out=P + 2), -6),
    (dict(rows=2 ** 30 + 1, ldo=2 ** 31), -9), (dict(rows=2 ** 20, cols=2 ** 20, ldx=2 ** 20, ldo=2 ** 20), -9), (dict(rows=0, x=None), 0),
    (dict(cols=0, ldx=0, x=None), 0)])
def test_transpose_arguments(change, status):
    assert transpose(**change) == status


def test_workspace_of_the_sums():
    size = _lib.lib().cascmm_epilogue_workspace_bytes
    assert size(-1, 8, F32) == size(8, -1, F32) == size(8, 8, 7) == size(4, 0, F32) == 0
    for rows, cols in ((0, 5), (1, 1280), (65536, 1280), (3, 20000)):
        for dtype in (F32, F16, BF16):
            assert size(rows, cols, dtype) >= 4 * cols and size(rows, cols, dtype) % (4 * cols) == 0


def test_tensors_off_the_gpu_are_refused():
    with pytest.raises(RuntimeError, match="only runs on an AMD GPU"):
        cascaded_lowp_matmul_epilogue(torch.zeros(2, 8), torch.zeros(8, 4))


def test_which_tensors_overlap():
    buf = torch.zeros(6, 32)
    assert _overlap(buf, buf) and _overlap(buf[1:3], buf[2:4]) and not _overlap(buf[:3], buf[3:])
    assert not _overlap(buf[:, :16], buf[:, 16:]) and not _overlap(buf[:, 16:], buf[:, :16]) and not _overlap(buf[1:, 16:], buf[:4, :16])
    assert _overlap(buf[:, :17], buf[:, 16:]) and _overlap(buf[:, 16:], buf[:, :17]) and _overlap(buf[:, 8:16], buf[0])
    assert not _overlap(buf[:0], buf) and not _overlap(buf, torch.zeros(6, 32))
    assert _overlap(buf[:1, :8], buf[0, 4:12]) and not _overlap(buf[:1, :8], buf[0, 8:12])


def test_rows_of_a_residual():
    t = torch.arange(24.0).view(4, 6)
    assert _residual_rows(t, 4, 6)[1] == 6 and _residual_rows(t[1:2], 1, 6)[1] == 6
    for r in (t[0].expand(4, 6), t[:1].expand(4, 6), t[0].expand(2, 2, 6)):
        row, ld = _residual_rows(r, 4, 6)
        assert ld == 0 and torch.equal(row, t[0])
    row, ld = _residual_rows(t[:, :1].expand(4, 6), 4, 6)
    assert ld == 6 and torch.equal(row, t[:, :1].expand(4, 6))
    row, ld = _residual_rows(t[0, 0].expand(4, 6), 4, 6)
    assert ld == 0 and torch.equal(row, torch.zeros(6))
    row, ld = _residual_rows(t.view(2, 2, 6)[:1].expand(2, 2, 6), 4, 6)
    assert ld == 6 and torch.equal(row, t[[0, 1, 0, 1]])
    assert _residual_rows(torch.zeros(4, 9)[:, 1:7], 4, 6)[1] == 9


def test_rows_longer_than_a_launch_can_sum():
    long = 2 ** 26 + 1
    assert backward(cols=long, lddy=long, ldz=long, lddz=long, nbytes=2 ** 62) == -9
    assert _lib.lib().cascmm_epilogue_workspace_bytes(4, long, F32) == 0


def operands(dy=P, z=P, dz=P, dbias=None, A=P, At=P, B=P, Bt=P, M=4, N=8, K=16, lddy=8, ldz=8, lddz=8, lda=16, ldat=4, ldb=8, ldbt=16, activation=2, dtype=F32, ws=None, nbytes=0):
    return _lib.lib().cascmm_epilogue_backward_operands(dy, z, dz, dbias, A, At, B, Bt, M, N, K, lddy, ldz, lddz, lda, ldat, ldb, ldbt, activation, dtype, ws, nbytes, None)


@pytest.mark.parametrize("change, status", [
    (dict(dtype=9), -3), (dict(activation=5), -4), (dict(M=-1), -2), (dict(K=-1), -2), (dict(lddy=7), -2), (dict(lda=15), -2), (dict(ldat=3), -2), (dict(ldb=7), -2),
    (dict(ldbt=15), -2), (dict(A=None), -1), (dict(B=None), -1), (dict(dy=None), -1), (dict(z=None), -1), (dict(At=P + 2), -6), (dict(B=P + 1), -6), (dict(dz=P + 2), -6),
    (dict(dbias=P), -5), (dict(dbias=P, ws=P + 4, nbytes=1 << 20), -6), (dict(M=2 ** 31, ldat=2 ** 31), -9),
    (dict(dz=None, At=None, Bt=None), 0), (dict(M=0, Bt=None), 0), (dict(N=0, ldb=0, At=None), 0), (dict(M=0, N=0, K=0, ldb=0), 0)])
def test_backward_with_operands_arguments(change, status):
    assert operands(**change) == status


# Calls in a child process that sees no GPU, on addresses that are never read: they have to reach the launch, which fails for want of a device
CHILD = """
import json, sys
from basedxl_amd import _lib
l = _lib.lib()
if l.cascmm_init() == 0:
    raise SystemExit("a GPU is visible")
A, B, C, Z, R, WS = (i << 44 for i in range(1, 7))
out = []
for c in json.load(sys.stdin):
    M, K, N, (dt, fmt, terms) = c["M"], c["K"], c["N"], c["cascade"]
    need = l.cascmm_workspace_bytes(M, N, K, dt, fmt, terms, 0)
    out.append(l.cascmm_gemm_epilogue(A + c.get("a_offset", 0), B, c.get("prepared", 0), C, None, R if c.get("residual") else None, Z if c.get("ldp") else None, M, N, K,
                                      c.get("lda", K), N, c.get("ldc", N), c.get("ldr", N), c.get("ldp", N), dt, fmt, terms, 0, c.get("act", 2), None,
                                      WS if need else None, need, None))
json.dump(out, sys.stdout)
"""
LAUNCH = -7
CASCADES = {"bf16x2": (0, 0, 2), "fp16x3": (0, 1, 3), "bf16x3": (0, 0, 3), "fp8x3": (0, 2, 3), "fp16": (1, 1, 1), "bf16": (2, 0, 1)}


def refused(cases):
    """The cases that do not reach the launch, with their statuses."""
    import json
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=root, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", CHILD], input=json.dumps(cases), cwd=root, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    return [(c, st) for c, st in zip(cases, json.loads(r.stdout)) if st != LAUNCH]


@pytest.mark.parametrize("cascade", CASCADES)
def test_rows_far_apart_reach_the_launch(cascade):
    """Results, residuals and z whose rows are further apart than the offsets of some kernel's stores."""
    cases = []
    for M, K, N in ((2, 320, 1280), (70, 640, 640), (300, 1280, 1280), (1024, 1280, 1280), (2048, 5120, 1280), (2048, 1280, 5120), (8192, 640, 640), (333, 456, 211), (4096, 640, 2560)):
        for prepared in (0, 1) if cascade in ("bf16x2", "fp16", "bf16") and K % 64 == 0 else (0,):
            for far in (1 << 20, 1 << 22, 1 << 24, 1 << 30):
                for at in ({"ldp": far}, {"ldc": far, "ldp": N}, {"ldc": far}, {"residual": 1, "ldr": far, "ldp": N}):
                    cases.append(dict(M=M, K=K, N=N, cascade=CASCADES[cascade], prepared=prepared, **at))
    assert not refused(cases)


@pytest.mark.parametrize("cascade", ["fp16", "bf16"])
def test_prepared_16_bit_weights_on_any_number_of_rows_reach_the_launch(cascade):
    """K off 8 and rows off dwords, whose copies are beyond 2 GiB as a whole."""
    cases = [dict(M=M, K=K, N=N, cascade=CASCADES[cascade], prepared=1, **more) for M, K in ((1 << 20, 1025), (1 << 21, 1283), (1 << 30, 9), (2 ** 31 - 1, 1), (3000, 500_001))
             for N in (1, 64, 211) for more in ({}, {"lda": K + 4}, {"residual": 1, "ldp": N, "a_offset": 2})]
    cases += [dict(M=1 << 20, K=1032, N=64, cascade=CASCADES[cascade], prepared=1, **more) for more in ({}, {"lda": 1040})]
    assert not refused(cases)
