"""The epilogue in the store of every kernel that calls choose, at sizes of whole tiles and over their edges: through the C entry with a workspace of the library's
own size, and the kernel's name asked for first, so that a size that goes to another kernel some day is noticed.  Against the formulas in 64 bits; the
tolerances are those of tests/test_gpu_matmul_epilogue.py."""
import math

import pytest
import torch

from basedxl_amd import _lib, PreparedWeight
from test_gpu_matmul_epilogue import ACTIVATIONS, CASCADES, HALF, TINY, U, within, z_of

pytestmark = pytest.mark.gpu

# (cascade, weight prepared, kernel, whole sizes M x K x N, sizes over the edges; None: calls choose it for whole tiles only)
KERNELS = [
    ("bf16x2", 0, "bd128x128x32_d3_p4", (200, 128, 10240), (197, 128, 10236)),
    ("bf16x2", 0, "bd192x128x64_d2_p4", (1536, 128, 3840), (1087, 320, 3844)),
    ("bf16x2", 0, "bd64x128x64_d3_p4", (77, 128, 10240), (74, 128, 10236)),
    ("bf16x2", 0, "bd96x128x64_d3_p4", (1100, 128, 1920), (1087, 128, 1924)),
    ("bf16x2", 0, "k64x160x16_wk4", (256, 5120, 128), (243, 5120, 125)),
    ("bf16x2", 0, "t128x128x64_w4x1x1_d2_p8", (1024, 640, 3840), (1541, 1280, 1924)),
    ("bf16x2", 0, "t16x16x32_wavek", (16, 128, 64), (3, 128, 61)),
    ("bf16x2", 0, "t16x32x32_wavek", (100, 128, 640), (97, 128, 637)),
    ("bf16x2", 0, "t16x64x32_wavek", (16, 128, 10240), (3, 128, 10237)),
    ("bf16x2", 0, "t256x128x32_w4x1x1_d2", (512, 128, 10240), (1963, 5120, 3836)),
    ("bf16x2", 0, "t256x128x32_w512_narrow", (1100, 128, 3840), (1087, 128, 3844)),
    ("bf16x2", 0, "t256x160x32_w4x1x1_d2", (1024, 128, 10240), (1963, 5120, 5116)),
    ("bf16x2", 0, "t256x192x32_w512_narrow", (1976, 128, 5120), (1963, 128, 5116)),
    ("bf16x2", 0, "t256x256x32_w512_edge", (1100, 128, 10240), (1087, 128, 10236)),
    ("bf16x2", 0, "t256x320x32_w512", (8192, 128, 1920), None),
    ("bf16x2", 0, "t256x320x32_w512_edge", (1976, 128, 10240), (1963, 128, 10236)),
    ("bf16x2", 0, "t32x32x32_wavek", (100, 128, 1280), (97, 128, 1277)),
    ("bf16x2", 0, "t32x64x32_wavek", (100, 128, 2560), (97, 128, 2557)),
    ("bf16x2", 0, "t64x160x64_w2x1x2_d2_p8", (8192, 128, 320), None),
    ("bf16x2", 0, "t64x64x32_wavek", (100, 320, 5120), (97, 320, 5117)),
    ("bf16x2", 0, "t64x64x64_w2x2x1_d3", (64, 128, 10240), (51, 128, 10236)),
    ("bf16x2", 1, "k64x160x16_wk4", (200, 128, 10240), (197, 128, 10237)),
    ("bf16x2", 1, "k64x80x32_wk4", (100, 128, 10240), (97, 128, 10237)),
    ("bf16x2", 1, "t128x128x64_w2x2x1_d2", (2048, 128, 1920), (2053, 128, 1917)),
    ("bf16x2", 1, "t128x160x32_w2x1x2_d3", (512, 128, 10240), (1097, 640, 3837)),
    ("bf16x2", 1, "t16x16x32_wavek", (16, 128, 64), (3, 128, 61)),
    ("bf16x2", 1, "t16x32x32_wavek", (100, 128, 640), (87, 128, 637)),
    ("bf16x2", 1, "t16x64x32_wavek", (16, 128, 10240), (3, 128, 10237)),
    ("bf16x2", 1, "t256x128x32_w4x1x1_d2", (1536, 128, 3840), (687, 640, 10237)),
    ("bf16x2", 1, "t256x128x32_w512_narrow", (1100, 128, 3840), (1087, 128, 3845)),
    ("bf16x2", 1, "t256x160x32_w4x1x1_d2", (1024, 128, 10240), (987, 1280, 10237)),
    ("bf16x2", 1, "t256x192x32_w512_narrow", (1976, 128, 5120), (1963, 128, 5117)),
    ("bf16x2", 1, "t256x256x32_w512_edge", (1100, 128, 10240), (1087, 128, 10237)),
    ("bf16x2", 1, "t256x320x32_w512", (8192, 320, 1920), None),
    ("bf16x2", 1, "t256x320x32_w512_edge", (1976, 128, 10240), (1963, 128, 10237)),
    ("bf16x2", 1, "t32x32x32_wavek", (100, 128, 1280), (97, 128, 1280)),
    ("bf16x2", 1, "t32x64x32_wavek", (100, 128, 2560), (97, 128, 2557)),
    ("bf16x2", 1, "t64x160x64_w2x1x2_d2", (256, 320, 10240), None),
    ("bf16x2", 1, "t64x256x32_w1x4x1_d3", (300, 128, 10240), (287, 128, 10237)),
    ("bf16x2", 1, "t64x64x32_wavek", (200, 128, 3840), (187, 128, 3837)),
    ("bf16x2", 1, "t64x64x64_w2x2x1_d3", (64, 128, 10240), (243, 128, 3837)),
    ("h16", 0, "t128x128x64_h16", (200, 128, 10240), (197, 128, 10234)),
    ("h16", 0, "t128x160x64_h16", (1100, 128, 3840), (1087, 128, 3846)),
    ("h16", 0, "t128x256x64_h16", (1100, 128, 5120), (1087, 128, 5114)),
    ("h16", 0, "t128x64x64_h16", (4096, 5120, 64), (4083, 5120, 58)),
    ("h16", 0, "t16x32x64_hwk", (16, 128, 64), (3, 128, 58)),
    ("h16", 0, "t16x64x64_hwk", (16, 128, 10240), (3, 128, 10234)),
    ("h16", 0, "t256x256x32_h16", (1536, 128, 10240), (1523, 128, 10234)),
    ("h16", 0, "t256x320x32_h16", (1976, 128, 10240), (1963, 128, 10234)),
    ("h16", 0, "t32x32x64_hwk", (100, 128, 1280), (97, 128, 1274)),
    ("h16", 0, "t32x64x64_hwk", (100, 128, 2560), (97, 128, 2554)),
    ("h16", 0, "t64x128x64_h16", (77, 128, 10240), (74, 128, 10234)),
    ("h16", 0, "t64x160x64_h16", (1100, 1280, 1920), (1087, 1280, 1926)),
    ("h16", 0, "t64x64x64_h16", (16, 5120, 64), (3, 5120, 58)),
    ("h16", 1, "t128x128x64_h16", (200, 128, 10240), (197, 128, 10237)),
    ("h16", 1, "t128x160x64_h16", (1100, 128, 3840), (1087, 128, 3845)),
    ("h16", 1, "t128x256x64_h16", (1100, 128, 5120), (1087, 128, 5117)),
    ("h16", 1, "t16x16x64_hwk", (16, 128, 64), (3, 128, 61)),
    ("h16", 1, "t16x32x64_hwk", (100, 128, 640), (97, 128, 637)),
    ("h16", 1, "t16x64x64_hwk", (100, 128, 1280), (97, 128, 1277)),
    ("h16", 1, "t256x256x32_h16", (1536, 128, 10240), (1523, 128, 10237)),
    ("h16", 1, "t256x320x32_h16", (1976, 128, 10240), (1963, 128, 10237)),
    ("h16", 1, "t32x32x64_hwk", (64, 128, 2560), (51, 128, 2557)),
    ("h16", 1, "t32x64x64_hwk", (100, 128, 2560), (97, 128, 2557)),
    ("h16", 1, "t64x128x64_h16", (77, 128, 10240), (74, 128, 10237)),
    ("h16", 1, "t64x160x64_h16", (200, 5120, 10240), (197, 5120, 10237)),
    ("h16", 1, "t64x64x64_h16", (100, 128, 5120), (97, 128, 5117)),
    ("fp16x3", 0, "k64x160x32_f16wk4", (1100, 640, 1920), (1087, 640, 1917)),
    ("fp16x3", 0, "t128x128x32_w4x2x1_d2", (200, 128, 10240), (197, 128, 10236)),
    ("fp16x3", 0, "t16x16x32_wavek", (16, 128, 64), (3, 128, 61)),
    ("fp16x3", 0, "t16x32x32_wavek", (100, 128, 640), (97, 128, 637)),
    ("fp16x3", 0, "t256x160x32_f16k", (1100, 128, 3840), (1087, 128, 3837)),
    ("fp16x3", 0, "t32x32x32_wavek", (100, 128, 1280), (97, 128, 1277)),
    ("fp16x3", 0, "t64x64x32_w2x2x1_d3", (100, 128, 5120), (97, 128, 5116)),
]
CODES = {"bf16x2": (_lib.DT_F32, _lib.FMT_BF16, 2), "fp16x3": (_lib.DT_F32, _lib.FMT_FP16, 3), "fp16": (_lib.DT_F16, _lib.FMT_FP16, 1), "bf16": (_lib.DT_BF16, _lib.FMT_BF16, 1)}
TYPES = {"bf16x2": "fp32", "fp16x3": "fp32x3", "fp16": "fp16", "bf16": "bf16"}   # (names in CASCADES)
# the sizes that the layers of the framework's own model have
MODEL = [(2048, 1280, 1280), (2048, 5120, 1280), (2048, 1280, 5120), (8192, 640, 640), (8192, 640, 2560), (1024, 1280, 1280), (154, 2048, 1280)]


class Case:
    def __init__(self, cascade, prepared, M, K, N, device):
        self.cascade, self.prepared, self.M, self.K, self.N = cascade, prepared, M, K, N
        self.dtype, _, self.lost = CASCADES[TYPES[cascade]]
        gen = torch.Generator(device=device).manual_seed(M + 3 * K + 7 * N)
        r = lambda *s: torch.randn(*s, generator=gen, device=device)   # noqa: E731
        self.a, self.b = r(M, K).to(self.dtype), (r(K, N) / math.sqrt(K)).to(self.dtype)
        self.bias, self.residual = r(N).to(self.dtype), r(M, N).to(self.dtype)
        self.z = {True: z_of(self.a, self.b, self.bias, self.dtype, self.lost)}
        self.z[False] = z_of(self.a, self.b, None, self.dtype, self.lost) if M * N <= 1 << 22 else None
        l, code = _lib.lib(), CODES[cascade]
        self.need = l.cascmm_workspace_bytes(M, N, K, *code, 0)
        self.ws = torch.empty(max(self.need, 16), dtype=torch.uint8, device=device)
        self.weight = PreparedWeight(self.b).slots if prepared else self.b
        v = l.cascmm_call_variant_prepared(self.a.data_ptr(), 0, M, N, K, K, N, *code, 0, self.need) if prepared else l.cascmm_call_variant(
            self.a.data_ptr(), self.b.data_ptr(), M, N, K, K, N, N, *code, 0, self.need)
        self.kernel = _lib.variant_names()[v & 0xFFFF]

    def run(self, act, bias=True, residual=None, keep=False, pad=0, shift=0):
        """residual: None, "rows" or "one" (a row for all); keep: z too; result, residual and z as columns `shift` .. of rows `pad` longer."""
        M, N, what = self.M, self.N, f"{self.kernel} {self.M}x{self.K}x{self.N} {act} bias={bias} residual={residual} z={keep} pad={pad}"
        device, dtype = self.a.device, self.dtype
        y, z = (torch.full((M + 1, N + pad), math.inf, dtype=dtype, device=device) for _ in range(2))
        ldr, r = 0, None
        if residual == "rows":
            wide = torch.full((M, N + pad), math.nan, dtype=dtype, device=device)
            wide[:, shift:shift + N] = self.residual
            r, ldr = wide[:, shift:shift + N], N + pad
        elif residual == "one":
            r = self.residual[0]
        assert _lib.lib().cascmm_gemm_epilogue(
            self.a.data_ptr(), self.weight.data_ptr(), 1 if self.prepared else 0, y[:, shift:].data_ptr(), self.bias.data_ptr() if bias else None,
            None if r is None else r.data_ptr(), z[:, shift:].data_ptr() if keep else None, M, N, self.K, self.K, N, N + pad, ldr, N + pad, *CODES[self.cascade], 0,
            _lib.ACT_BY_NAME[act], None, self.ws.data_ptr(), self.need, torch.cuda.current_stream().cuda_stream) == 0, what
        zd, tol, stored = self.z[bias]
        want = ACTIVATIONS[act](zd)
        off = 1.13 * (stored if dtype == torch.float32 else tol) + 8 * U * (1 + zd.abs())    # (16-bit kernels do not round z on their way)
        if r is not None:
            want = want + r.double()
            off = off + U * (want.abs() + r.double().abs())
        within(y[:M, shift:shift + N], want, off + HALF[dtype] * want.abs() + TINY[dtype], what)
        if keep:
            within(z[:M, shift:shift + N], zd, stored, what + ": z")
        for t in (y, z) if keep else (y,):     # (what lies around the result stays)
            assert all(bool((part == math.inf).all()) for part in (t[M], t[:, :shift], t[:, shift + N:])), what

    def run_all(self):
        self.run("gelu", residual="rows", keep=True)
        self.run("silu", residual="one")
        self.run(None, residual="rows", keep=True, pad=7, shift=3)
        self.run("relu", keep=True)
        self.run("gelu_tanh", pad=8, shift=4)
        self.run(None, residual="rows")
        if self.z[False] is not None:
            self.run("silu", bias=False, residual="rows", pad=1)


def split(cascade):
    return ["fp16", "bf16"] if cascade == "h16" else [cascade]


@pytest.mark.parametrize("cascade, prepared, kernel, sizes", [pytest.param(c, p, k, s, id=f"{c}-{'prepared' if p else 'raw'}-{k}-{'x'.join(map(str, s))}")
                                                              for cc, p, k, whole, ragged in KERNELS for c in split(cc) for s in (whole, ragged) if s is not None])
def test_every_kernel_holds_the_epilogue(gpu_device, cascade, prepared, kernel, sizes):
    case = Case(cascade, prepared, *sizes, gpu_device)
    assert case.kernel.startswith(kernel + "_")
    case.run_all()


@pytest.mark.parametrize("cascade, prepared", [("bf16x2", 0), ("bf16x2", 1), ("fp16x3", 0), ("fp16", 0), ("fp16", 1), ("bf16", 0), ("bf16", 1)])
@pytest.mark.parametrize("M, K, N", MODEL)
def test_sizes_of_the_model(gpu_device, cascade, prepared, M, K, N):
    Case(cascade, prepared, M, K, N, gpu_device).run_all()
