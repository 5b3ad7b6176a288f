"""activation(a @ b + bias) + residual and its gradients against the formulas in 64 bits.

Tolerances, element by element.  u = 2^-24, ``half`` the half step of the tensors' type, S = |a| @ |b|.  K products summed in fp32 are off by at
most K u S whatever the order; splitting fp32 into terms leaves out ``lost`` S: two bf16 terms hold 2^-16 of an operand and leave out lo lo (three
times 2^-16), three fp16 terms less than u.  Activations have slopes up to 1.13, curvatures up to 0.8 and are computed to 8 u (1 + |z|).  Where
a kernel stores z first (no fused store, or z kept for the backward pass), z is off by half |z| more.
"""
import math

import pytest
import torch

from basedxl_amd import _lib, PreparedWeight, add_layer_norm, cascaded_lowp_matmul, cascaded_lowp_matmul_epilogue, layer_norm

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    """Ordinary eager calls by the host extension, and everything by the Python code."""
    if request.param == "python":
        monkeypatch.setattr(_lib, "_short_cut", _lib._NoShortCut)
    else:
        assert _lib.short_cut() is _lib.native()
    return request.param


U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
CASCADES = {"fp32": (torch.float32, {}, 3 * 2.0 ** -16), "fp32x3": (torch.float32, {"lowp": "fp16", "terms": 3}, 2.0 ** -24), "fp16": (torch.float16, {}, 0.0),
            "bf16": (torch.bfloat16, {}, 0.0)}
F = torch.nn.functional
ACTIVATIONS = {None: lambda z: z, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}
SIZES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (2, 320, 1280), (77, 50, 30), (154, 128, 320), (64, 64, 64), (333, 456, 211), (257, 136, 130), (513, 72, 1032),
         (64, 5120, 640), (16, 2048, 66), (300, 1280, 1280), (1100, 640, 2560), (130, 33, 4100)]


def slope_of(z, name):
    z = z.detach().clone().requires_grad_()
    return torch.autograd.grad(ACTIVATIONS[name](z).sum(), z)[0] if name else torch.ones_like(z)


def within(got, want, tol, what, mean=True):
    assert got.shape == want.shape, what
    got = got.detach()
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, the worst {float((off / tol).nan_to_num(nan=math.inf).max()):.2f} of the tolerance"
    norm = float(want.norm())
    if mean and want.numel() >= 1000 and norm > 0:
        # (single errors are at most a few half steps, mostly of independent signs: twice a half step in the mean square is beyond what they add up to)
        assert float((got.double() - want).norm()) <= 2 * max(HALF[got.dtype], 2.0 ** -16 if got.dtype == torch.float32 else 0) * norm, what


def operands(M, K, N, dtype, device, seed=0, w_std=None):
    gen = torch.Generator().manual_seed(seed + 7 * M + 13 * K + 17 * N)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=gen) * std).to(dtype).to(device)   # noqa: E731
    return r(M, K), r(K, N, std=w_std or 1.0 / math.sqrt(K)), r(N), r(M, N), r(M, N)


def z_of(a, b, bias, dtype, lost):
    """(z, its error before any rounding, its error where it is stored), in 64 bits."""
    A, B = a.double(), b.double()
    z = A @ B + (0 if bias is None else bias.double())
    S = A.abs() @ B.abs()
    tol = (a.shape[1] + 4) * U * S + lost * S + 2 * U * z.abs() + (0 if bias is None else U * bias.double().abs())
    return z, tol, tol + HALF[dtype] * z.abs() + TINY[dtype]


def check_forward(y, a, b, bias, act, residual, dtype, lost, what, fused=False):
    z, tol, stored = z_of(a, b, bias, dtype, lost)
    want = ACTIVATIONS[act](z)
    tol = 1.13 * (tol if fused else stored) + 8 * U * (1 + z.abs())
    if residual is not None:
        want = want + residual.double()
        tol = tol + U * (want.abs() + residual.double().abs())
    within(y, want, tol + HALF[dtype] * want.abs() + TINY[dtype], what)


def check_backward(grads, dy, a, b, bias, act, residual, dtype, lost, what):
    z, _, stored = z_of(a, b, bias, dtype, lost)
    A, B, dy = a.double(), b.double(), dy.double()
    slope = slope_of(z, act)
    dz = dy * slope
    if act == "relu":
        off = (z.abs() <= stored).double()
    else:
        off = 0.8 * stored + 8 * U * (1 + z.abs()) if act else torch.zeros_like(z)
    sum_tol = dy.abs() * off + 2 * U * dz.abs()
    tol = sum_tol + (HALF[dtype] * dz.abs() + TINY[dtype] if act else 0)
    # (relu's slope jumps: a z within its error of 0 changes dz by all of dy, and of 70000 values some are there (error 2^-15: two of them), which
    # is (2 / 70000)^1/2 = 5e-3 in the mean square, far above the half steps of the others; the elements' own tolerances hold it)
    mean = act != "relu"
    got = iter(grads)
    M, K = a.shape
    N = b.shape[1]
    want = dz @ B.t()
    within(next(got), want, tol @ B.abs().t() + ((N + 4) * U + lost) * ((dz.abs() + tol) @ B.abs().t()) + HALF[dtype] * want.abs() + TINY[dtype], what + " da", mean)
    want = A.t() @ dz
    within(next(got), want, A.abs().t() @ tol + ((M + 4) * U + lost) * (A.abs().t() @ (dz.abs() + tol)) + HALF[dtype] * want.abs() + TINY[dtype], what + " db", mean)
    if bias is not None:
        want = dz.sum(0)
        within(next(got), want, sum_tol.sum(0) + (64 + M // 8) * U * dz.abs().sum(0) + HALF[dtype] * want.abs() + TINY[dtype], what + " dbias", mean)
    if residual is not None:
        assert torch.equal(next(got).double(), dy), what


@pytest.mark.parametrize("cascade", CASCADES)
@pytest.mark.parametrize("M, K, N", SIZES)
def test_forward_and_backward(gpu_device, path, M, K, N, cascade):
    dtype, options, lost = CASCADES[cascade]
    a, b, bias, residual, dy = operands(M, K, N, dtype, gpu_device)
    for act in ACTIVATIONS:
        for bi, r in ((bias, residual), (None, None), (None, residual), (bias, None)):
            what = f"{act} bias={bi is not None} residual={r is not None}"
            y = cascaded_lowp_matmul_epilogue(a, b, bias=bi, activation=act, residual=r, **options)
            # (16-bit tensors: the store itself holds the epilogue, z is not rounded on the way)
            check_forward(y, a, b, bi, act, r, dtype, lost, what, fused=dtype != torch.float32)
            if (bi is None) != (r is None):
                continue
            leaves = [None if t is None else t.clone().requires_grad_() for t in (a, b, bi, r)]
            y1 = cascaded_lowp_matmul_epilogue(leaves[0], leaves[1], bias=leaves[2], activation=act, residual=leaves[3], **options)
            check_forward(y1, a, b, bi, act, r, dtype, lost, what + " differentiated")
            check_backward(torch.autograd.grad(y1, [t for t in leaves if t is not None], dy), dy, a, b, bi, act, r, dtype, lost, what)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M, K, N", [(1, 64, 64), (2, 320, 1280), (154, 1280, 5120), (2048, 1280, 1280), (333, 456, 212), (70, 136, 33), (40, 5120, 640), (700, 1280, 100)])
def test_prepared_weights(gpu_device, path, M, K, N, dtype):
    a, b, bias, residual, _ = operands(M, K, N, dtype, gpu_device)
    lost = CASCADES["fp32"][2] if dtype == torch.float32 else 0.0
    pw = PreparedWeight(b)
    for act in ACTIVATIONS:
        y = cascaded_lowp_matmul_epilogue(a, pw, bias=bias, activation=act, residual=residual)
        check_forward(y, a, b, bias, act, residual, dtype, lost, f"{act}", fused=dtype != torch.float32)
    y = cascaded_lowp_matmul_epilogue(a, pw)
    check_forward(y, a, b, None, None, None, dtype, lost, "plain")
    # rows off 16-byte boundaries
    wide = torch.zeros(M, K + 11, dtype=dtype, device=gpu_device)
    wide[:, 3:3 + K] = a
    y = cascaded_lowp_matmul_epilogue(wide[:, 3:3 + K], pw, bias=bias, activation="silu", residual=residual)
    check_forward(y, a, b, bias, "silu", residual, dtype, lost, "off the boundaries")


def test_other_cascades_are_the_plain_product_with_the_epilogue_behind(gpu_device):
    for lowp, terms in (("fp8", 3), ("fp8", 2), ("bf16", 3), ("fp16", 2)):
        for M, K, N in ((130, 192, 320), (3, 77, 50)):
            a, b, bias, residual, _ = operands(M, K, N, torch.float32, gpu_device)
            z = cascaded_lowp_matmul(a, b, bias=bias, lowp=lowp, terms=terms).double()
            y = cascaded_lowp_matmul_epilogue(a, b, bias=bias, activation="gelu", residual=residual, lowp=lowp, terms=terms)
            want = F.gelu(z) + residual.double()
            within(y, want, 8 * U * (1 + z.abs()) + 2 * U * (want.abs() + residual.double().abs()), f"{lowp} x {terms}")


@pytest.mark.parametrize("cascade", CASCADES)
def test_no_inputs_rows_or_outputs(gpu_device, path, cascade):
    dtype, options, _ = CASCADES[cascade]
    for M, K, N in ((0, 8, 8), (4, 8, 0), (5, 0, 9), (0, 0, 0)):
        a, b = torch.ones(M, K, dtype=dtype, device=gpu_device, requires_grad=True), torch.ones(K, N, dtype=dtype, device=gpu_device, requires_grad=True)
        bias = torch.linspace(-1, 1, max(N, 1)).to(dtype).to(gpu_device)[:N].requires_grad_()
        residual = torch.ones(M, N, dtype=dtype, device=gpu_device)
        with torch.no_grad():
            y = cascaded_lowp_matmul_epilogue(a, b, bias=bias, activation="relu", residual=residual, **options)
        assert torch.equal(y, (F.relu(bias.detach()) + 1).expand(M, N))
        y = cascaded_lowp_matmul_epilogue(a, b, bias=bias, activation="relu", residual=residual, **options)
        da, db, dbias = torch.autograd.grad(y, (a, b, bias), torch.ones_like(y))
        assert torch.equal(dbias, M * (bias > 0).to(dtype)) and bool((db == 0).all()) and da.shape == a.shape


@pytest.mark.parametrize("cascade", CASCADES)
def test_shapes_strides_and_results_in_place(gpu_device, path, cascade):
    dtype, options, lost = CASCADES[cascade]
    a, b, bias, residual, _ = operands(60, 136, 72, dtype, gpu_device)
    want = cascaded_lowp_matmul_epilogue(a, b, bias=bias, activation="gelu", residual=residual, **options)
    how = dict(bias=bias, activation="gelu", **options)
    y = cascaded_lowp_matmul_epilogue(a.view(3, 4, 5, 136), b, residual=residual.view(3, 4, 5, 72), **how)
    assert y.shape == (3, 4, 5, 72) and torch.equal(y.view(60, 72), want)
    assert torch.equal(cascaded_lowp_matmul_epilogue(a[7], b, residual=residual[7], **how), cascaded_lowp_matmul_epilogue(a[7:8], b, residual=residual[7:8], **how)[0])
    # rows of larger tensors, for every operand and the result; what lies around the result stays
    for pad in (8, 3):
        big = [torch.full((62, w + 2 * pad), 5.0, dtype=dtype, device=gpu_device) for w in (136, 72, 72)]
        va, vr, vo = big[0][1:61, pad:pad + 136], big[1][1:61, pad:pad + 72], big[2][1:61, pad:pad + 72]
        va.copy_(a)
        vr.copy_(residual)
        got = cascaded_lowp_matmul_epilogue(va, b, residual=vr, out=vo, **how)
        assert got.data_ptr() == vo.data_ptr()
        check_forward(vo, a, b, bias, "gelu", residual, dtype, lost, f"strided {pad}")
        vo.fill_(5.0)
        assert bool((big[2] == 5.0).all())
    # result and residual as columns of one tensor
    both = torch.zeros(60, 144, dtype=dtype, device=gpu_device)
    both[:, 72:] = residual
    cascaded_lowp_matmul_epilogue(a, b, residual=both[:, 72:], out=both[:, :72], **how)
    check_forward(both[:, :72], a, b, bias, "gelu", residual, dtype, lost, "side by side")
    assert torch.equal(both[:, 72:], residual)
    # transposed a
    at = a.t().contiguous().t()
    assert torch.equal(cascaded_lowp_matmul_epilogue(at, b, residual=residual, **how), want)


@pytest.mark.parametrize("cascade", CASCADES)
def test_broadcast_residuals(gpu_device, path, cascade):
    dtype, options, lost = CASCADES[cascade]
    a, b, bias, residual, dy = operands(60, 136, 72, dtype, gpu_device)
    a3, dy3 = a.view(4, 15, 136), dy.view(4, 15, 72)
    for r in (residual[0], residual[:1], residual[:15].view(1, 15, 72), residual[:4].view(4, 1, 72), residual[0, :1], residual[0, 0]):
        full = r.expand(4, 15, 72).reshape(60, 72)
        leaf = r.clone().requires_grad_()
        y = cascaded_lowp_matmul_epilogue(a3, b, bias=bias, activation="silu", residual=r, **options)
        check_forward(y.view(60, 72), a, b, bias, "silu", full, dtype, lost, f"{tuple(r.shape)}")
        y = cascaded_lowp_matmul_epilogue(a3, b, bias=bias, activation="silu", residual=leaf, **options)
        (g,) = torch.autograd.grad(y, leaf, dy3)
        want = dy3.double().sum_to_size(r.shape)
        within(g, want, HALF[dtype] * want.abs() + 72 * HALF[dtype] * dy3.double().abs().sum_to_size(r.shape), "its gradient")


def test_gradients_of_some_operands(gpu_device, path):
    a, b, bias, residual, dy = operands(90, 136, 72, torch.float16, gpu_device)
    every = [t.clone().requires_grad_() for t in (a, b, bias, residual)]
    want = torch.autograd.grad(cascaded_lowp_matmul_epilogue(every[0], every[1], bias=every[2], activation="gelu", residual=every[3]), every, dy)
    for mask in range(1, 16):
        leaves = [t.clone().requires_grad_(bool(mask >> i & 1)) for i, t in enumerate((a, b, bias, residual))]
        y = cascaded_lowp_matmul_epilogue(leaves[0], leaves[1], bias=leaves[2], activation="gelu", residual=leaves[3])
        y.backward(dy)
        for leaf, grad in zip(leaves, want):
            assert leaf.grad is None if not leaf.requires_grad else torch.equal(leaf.grad, grad)
    # a gradient that is one value for every element, as a sum gives
    y = cascaded_lowp_matmul_epilogue(every[0], every[1], bias=every[2], activation="gelu", residual=every[3])
    ones = torch.autograd.grad(y.sum(), every, retain_graph=True)
    again = torch.autograd.grad(y, every, torch.ones_like(y))
    assert all(torch.equal(p, q) for p, q in zip(ones, again))


def test_against_differences(gpu_device):
    gen = torch.Generator().manual_seed(5)
    a, b, bias, residual, dy = (torch.randn(*s, generator=gen) for s in ((20, 24), (24, 30), (30,), (20, 30), (20, 30)))
    for act in ("gelu", "gelu_tanh", "silu", None):
        def loss(a, b, bias, residual):
            return ((ACTIVATIONS[act](a @ b / 5 + bias) + residual) * dy.double()).sum()

        leaves = [t.to(gpu_device).requires_grad_() for t in (a, b / 5, bias, residual)]
        y = cascaded_lowp_matmul_epilogue(leaves[0], leaves[1], bias=leaves[2], activation=act, residual=leaves[3], lowp="fp16", terms=3)
        grads = list(torch.autograd.grad(y, leaves, dy.to(gpu_device)))
        grads[1] = grads[1] / 5
        at = [t.double() for t in (a, b, bias, residual)]
        for i, grad in enumerate(grads):
            direction = torch.randn(at[i].shape, generator=gen).double()
            plus, minus = [t.clone() for t in at], [t.clone() for t in at]
            plus[i] += 1e-5 * direction
            minus[i] -= 1e-5 * direction
            slope = (loss(*plus) - loss(*minus)) / 2e-5
            scale = (grad.cpu().double() * direction).abs().sum()
            assert abs(slope - (grad.cpu().double() * direction).sum()) <= 500 * U * scale + 1e-8 * scale


@pytest.mark.parametrize("dtype", HALF)
def test_activations_over_the_whole_range(gpu_device, dtype):
    """z as the bias of a product without inputs: single points, infinities and NaN."""
    z = torch.cat([torch.linspace(-12, 12, 4801), torch.logspace(-30, 4, 400), -torch.logspace(-30, 4, 400), torch.zeros(1)]).to(dtype).to(gpu_device)
    z = z[z.isfinite()]
    none = torch.zeros(1, 0, dtype=dtype, device=gpu_device), torch.zeros(0, z.numel(), dtype=dtype, device=gpu_device)
    for act in ("relu", "gelu", "gelu_tanh", "silu"):
        leaf = z.clone().requires_grad_()
        y = cascaded_lowp_matmul_epilogue(*none, bias=leaf, activation=act)[0]
        want = ACTIVATIONS[act](z.double())
        # (behind 12 relative only: an exponential's argument x log2(e), rounded, is off by u |x| log2(e), and the exponential by a relative u |x|: silu(-80)
        # is off by 80 u of itself; a sigmoid below the normal numbers, 2^-126, counts as zero, and z times it, z from -88 to -104, is below 2^-119)
        within(y, want, 8 * U * (1 + z.double().abs()) * (z.double().abs() < 12) + (4 + 2 * z.double().abs().clamp(max=150)) * U * want.abs() + HALF[dtype] * want.abs() + TINY[dtype] + 2.0 ** -119, act)
        (g,) = torch.autograd.grad(y.sum(), leaf)
        slope = slope_of(z.double(), act)
        within(g, slope, 8 * U * (1 + z.double().abs()) * (z.double().abs() < 20) + (4 + 2 * z.double().abs().clamp(max=150)) * U * slope.abs() + HALF[dtype] * slope.abs() + TINY[dtype] + 2.0 ** -100, act + " slope")
    ends = torch.tensor([math.inf, math.nan], dtype=dtype, device=gpu_device)
    none = torch.zeros(1, 0, dtype=dtype, device=gpu_device), torch.zeros(0, 2, dtype=dtype, device=gpu_device)
    for act in ("relu", "gelu", "gelu_tanh", "silu"):
        y = cascaded_lowp_matmul_epilogue(*none, bias=ends, activation=act)[0]
        assert float(y[0]) == math.inf and bool(y[1].isnan())


@pytest.mark.parametrize("cascade", CASCADES)
def test_nan_and_infinity_stay_in_their_rows(gpu_device, cascade):
    dtype, options, _ = CASCADES[cascade]
    if cascade == "fp32x3":
        return      # (the scale of an operand is one for all its rows there)
    a, b, bias, residual, _ = operands(140, 136, 72, dtype, gpu_device)
    want = cascaded_lowp_matmul_epilogue(a, b, bias=bias, activation="gelu", residual=residual, **options)
    a[37, 5] = math.nan
    residual[99, 3] = math.inf
    y = cascaded_lowp_matmul_epilogue(a, b, bias=bias, activation="gelu", residual=residual, **options)
    assert bool(y[37].isnan().all()) and float(y[99, 3]) == math.inf
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[37], keep[99, 3] = False, False
    assert torch.equal(y[keep], want[keep])


@pytest.mark.parametrize("cascade", CASCADES)
def test_streams_graphs_and_repetition(gpu_device, path, cascade):
    dtype, options, _ = CASCADES[cascade]
    a, b, bias, residual, dy = operands(300, 640, 320, dtype, gpu_device)

    def step(a, b, bias, residual, dy):
        y = cascaded_lowp_matmul_epilogue(a, b, bias=bias, activation="gelu", residual=residual, **options)
        return (y, *torch.autograd.grad(y, (a, b, bias, residual), dy))

    side, graphs = torch.cuda.Stream(), []
    for seed in (1, 2):
        ins = [t.clone().requires_grad_() for t in (a, b, bias, residual)] + [dy.clone()]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*ins)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(*ins)
        graphs.append((graph, ins, outs, torch.Generator().manual_seed(seed)))
    for _ in range(4):
        for graph, ins, outs, gen in graphs:
            with torch.no_grad():
                for t in ins:
                    t.copy_(torch.randn(t.shape, generator=gen) * 0.2)
            graph.replay()
            want = step(*[t.detach().clone().requires_grad_() for t in ins[:4]], ins[4])
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs, want))


def test_a_block_of_them(gpu_device, path):
    """A pre-norm feed-forward block and the norm of the next one, forward and backward: x1 = x + W2 gelu(W1 norm(x)), y = norm(x1)."""
    gen = torch.Generator().manual_seed(77)
    M, D, H = 700, 320, 1280
    P = {"x": torch.randn(M, D, generator=gen), "g1": 1 + 0.1 * torch.randn(D, generator=gen), "c1": 0.1 * torch.randn(D, generator=gen),
         "w1": torch.randn(D, H, generator=gen) / D ** 0.5, "b1": 0.1 * torch.randn(H, generator=gen), "w2": torch.randn(H, D, generator=gen) / H ** 0.5,
         "b2": 0.1 * torch.randn(D, generator=gen), "g2": 1 + 0.1 * torch.randn(D, generator=gen), "c2": 0.1 * torch.randn(D, generator=gen)}
    dy, ds = torch.randn(M, D, generator=gen), torch.randn(M, D, generator=gen)

    def block(p, norm, add_norm, product, split):
        h = product(norm(p["x"], p["g1"], p["c1"]), p["w1"], p["b1"], "gelu", None)
        if split:
            return add_norm(product(h, p["w2"], p["b2"], None, None), p["x"], p["g2"], p["c2"])
        s = product(h, p["w2"], p["b2"], None, p["x"])
        return norm(s, p["g2"], p["c2"]), s

    def plain(p):
        n = lambda x, g, c: F.layer_norm(x, (D,), g, c, 1e-5)   # noqa: E731
        def pr(a, b, bias, act, r):
            y = ACTIVATIONS[act](a @ b + bias)
            return y if r is None else y + r
        return block(p, n, None, pr, False)

    for dtype, options, bound in ((torch.float32, {"lowp": "fp16", "terms": 3}, 2e-6), (torch.float16, {}, 4 * HALF[torch.float16]), (torch.bfloat16, {}, 4 * HALF[torch.bfloat16])):
        own = lambda a, b, bias, act, r: cascaded_lowp_matmul_epilogue(a, b, bias=bias, activation=act, residual=r, **options)   # noqa: E731
        q = {k: v.to(dtype).to(gpu_device) for k, v in P.items()}
        e = {k: v.double().requires_grad_() for k, v in q.items()}
        d1, d2 = dy.to(dtype).to(gpu_device), ds.to(dtype).to(gpu_device)
        want = plain(e)
        wanted = [*want, *torch.autograd.grad(want, list(e.values()), (d1.double(), d2.double()))]
        for split in (False, True):
            leaves = {k: v.clone().requires_grad_() for k, v in q.items()}
            got = block(leaves, layer_norm, add_layer_norm, own, split)
            gots = [*got, *torch.autograd.grad(got, list(leaves.values()), (d1, d2))]
            for name, p, w in zip(["y", "s", *P], gots, wanted):
                # (a handful of roundings one behind the other, each of at most a half step and of independent signs: four in the mean square)
                assert float((p.detach().double() - w.detach()).norm() / w.detach().norm()) <= bound, (dtype, split, name)


def test_refusals(gpu_device, path):
    a, b = torch.zeros(4, 16, device=gpu_device), torch.zeros(16, 8, device=gpu_device)
    bad = [(dict(activation="tanh"), ValueError), (dict(products="all"), ValueError), (dict(lowp="fp4"), ValueError), (dict(bias=torch.zeros(7, device=gpu_device)), ValueError),
           (dict(bias=torch.zeros(8, device=gpu_device, dtype=torch.float16)), ValueError), (dict(residual=torch.zeros(4, 8)), ValueError),
           (dict(residual=torch.zeros(4, 8, device=gpu_device, dtype=torch.float16)), ValueError), (dict(residual=torch.zeros(3, 8, device=gpu_device)), ValueError),
           (dict(residual=torch.zeros(2, 4, 8, device=gpu_device)), ValueError), (dict(out=torch.zeros(4, 9, device=gpu_device)), ValueError),
           (dict(out=torch.zeros(4, 8, device=gpu_device, dtype=torch.float16)), ValueError), (dict(out=torch.zeros(8, 4, device=gpu_device).t()), ValueError),
           (dict(out=torch.zeros(1, 8, device=gpu_device).expand(4, 8)), ValueError), (dict(out=a.view(8, 8)[:4]), ValueError)]
    for change, error in bad:
        with pytest.raises(error):
            cascaded_lowp_matmul_epilogue(a, b, **change)
    r = torch.zeros(4, 8, device=gpu_device)
    with pytest.raises(ValueError, match="overlaps"):
        cascaded_lowp_matmul_epilogue(a, b, residual=r, out=r)
    for pair, error in (((a, b.t()), ValueError), ((a, b.half()), TypeError), ((a.double(), b.double()), TypeError), ((a, b.view(1, 16, 8)), ValueError),
                        ((a[:, :8], b), ValueError), ((a, b.t().contiguous().t()), ValueError), ((a, b.cpu()), RuntimeError)):
        with pytest.raises(error):
            cascaded_lowp_matmul_epilogue(*pair)
    pw = PreparedWeight(torch.zeros(64, 8, device=gpu_device))
    x = torch.zeros(4, 64, device=gpu_device)
    assert cascaded_lowp_matmul_epilogue(x, pw).shape == (4, 8)
    for args, change in (((x.requires_grad_(), pw), {}), ((x.detach(), pw), dict(bias=torch.zeros(8, device=gpu_device, requires_grad=True))),
                         ((a.clone().requires_grad_(), b), dict(out=torch.zeros(4, 8, device=gpu_device)))):
        with pytest.raises(RuntimeError):
            cascaded_lowp_matmul_epilogue(*args, **change)
    with torch.no_grad():
        assert cascaded_lowp_matmul_epilogue(x, pw).shape == (4, 8)
    for change in (dict(lowp="fp16"), dict(terms=3)):
        with pytest.raises(ValueError):
            cascaded_lowp_matmul_epilogue(x.detach(), pw, **change)
    with pytest.raises(ValueError):
        cascaded_lowp_matmul_epilogue(x.detach(), PreparedWeight(torch.zeros(64, 128, device=gpu_device), glu=True))
    leaf = a.clone().requires_grad_()
    (g,) = torch.autograd.grad(cascaded_lowp_matmul_epilogue(leaf, b).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_the_host_extension_takes_ordinary_calls(gpu_device):
    native = _lib.native()
    a, b, bias, residual, _ = operands(24, 64, 32, torch.float16, gpu_device)
    cascaded_lowp_matmul_epilogue(a, b)     # (the stream's workspace exists)
    want = cascaded_lowp_matmul_epilogue(a, b, bias=bias, activation="gelu", residual=residual)
    assert torch.equal(native.epilogue(a, b, bias, residual, 2, None, None, "tri"), want)
    assert native.epilogue(a.clone().requires_grad_(), b, bias, residual, 2, None, None, "tri").requires_grad
    pw = PreparedWeight(b)
    args = (pw.K, pw.N, pw.fmt, pw.terms, "tri", pw.dt)
    assert torch.equal(native.epilogue_prepared(a, pw.slots, bias, residual, 2, *args), cascaded_lowp_matmul_epilogue(a, pw, bias=bias, activation="gelu", residual=residual))
    assert native.epilogue_prepared(a.clone().requires_grad_(), pw.slots, bias, residual, 2, *args) is None
    assert native.epilogue_prepared(a, pw.slots[:-1].clone(), bias, residual, 2, *args) is None
    for change in ({0: a.cpu()}, {1: b.t()}, {1: b[:60]}, {2: bias[:3]}, {2: bias.float()}, {3: residual[:3]}, {3: residual.float()}, {3: residual[0]}, {4: 5}, {4: -1}, {4: None},
                   {5: "fp8"}, {5: 3}, {6: "a"}, {7: "all"}, {0: a[:0]}, {0: a.double()}):
        call = [a, b, bias, residual, 2, None, None, "tri"]
        for k, v in change.items():
            call[k] = v
        assert native.epilogue(*call) is None, change


@pytest.mark.parametrize("cascade", [*CASCADES, "fp8x3"])
def test_rows_far_apart(gpu_device, cascade):
    """Results and residuals whose rows are 2.2 GB apart, beyond what a store's offsets span, and a single row whose distance to the next is beyond all numbers."""
    dtype, options, lost = CASCADES[cascade] if cascade in CASCADES else (torch.float32, {"lowp": "fp8", "terms": 3}, None)

    def check(y, a, b, bias, act, residual):
        if lost is not None:
            return check_forward(y, a, b, bias, act, residual, dtype, lost, cascade)
        # (three fp8 terms leave out 2^-12 of an operand and products of 2^-12 twice: below 2^-9 S, and S is some 0.8 K^1/2 of z: 0.06 z; a lost row is 0.7 of it)
        z = ACTIVATIONS[act](z_of(a, b, bias, dtype, 0)[0]) + (0 if residual is None else residual.double())
        assert float((y.double() - z).norm()) <= 0.1 * float(z.norm())

    for M, K, N in ((1, 64, 64), (2, 640, 320), (2, 1280, 2560)):
        a, b, bias, residual, _ = operands(M, K, N, dtype, gpu_device)
        far = 2_200_000_000 // a.element_size()
        store = torch.empty(far * (M - 1) + N, dtype=dtype, device=gpu_device)
        rows = store.as_strided((M, N), (far if M > 1 else 2 ** 59, 1))
        for act, r in (("silu", residual), (None, None)):
            rows.fill_(math.nan)
            check(cascaded_lowp_matmul_epilogue(a, b, bias=bias, activation=act, residual=r, out=rows, **options), a, b, bias, act, r)
        rows.copy_(residual)
        check(cascaded_lowp_matmul_epilogue(a, b, bias=bias, activation="silu", residual=rows, **options), a, b, bias, "silu", residual)


@pytest.mark.parametrize("cascade", CASCADES)
@pytest.mark.parametrize("act", [None, "gelu"])
def test_gradients_that_arrive_strided(gpu_device, path, cascade, act):
    """dy as columns of wider rows, at a distance and an offset of their own."""
    dtype, options, lost = CASCADES[cascade]
    for M, K, N in ((70, 33, 45), (64, 128, 96), (5, 640, 1283)):
        a, b, bias, residual, dy = operands(M, K, N, dtype, gpu_device)
        wide = torch.full((M, N + 13), math.nan, dtype=dtype, device=gpu_device)
        wide[:, 5:5 + N] = dy
        leaves = [t.clone().requires_grad_() for t in (a, b, bias, residual)]
        y = cascaded_lowp_matmul_epilogue(leaves[0], leaves[1], bias=leaves[2], activation=act, residual=leaves[3], **options)
        grads = torch.autograd.grad(y, leaves, wide[:, 5:5 + N])
        check_backward(grads, dy, a, b, bias, act, residual, dtype, lost, f"{M} {K} {N}")


def test_two_threads_on_one_stream(gpu_device):
    """Calls whose launches meet in the stream's workspace, from two threads at once."""
    import threading
    stream, wrong = torch.cuda.current_stream(gpu_device), []
    sets = [operands(154, 1280, 640, torch.float32, gpu_device, seed=s) for s in (1, 2)]
    options = {"lowp": "fp16", "terms": 3}
    wants = [cascaded_lowp_matmul_epilogue(s[0], s[1], bias=s[2], activation="gelu", residual=s[3], **options) for s in sets]

    def work(ops, want):
        with torch.cuda.stream(stream):
            for _ in range(50):
                got = cascaded_lowp_matmul_epilogue(ops[0], ops[1], bias=ops[2], activation="gelu", residual=ops[3], **options)
                if not torch.equal(got, want):
                    wrong.append(1)

    threads = [threading.Thread(target=work, args=pair) for pair in zip(sets, wants)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_forward_mode_tangents_are_refused(gpu_device, path):
    from torch.autograd import forward_ad
    a, b, bias, residual, _ = operands(24, 64, 32, torch.float16, gpu_device)
    with forward_ad.dual_level():
        for k in range(4):
            ops = [forward_ad.make_dual(t, t) if i == k else t for i, t in enumerate((a, b, bias, residual))]
            with pytest.raises(NotImplementedError):
                cascaded_lowp_matmul_epilogue(ops[0], ops[1], bias=ops[2], residual=ops[3])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M, K, N", [(131, 881, 512), (1, 9, 7), (5, 1, 64), (300, 1283, 130), (40, 50, 640), (2000, 333, 1280), (64, 5119, 64), (513, 4001, 96)])
def test_prepared_weights_of_any_depth(gpu_device, path, M, K, N, dtype):
    a, b, bias, residual, _ = operands(M, K, N, dtype, gpu_device)
    wide = torch.full((M, K + 3), math.nan, dtype=dtype, device=gpu_device)
    wide[:, 1:1 + K] = a
    pw = PreparedWeight(b)
    for rows in (a, wide[:, 1:1 + K]):
        for act, r in ((None, None), (None, residual), ("gelu", residual), ("silu", None)):
            y = cascaded_lowp_matmul_epilogue(rows, pw, bias=bias, activation=act, residual=r)
            check_forward(y, a, b, bias, act, r, dtype, 0.0, f"{act} {r is not None} {rows.stride(0)}", fused=True)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_what_a_backward_pass_in_16_bits_rounds(gpu_device, path, dtype):
    """z and dz are held in the tensors' type between the kernels, dbias is summed before dz is rounded: bit by bit what the separate steps give."""
    M, K, N = 333, 456, 640
    a, b, bias, _, dy = operands(M, K, N, dtype, gpu_device)
    z = cascaded_lowp_matmul_epilogue(a, b, bias=bias)
    l, code, act = _lib.lib(), {torch.float16: _lib.DT_F16, torch.bfloat16: _lib.DT_BF16}[dtype], _lib.ACT_BY_NAME["gelu"]
    dz, dbias = torch.empty_like(dy), torch.empty_like(bias)
    ws = torch.empty(l.cascmm_epilogue_workspace_bytes(M, N, code), dtype=torch.uint8, device=gpu_device)
    assert l.cascmm_epilogue_backward(dy.data_ptr(), z.data_ptr(), dz.data_ptr(), dbias.data_ptr(), M, N, N, N, N, act, code, ws.data_ptr(), ws.numel(),
                                      torch.cuda.current_stream().cuda_stream) == 0
    want = dy.double() * slope_of(z.double(), "gelu")
    off = dy.double().abs() * 8 * U * (1 + z.double().abs()) + 2 * U * want.abs()
    within(dz, want, off + HALF[dtype] * want.abs() + TINY[dtype], "dz")
    within(dbias, want.sum(0), off.sum(0) + (64 + M // 8) * U * want.abs().sum(0) + HALF[dtype] * want.sum(0).abs() + TINY[dtype], "dbias")
    leaves = [t.clone().requires_grad_() for t in (a, b, bias)]
    da, db, got = torch.autograd.grad(cascaded_lowp_matmul_epilogue(*leaves[:2], bias=leaves[2], activation="gelu"), leaves, dy)
    assert torch.equal(got, dbias)
    assert torch.equal(da, cascaded_lowp_matmul(dz, b.t().contiguous())) and torch.equal(db, cascaded_lowp_matmul(a.t().contiguous(), dz))


@pytest.mark.parametrize("cascade, M, K, N, far", [("fp32", 2, 320, 1280, 1 << 29), ("fp32", 256, 5120, 128, 8_600_000), ("fp32", 512, 64, 1280, 2_200_000),
                                                   ("fp32", 2048, 64, 10240, 2_200_000), ("fp32x3", 400, 640, 5120, 8_600_000), ("fp32x3", 2, 320, 1280, 1 << 29),
                                                   ("fp16", 70, 640, 320, 9_000_000), ("bf16", 300, 640, 2560, 9_000_000)])
def test_z_with_rows_far_apart(gpu_device, cascade, M, K, N, far):
    """z kept in rows further apart than the offsets of a tile's stores, beside results that are not, through the C entry."""
    dtype, options, lost = CASCADES[cascade]
    a, b, bias, residual, _ = operands(M, K, N, dtype, gpu_device)
    code, fmt, terms = {"fp32": (0, 0, 2), "fp32x3": (0, 1, 3), "fp16": (1, 1, 1), "bf16": (2, 0, 1)}[cascade]
    l = _lib.lib()
    need = l.cascmm_workspace_bytes(M, N, K, code, fmt, terms, 0)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=gpu_device)
    z = torch.empty((M - 1) * far + N, dtype=dtype, device=gpu_device).as_strided((M, N), (far, 1))
    z.fill_(math.nan)
    y = torch.full((M, N), math.nan, dtype=dtype, device=gpu_device)
    assert l.cascmm_gemm_epilogue(a.data_ptr(), b.data_ptr(), 0, y.data_ptr(), bias.data_ptr(), residual.data_ptr(), z.data_ptr(), M, N, K, K, N, N, N, far, code, fmt, terms, 0,
                                  _lib.ACT_BY_NAME["silu"], None, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream) == 0
    check_forward(y, a, b, bias, "silu", residual, dtype, lost, "y")
    want, _, stored = z_of(a, b, bias, dtype, lost)
    within(z.contiguous(), want, stored, "z")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("act, broadcast", [(None, False), ("gelu", True), ("silu", False)])
def test_copied_rows_a_block_at_a_time(gpu_device, dtype, act, broadcast):
    """Prepared 16-bit weights on rows that are copied first, in workspaces that hold some of the copies."""
    l, (code, fmt) = _lib.lib(), {torch.float16: (1, 1), torch.bfloat16: (2, 0)}[dtype]
    for M, K, N, shift in ((1000, 283, 64, 0), (777, 129, 211, 1), (300, 128, 320, 1), (65, 1, 8, 0)):
        a, b, bias, residual, _ = operands(M, K, N, dtype, gpu_device)
        pw = PreparedWeight(b)
        wide = torch.full((M, K + 3), math.nan, dtype=dtype, device=gpu_device)
        wide[:, shift:shift + K] = a
        r = residual[0] if broadcast else residual
        row = (2 * K + 127) // 128 * 128
        for held in (1, 40, 256, 300, 600, M):
            room = held * row + 256
            ws = torch.empty(room + 1, dtype=torch.uint8, device=gpu_device)
            ws[room] = 77
            z, y = (torch.full((M + 1, N + 5), math.inf, dtype=dtype, device=gpu_device) for _ in range(2))
            assert l.cascmm_gemm_epilogue(wide[:, shift:].data_ptr(), pw.slots.data_ptr(), 1, y.data_ptr(), bias.data_ptr(), r.data_ptr(), z.data_ptr(), M, N, K, K + 3, N,
                                          N + 5, 0 if broadcast else N, N + 5, code, fmt, 1, 0, _lib.ACT_BY_NAME[act], None, ws.data_ptr(), room,
                                          torch.cuda.current_stream().cuda_stream) == 0
            check_forward(y[:M, :N], a, b, bias, act, r.expand(M, N), dtype, 0.0, f"{M} {K} {N} {held}", fused=True)
            want, _, stored = z_of(a, b, bias, dtype, 0.0)
            within(z[:M, :N], want, stored, "z")
            assert int(ws[room]) == 77
            assert all(bool((t[M] == math.inf).all()) and bool((t[:, N:] == math.inf).all()) for t in (y, z))


def test_prepared_weights_of_any_depth_on_more_rows_than_one_copy_holds(gpu_device, path):
    """Copies of A beyond 2 GiB as a whole: every row is its weights' row, at the ends of blocks too."""
    M, K, N = 1 << 20, 1025, 16
    b = torch.randn(K, N, device=gpu_device).half()
    a = (torch.arange(M, device=gpu_device, dtype=torch.int32) % 7 - 3).half()[:, None].expand(M, K).contiguous()
    y = cascaded_lowp_matmul_epilogue(a, PreparedWeight(b), activation="relu")
    one = cascaded_lowp_matmul_epilogue(a[:7].contiguous(), PreparedWeight(b), activation="relu")
    want = F.relu(a[:7].double() @ b.double())
    for m in range(7):     # (rows of one kind are alike whichever block they are in, up to the order of K products)
        S = a[m].double().abs() @ b.double().abs()
        tol = K * U * S + HALF[torch.float16] * want[m] + TINY[torch.float16]
        assert bool(((y[m::7].double() - want[m]).abs() <= tol).all()) and bool(((one[m].double() - want[m]).abs() <= tol).all())


@pytest.mark.parametrize("dtype", HALF)
def test_slopes_at_infinite_z(gpu_device, path, dtype):
    """Their limits: one and zero; a NaN stays one (of relu, whose slope asks for z <= 0 only, it passes the gradient on)."""
    z = torch.tensor([math.inf, -math.inf, math.nan] * 9, dtype=dtype, device=gpu_device)
    none = torch.zeros(1, 0, dtype=dtype, device=gpu_device), torch.zeros(0, z.numel(), dtype=dtype, device=gpu_device)
    for act in ("relu", "gelu", "gelu_tanh", "silu"):
        leaf = z.clone().requires_grad_()
        (g,) = torch.autograd.grad(cascaded_lowp_matmul_epilogue(*none, bias=leaf, activation=act).sum(), leaf)
        g = g.double().view(9, 3)
        assert bool(((g[:, 0] - 1).abs() <= 8 * U).all()) and bool((g[:, 1].abs() <= 8 * U).all()), act
        assert bool((g[:, 2] == 1).all()) if act == "relu" else bool(g[:, 2].isnan().all()), act


@pytest.mark.parametrize("cascade", CASCADES)
@pytest.mark.parametrize("act", [None, "relu", "gelu", "gelu_tanh", "silu"])
def test_infinities_and_nan_in_gradients_stay_in_their_rows_and_columns(gpu_device, path, cascade, act):
    dtype, options, _ = CASCADES[cascade]
    if cascade == "fp32x3":
        return      # (the scale of an operand is one for all its rows there)
    a, b, bias, residual, dy = operands(140, 136, 72, dtype, gpu_device)

    def grads(a, dy):
        leaves = [t.clone().requires_grad_() for t in (a, b, bias, residual)]
        return torch.autograd.grad(cascaded_lowp_matmul_epilogue(leaves[0], leaves[1], bias=leaves[2], activation=act, residual=leaves[3], **options), leaves, dy)

    a[37] = a[37].abs()
    z = a.double() @ b.double() + bias.double()
    j = int(z[37].argmax())         # (where every activation has a slope)
    assert float(z[37, j]) > 0.5
    clean = grads(a, dy)
    other, column = torch.arange(140, device=gpu_device) != 37, torch.arange(72, device=gpu_device) != j
    for value in (math.inf, -math.inf, math.nan):
        bad = dy.clone()
        bad[37, j] = value
        da, db, dbias, dr = grads(a, bad)
        assert torch.equal(da[other], clean[0][other]) and not bool(da[37].isfinite().any())
        assert torch.equal(db[:, column], clean[1][:, column]) and not bool(db[:, j].isfinite().any())
        assert torch.equal(dbias[column], clean[2][column]) and not bool(dbias[j].isfinite())
        assert torch.equal(dr[other], dy[other]) and torch.equal(dr[37][column], dy[37][column])
    # a NaN in a: its row of z, so of dz where the activation has a slope; all of db's row of that input
    bad = a.clone()
    bad[37, 5] = math.nan
    da, db, dbias, dr = grads(bad, dy)
    assert torch.equal(da[other], clean[0][other]) and torch.equal(dr, dy) and bool(db[5].isnan().all())
    if act in (None, "relu"):
        assert bool(da[37].isfinite().all()) and bool(dbias.isfinite().all())
    else:
        assert bool(da[37].isnan().all()) and bool(dbias.isnan().all()) and bool(db.isnan().all())


def off_dwords(t, how):
    """The same values in rows that start between dwords, or lie too far apart for 32-bit offsets."""
    M, N = t.shape
    if how == "start":          # dense, one element off
        v = torch.empty(M * N + 1, dtype=t.dtype, device=t.device)[1:].view(M, N)
    elif how == "rows":         # odd distances
        v = torch.full((M, N + 3), math.nan, dtype=t.dtype, device=t.device)[:, 2:2 + N]
    else:
        far = 2_200_000
        v = torch.empty((M - 1) * far + N, dtype=t.dtype, device=t.device).as_strided((M, N), (far, 1))
    v.copy_(t)
    return v


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("how", ["start", "rows", "far"])
@pytest.mark.parametrize("M, K, N", [(4, 8, 46), (85, 64, 1000), (300, 640, 320), (700, 72, 1700), (2, 5120, 64)])
def test_rows_off_dwords_are_rounded_once_too(gpu_device, path, dtype, how, M, K, N):
    """z is not rounded on its way to the result, whatever the rows: a residual that takes nearly all of z away shows it."""
    a, b, bias, _, dy = operands(M, K, N, dtype, gpu_device)
    pw = PreparedWeight(b)
    b1 = off_dwords(b.view(1, -1), "start").view(K, N)
    rows = off_dwords(a, how)
    for act in ACTIVATIONS:
        residual = -ACTIVATIONS[act](z_of(a, b, bias, dtype, 0.0)[0]).to(dtype)
        for w in (b, b1, pw):
            y = cascaded_lowp_matmul_epilogue(rows, w, bias=bias, activation=act, residual=residual)
            check_forward(y, a, b, bias, act, residual, dtype, 0.0, f"{act} {type(w).__name__}", fused=True)
        leaves = [t.detach().requires_grad_() for t in (rows, b1, bias, residual)]
        y = cascaded_lowp_matmul_epilogue(leaves[0], leaves[1], bias=leaves[2], activation=act, residual=leaves[3])
        check_forward(y, a, b, bias, act, residual, dtype, 0.0, f"{act} differentiated", fused=True)
        grads = torch.autograd.grad(y, leaves, off_dwords(dy, "rows"))
        check_backward(grads, dy, a, b, bias, act, residual, dtype, 0.0, f"{act}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_same_bits_whatever_the_workspace_has_grown_to(gpu_device, path, dtype):
    # (a workspace of 10 MB by the library's own count, 26 MB of rows)
    a, b, bias, residual, dy = operands(20000, 640, 64, dtype, gpu_device)
    pw, rows, b1 = PreparedWeight(b), off_dwords(a, "rows"), off_dwords(b.view(1, -1), "start").view(640, 64)
    big = torch.zeros(40_000, 1283, dtype=dtype, device=gpu_device), torch.zeros(1283, 64, dtype=dtype, device=gpu_device)

    def calls():
        leaf, wide = rows.detach().requires_grad_(), off_dwords(dy, "rows")
        y = cascaded_lowp_matmul_epilogue(leaf, b1, bias=bias, residual=residual)
        with torch.no_grad():
            return [cascaded_lowp_matmul_epilogue(rows, w, bias=bias, activation="gelu", residual=residual) for w in (b, b1, pw)] + list(torch.autograd.grad(y, leaf, wide))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        before = calls()
        cascaded_lowp_matmul(*big)         # (rows copied first: 100 MB of workspace on this stream)
        after = calls()
        torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(before, after))
