"""Layer norm and residual add with layer norm against the formulas in 64 bits.

Tolerances, element by element, from the arithmetic: u = 2^-24 is fp32's half step, ``half`` that of the result's type.  A lane adds at most
D numbers one behind the other (a row's elements over 64 lanes or more, then the lanes), so the mean is off by D u mean|x|, and xhat by
e = rstd (D u mean|x| + 2 u (|x| + |mean|)) + (D / 2 + 4) u |xhat|: the last term is rstd's, half of the variance's relative error.
"""
import math

import pytest
import torch

from basedxl_amd import _lib, add_layer_norm, layer_norm

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
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}   # (results below the normal numbers: half a step there)
TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
         (torch.bfloat16, torch.float32)]
SIZES = [(1, 1), (1, 2), (3, 7), (5, 64), (2, 1280), (9, 512), (77, 640), (333, 457), (260, 1024), (4, 1536), (5, 1537), (6, 2048), (3, 2049), (3, 3001), (2, 4096),
         (2, 6144), (3, 8192), (3, 8193), (2, 20001), (5000, 8), (2049, 96), (130, 65), (1000, 128), (77, 130), (40, 256), (41, 257)]


def rows_of(gen, rows, cols, dtype, device, spread=1.0, mean=0.5):
    return (torch.randn(rows, cols, generator=gen) * spread + mean * torch.randn(cols, generator=gen)).to(dtype).to(device)


def within(got, want, tol, what):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, the worst {float((off / tol).nan_to_num(nan=math.inf).max()):.2f} of the tolerance"


def parts_of(s, weight, bias, eps):
    """The formulas' pieces in 64 bits and the error of xhat."""
    s = s.double()
    cols = s.shape[-1]
    w = torch.ones(cols, dtype=torch.float64, device=s.device) if weight is None else weight.double()
    b = torch.zeros(cols, dtype=torch.float64, device=s.device) if bias is None else bias.double()
    mean = s.mean(-1, keepdim=True)
    var = ((s - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xhat = (s - mean) * rstd
    depth = -(-cols // 64) + 16
    e = rstd * (depth * U * s.abs().mean(-1, keepdim=True) + 2 * U * (s.abs() + mean.abs())) + (depth / 2 + 4) * U * xhat.abs()
    return w, b, rstd, xhat, e, depth


def check_forward(y, s, weight, bias, eps, what):
    w, b, _, xhat, e, _ = parts_of(s, weight, bias, eps)
    want = xhat * w + b
    within(y, want, HALF[y.dtype] * want.abs() + TINY[y.dtype] + w.abs() * e + 4 * U * ((xhat * w).abs() + b.abs()), what)


def check_backward(dx, dw, db, dy, ds, s, weight, bias, eps, what):
    w, b, rstd, xhat, e, depth = parts_of(s, weight, bias, eps)
    dy = dy.double()
    g = dy * w
    c1, c2 = g.mean(-1, keepdim=True), (g * xhat).mean(-1, keepdim=True)
    want = rstd * (g - c1 - xhat * c2)
    d1 = depth * U * g.abs().mean(-1, keepdim=True)
    d2 = depth * U * (g * xhat).abs().mean(-1, keepdim=True) + (g.abs() * e).mean(-1, keepdim=True)
    tol = rstd * (4 * U * (g.abs() + c1.abs() + (xhat * c2).abs()) + d1 + xhat.abs() * d2 + e * c2.abs()) + (depth / 2 + 4) * U * want.abs()
    if ds is not None:
        want = want + ds.double()
        tol = tol + 2 * U * (want.abs() + ds.double().abs())
    if dx is not None:
        within(dx, want, tol + HALF[dx.dtype] * want.abs() + TINY[dx.dtype], what + " dx")
    deep = 64 + s.shape[0] // 16     # (numbers added one behind the other over the rows)
    if dw is not None:
        want = (dy * xhat).sum(0)
        within(dw, want, HALF[dw.dtype] * want.abs() + TINY[dw.dtype] + deep * U * (dy * xhat).abs().sum(0) + (dy.abs() * e).sum(0), what + " dweight")
    if db is not None:
        want = dy.sum(0)
        within(db, want, HALF[db.dtype] * want.abs() + TINY[db.dtype] + deep * U * dy.abs().sum(0), what + " dbias")


@pytest.mark.parametrize("dtype, wdtype", TYPES)
@pytest.mark.parametrize("rows, cols", SIZES)
def test_forward_and_backward(gpu_device, path, rows, cols, dtype, wdtype):
    gen = torch.Generator().manual_seed(rows * 131 + cols)
    x, r, dy, ds = (rows_of(gen, rows, cols, dtype, gpu_device) for _ in range(4))
    w = (1 + 0.2 * torch.randn(cols, generator=gen)).to(wdtype).to(gpu_device)
    b = (0.2 * torch.randn(cols, generator=gen)).to(wdtype).to(gpu_device)
    check_forward(layer_norm(x, w, b), x, w, b, 1e-5, "forward")
    y, s = add_layer_norm(x, r, w, b, eps=1e-3)
    assert torch.equal(s, (x.float() + r.float()).to(dtype))
    check_forward(y, s, w, b, 1e-3, "sum's forward")
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y1 = layer_norm(*leaves)
    assert torch.equal(y1, layer_norm(x, w, b))
    check_backward(*torch.autograd.grad(y1, leaves, dy), dy, None, x, w, b, 1e-5, "backward")
    leaves = [t.clone().requires_grad_() for t in (x, r, w, b)]
    y2, s2 = add_layer_norm(*leaves, eps=1e-3)
    dx, dr, dw, db = torch.autograd.grad((y2, s2), leaves, (dy, ds))
    assert torch.equal(dx, dr)
    check_backward(dx, dw, db, dy, ds, s, w, b, 1e-3, "sum's backward")


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("cols", [640, 457, 2500, 9000])
def test_strided_rows_leave_their_surroundings_alone(gpu_device, path, cols, dtype):
    gen = torch.Generator().manual_seed(cols)
    wide = rows_of(gen, 23, cols + 37, dtype, gpu_device)
    for first in (0, 1, 3, 8):
        x = wide[:, first:first + cols]
        assert torch.equal(layer_norm(x), layer_norm(x.contiguous()))
        a = x.detach().requires_grad_()
        dy = wide[:, 37 - first:37 - first + cols]
        (g,) = torch.autograd.grad(layer_norm(a), a, dy)
        c = x.contiguous().requires_grad_()
        assert torch.equal(g, torch.autograd.grad(layer_norm(c), c, dy.contiguous())[0])
    # other orders and dimensions: transposed, expanded, three-dimensional, one row
    t = rows_of(gen, cols, 6, dtype, gpu_device).t()
    assert torch.equal(layer_norm(t), layer_norm(t.contiguous()))
    e = wide[:1, :cols].expand(5, cols)
    assert torch.equal(layer_norm(e), layer_norm(e.contiguous()))
    d = wide[:20, :cols].reshape(4, 5, cols)
    assert torch.equal(layer_norm(d).reshape(20, cols), layer_norm(d.reshape(20, cols)))
    assert torch.equal(layer_norm(wide[0, :cols]), layer_norm(wide[:1, :cols])[0])
    # the C entry with results inside larger ones: what lies behind the rows and around the columns stays
    l, code = _lib.lib(), {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    out = torch.full((25, cols + 11), 7.0, dtype=dtype, device=gpu_device)
    x = wide[:, :cols]
    stream = torch.cuda.current_stream().cuda_stream
    assert l.cascmm_layer_norm(x.data_ptr(), None, None, None, out[1:, 5:].data_ptr(), None, None, None, 23, cols, wide.stride(0), 0, out.stride(0), 0,
                               1e-5, code, code, stream) == 0
    assert torch.equal(out[1:24, 5:5 + cols], layer_norm(x))
    out[1:24, 5:5 + cols] = 7.0
    assert bool((out == 7.0).all())


def test_optional_weight_and_bias(gpu_device, path):
    gen = torch.Generator().manual_seed(3)
    x, dy = rows_of(gen, 50, 320, torch.float32, gpu_device), rows_of(gen, 50, 320, torch.float32, gpu_device)
    w, b = torch.randn(320, generator=gen).to(gpu_device), torch.randn(320, generator=gen).to(gpu_device)
    for weight, bias in ((None, None), (w, None), (None, b)):
        check_forward(layer_norm(x, weight, bias), x, weight, bias, 1e-5, "forward")
        leaves = [t.clone().requires_grad_() for t in (x, weight, bias) if t is not None]
        it = iter(leaves[1:])
        y = layer_norm(leaves[0], None if weight is None else next(it), None if bias is None else next(it))
        grads = list(torch.autograd.grad(y, leaves, dy))
        dx = grads.pop(0)
        check_backward(dx, grads.pop(0) if weight is not None else None, grads.pop(0) if bias is not None else None, dy, None, x, weight, bias, 1e-5, "backward")
    # gradients of some inputs only
    for keep in ((True, False, False), (False, True, False), (False, False, True), (False, True, True)):
        leaves = [t.clone().requires_grad_(k) for t, k in zip((x, w, b), keep)]
        layer_norm(*leaves).backward(dy)
        check_backward(leaves[0].grad, leaves[1].grad, leaves[2].grad, dy, None, x, w, b, 1e-5, f"some {keep}")
        assert [t.grad is not None for t in leaves] == list(keep)


def test_one_result_of_the_sum_only(gpu_device, path):
    gen = torch.Generator().manual_seed(4)
    x, r, d = (rows_of(gen, 30, 200, torch.float32, gpu_device).requires_grad_() for _ in range(3))
    d = d.detach()
    y, s = add_layer_norm(x, r)
    gx, gr = torch.autograd.grad(s, (x, r), d, retain_graph=True)
    assert torch.equal(gx, d) and torch.equal(gr, d)
    (gx,) = torch.autograd.grad(y, x, d)
    check_backward(gx, None, None, d, None, s.detach(), None, None, 1e-5, "norm only")
    # accumulated into leaves: two gradients that are one tensor do not become one .grad
    x2, r2 = x.detach().clone().requires_grad_(), r.detach().clone().requires_grad_()
    for _ in range(2):
        y, s = add_layer_norm(x2, r2)
        (y * d).sum().backward()
    assert x2.grad.data_ptr() != r2.grad.data_ptr() and torch.equal(x2.grad, r2.grad)
    assert torch.equal(x2.grad, 2 * gx)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("cols", [1, 40, 1280, 4100, 10000])
def test_rows_of_one_value_and_rows_far_from_zero(gpu_device, cols, dtype):
    x = torch.full((3, cols), 3.25, dtype=dtype, device=gpu_device)
    x[1] = 0
    b = torch.linspace(-1, 1, cols).to(dtype).to(gpu_device)
    assert torch.equal(layer_norm(x, None, b), b.expand(3, cols))       # (every difference from the mean is zero: 3.25 cols is exact)
    a = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(layer_norm(a), a, torch.ones_like(x))
    assert bool((g.abs() <= 320 * 64 * U).all())                       # (rstd = eps^-1/2 = 316 times 1 - 1)
    if dtype == torch.float32:
        gen = torch.Generator().manual_seed(cols)
        far = rows_of(gen, 7, cols, dtype, gpu_device, spread=3.0, mean=0.0) + 1.0e4
        check_forward(layer_norm(far), far, None, None, 1e-5, "far from zero")


def test_infinities_and_nan_stay_in_their_rows(gpu_device):
    gen = torch.Generator().manual_seed(8)
    for cols in (300, 3000, 9000):
        x = rows_of(gen, 9, cols, torch.float32, gpu_device)
        clean = layer_norm(x)
        for value in (math.inf, -math.inf, math.nan):
            bad = x.clone()
            bad[4, 17] = value
            y = layer_norm(bad)
            assert bool(y[4].isnan().all())
            assert torch.equal(y[:4], clean[:4]) and torch.equal(y[5:], clean[5:])


def test_empty_tensors(gpu_device, path):
    for shape in ((0, 64), (4, 0), (2, 0, 8)):
        x = torch.empty(shape, device=gpu_device, requires_grad=True)
        w = torch.ones(shape[-1], device=gpu_device, requires_grad=True)
        y = layer_norm(x, w)
        assert y.shape == x.shape
        dx, dw = torch.autograd.grad(y, (x, w), torch.empty(shape, device=gpu_device))
        assert dx.shape == x.shape and bool((dw == 0).all())
        assert all(t.shape == x.shape for t in add_layer_norm(x, x, w))


def test_the_same_call_gives_the_same_bits(gpu_device):
    gen = torch.Generator().manual_seed(12)
    x, dy = rows_of(gen, 4099, 330, torch.bfloat16, gpu_device), rows_of(gen, 4099, 330, torch.bfloat16, gpu_device)
    w = torch.ones(330, device=gpu_device, requires_grad=True)
    a = x.requires_grad_()
    first = torch.autograd.grad(layer_norm(a, w), (a, w), dy)
    for _ in range(5):
        again = torch.autograd.grad(layer_norm(a, w), (a, w), dy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_against_differences(gpu_device):
    """The gradient along a direction against central differences of the formula in 64 bits."""
    gen = torch.Generator().manual_seed(21)
    x, r, dy, ds = (torch.randn(6, 50, generator=gen) for _ in range(4))
    w, b = torch.randn(50, generator=gen), torch.randn(50, generator=gen)

    def loss(x, r, w, b):
        s = x + r
        c = s - s.mean(-1, keepdim=True)
        y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-5) * w + b
        return (y * dy.double()).sum() + (s * ds.double()).sum()

    leaves = [t.to(gpu_device).requires_grad_() for t in (x, r, w, b)]
    grads = torch.autograd.grad(add_layer_norm(*leaves), leaves, (dy.to(gpu_device), ds.to(gpu_device)))
    at = [t.double() for t in (x, r, w, b)]
    for i, grad in enumerate(grads):
        direction = torch.randn(at[i].shape, generator=gen).double()
        h = 1e-5
        plus, minus = [t.clone() for t in at], [t.clone() for t in at]
        plus[i] += h * direction
        minus[i] -= h * direction
        slope = (loss(*plus) - loss(*minus)) / (2 * h)
        # (differences: h^2 times third derivatives and rounding / h, 1e-8 of the terms; the kernel: fp32, a few hundred half steps of them)
        scale = (grad.cpu().double() * direction).abs().sum()
        assert abs(slope - (grad.cpu().double() * direction).sum()) <= 500 * U * scale + 1e-8 * scale


def test_other_streams_and_recorded_calls(gpu_device, path):
    gen = torch.Generator().manual_seed(30)
    x, dy = rows_of(gen, 700, 640, torch.float16, gpu_device), rows_of(gen, 700, 640, torch.float16, gpu_device)
    w = torch.ones(640, device=gpu_device, dtype=torch.float16)
    want = layer_norm(x, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = layer_norm(x, w)
    side.synchronize()
    assert torch.equal(got, want)

    def step(x, w, dy):
        y = layer_norm(x, w)
        return (y, *torch.autograd.grad(y, (x, w), dy))

    # two recorded steps, replayed in turn between eager ones
    steps = []
    for seed in (1, 2):
        g = torch.Generator().manual_seed(seed)
        sx, sw, sdy = x.clone().requires_grad_(), w.clone().requires_grad_(), dy.clone()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            step(sx, sw, sdy)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(sx, sw, sdy)
        steps.append((graph, sx, sw, sdy, outs, g))
    for _ in range(4):
        for graph, sx, sw, sdy, outs, g in steps:
            with torch.no_grad():
                sx.copy_(torch.randn(700, 640, generator=g))
                sdy.copy_(torch.randn(700, 640, generator=g))
            graph.replay()
            ex, ew = sx.detach().clone().requires_grad_(), sw.detach().clone().requires_grad_()
            want = step(ex, ew, sdy)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(outs, want))


def test_offsets_beyond_32_bits(gpu_device):
    """Rows far apart: the last one starts 5 GB behind the first."""
    x = torch.empty(3, 1_300_000_000, dtype=torch.bfloat16, device=gpu_device)[:, 7:7 + 1280]
    x.copy_(torch.randn(3, 1280, generator=torch.Generator().manual_seed(2)))
    assert torch.equal(layer_norm(x), layer_norm(x.contiguous()))


def test_refusals(gpu_device, path):
    x = torch.zeros(4, 8, device=gpu_device)
    ok = torch.zeros(8, device=gpu_device)
    for bad, error in ((dict(weight=ok[:7]), ValueError), (dict(bias=torch.zeros(8, 1, device=gpu_device)), ValueError), (dict(weight=ok.cpu()), ValueError),
                       (dict(weight=ok.half()), TypeError), (dict(weight=ok.double()), TypeError), (dict(eps=-1.0), ValueError), (dict(eps=math.nan), ValueError)):
        with pytest.raises(error):
            layer_norm(x, **bad)
    with pytest.raises(TypeError):
        layer_norm(x.half(), ok.half(), ok)
    with pytest.raises(TypeError):
        layer_norm(x.double())
    with pytest.raises(ValueError):
        layer_norm(x[0, 0])
    for r in (x[:3], x.half(), x.cpu(), x[:1]):
        with pytest.raises(ValueError):
            add_layer_norm(x, r)
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(layer_norm(leaf).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_the_host_extension_takes_ordinary_calls(gpu_device):
    native = _lib.native()
    x, w = torch.randn(3, 5, 64, device=gpu_device), torch.ones(64, device=gpu_device)
    y = native.layer_norm(x, w, None, 1e-5)
    assert torch.equal(y, layer_norm(x, w))
    assert native.layer_norm(x.clone().requires_grad_(), w, None, 1e-5).requires_grad
    y, s = native.add_layer_norm(x, x, w, w, 1e-5)
    assert torch.equal(s, 2 * x) and torch.equal(y, add_layer_norm(x, x, w, w)[0])
    # what is left to the Python code, which refuses or copies
    for args in ((x.cpu(), w, None, 1e-5), (x, w[:7], None, 1e-5), (x, w.half(), None, 1e-5), (x, w, w.half(), 1e-5), (x, w, None, -1.0), (x, w, None, math.nan),
                 (x, w, None, "a"), (x.double(), None, None, 1e-5), (x[:0], w, None, 1e-5), (x.transpose(0, 1), w, None, 1e-5), (x, w, None), (x, 3, None, 1e-5)):
        assert native.layer_norm(*args) is None
    assert native.add_layer_norm(x, x[:2], w, None, 1e-5) is None and native.add_layer_norm(x, x.half(), w, None, 1e-5) is None


def test_forward_mode_tangents_are_refused(gpu_device, path):
    from torch.autograd import forward_ad
    x, w = torch.randn(4, 8, device=gpu_device), torch.ones(8, device=gpu_device)
    with forward_ad.dual_level():
        for call in ((forward_ad.make_dual(x, x), w, w), (x, forward_ad.make_dual(w, w), w), (x, w, forward_ad.make_dual(w, w))):
            with pytest.raises(NotImplementedError):
                layer_norm(*call)
        with pytest.raises(NotImplementedError):
            add_layer_norm(x, forward_ad.make_dual(x, x), w, w)
        assert torch.equal(layer_norm(x, w, w), layer_norm(x, w, w))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [2, 5, 40, 200, 457, 640, 1281, 2049, 8200, 8201, 9003])
def test_gradients_of_rows_of_one_large_value(gpu_device, path, cols, dtype):
    """Rows of 2^112 with eps = 1e-12: the mean is exact and xhat zero, while mean times rstd is beyond fp32."""
    gen = torch.Generator().manual_seed(cols)
    x = torch.full((70, cols), 2.0 ** 112, dtype=dtype, device=gpu_device)
    dy, w, b = rows_of(gen, 70, cols, dtype, gpu_device), rows_of(gen, 1, cols, dtype, gpu_device)[0], rows_of(gen, 1, cols, dtype, gpu_device)[0]
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = layer_norm(*leaves, eps=1e-12)
    assert torch.equal(y, b.expand(70, cols))
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    g = dy.double() * w.double()
    c1 = g.mean(-1, keepdim=True)
    want = 1e6 * (g - c1)
    # (g and its difference are rounded, the mean is a sum of cols / 64 + 16 numbers and two roundings, rstd and the product with it some more)
    tol = 1e6 * U * (4 * (g.abs() + c1.abs()) + (cols / 64 + 18) * g.abs().mean(-1, keepdim=True)) + 8 * U * want.abs()
    within(dx, want, tol + HALF[dtype] * want.abs() + TINY[dtype], "dx")
    assert bool((dw == 0).all())
    want = dy.double().sum(0)
    within(db, want, HALF[dtype] * want.abs() + 70 * U * dy.double().abs().sum(0) + TINY[dtype], "dbias")


@pytest.mark.parametrize("dtype, wdtype", TYPES)
@pytest.mark.parametrize("rows, cols", [(70000, 96), (20000, 457), (3000, 2500), (777, 9001), (50000, 3)])
def test_gradients_of_weight_and_bias_alone(gpu_device, path, rows, cols, dtype, wdtype):
    """No gradient of x: a thread a column sums over many rows."""
    gen = torch.Generator().manual_seed(rows + cols)
    x, dy = rows_of(gen, rows, cols, dtype, gpu_device), rows_of(gen, rows, cols, dtype, gpu_device)
    w, b = ((1 + 0.2 * torch.randn(cols, generator=gen)).to(wdtype).to(gpu_device).requires_grad_() for _ in range(2))
    dw, db = torch.autograd.grad(layer_norm(x, w, b), (w, b), dy)
    _, _, _, xhat, e, _ = parts_of(x, w.detach(), b.detach(), 1e-5)
    d, deep = dy.double(), 64 + rows // 16
    for got, want, off, what in ((dw, (d * xhat).sum(0), deep * U * (d * xhat).abs().sum(0) + (d.abs() * e).sum(0), "dweight"), (db, d.sum(0), deep * U * d.abs().sum(0), "dbias")):
        tol = HALF[wdtype] * want.abs() + TINY[wdtype] + off
        # (a sum that rounds beyond the type's largest number is infinite: a computed one is within tol of it, so where |want| + tol is larger than that number it may be)
        beyond = (got == want.sign() * math.inf) & (want.abs() + tol > torch.finfo(wdtype).max)
        within(got[~beyond], want[~beyond], tol[~beyond], what)
    (dw1,) = torch.autograd.grad(layer_norm(x, w, b.detach()), w, dy)
    (db1,) = torch.autograd.grad(layer_norm(x, w.detach(), b), b, dy)
    assert torch.equal(dw1, dw) and torch.equal(db1, db)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("cols", [3, 40, 457, 1280, 2500, 9001])
def test_gradients_of_rows_with_infinities_and_nan(gpu_device, path, cols, dtype):
    """They reach dx of their own rows, dbias of their own columns, and dweight where xhat or dy is one."""
    gen = torch.Generator().manual_seed(cols)
    rows = 300
    x, r, dy, ds = (rows_of(gen, rows, cols, dtype, gpu_device) for _ in range(4))
    w, b = rows_of(gen, 1, cols, dtype, gpu_device)[0], rows_of(gen, 1, cols, dtype, gpu_device)[0]

    def grads(x, r, dy, ds):
        leaves = [t.clone().requires_grad_() for t in (x, r, w, b)]
        return torch.autograd.grad(add_layer_norm(*leaves), leaves, (dy, ds))

    clean = grads(x, r, dy, ds)
    last = cols - 1
    for value in (math.inf, -math.inf, math.nan):
        # in dy: its row of dx, its column of the sums
        bad = dy.clone()
        bad[17, last] = value
        dx, dr, dw, db = grads(x, r, bad, ds)
        other, column = torch.arange(rows, device=gpu_device) != 17, torch.arange(cols, device=gpu_device) != last
        assert torch.equal(dx[other], clean[0][other]) and torch.equal(dr[other], clean[0][other]) and not bool(dx[17].isfinite().any())
        assert torch.equal(dw[column], clean[2][column]) and torch.equal(db[column], clean[3][column])
        assert not bool(dw[last].isfinite()) and (bool(db[last].isnan()) if math.isnan(value) else float(db[last]) == value)
        # in ds: one element of dx
        bad = ds.clone()
        bad[17, last] = value
        dx, _, dw, db = grads(x, r, dy, bad)
        assert not bool(dx[17, last].isfinite())
        dx[17, last] = clean[0][17, last]
        assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), (clean[0], clean[2], clean[3])))
        # in the sum: its row of dx, all of dweight, nothing of dbias
        bad = x.clone()
        bad[17, last] = value
        dx, _, dw, db = grads(bad, r, dy, ds)
        assert torch.equal(dx[other], clean[0][other]) and bool(dx[17].isnan().all()) and bool(dw.isnan().all()) and torch.equal(db, clean[3])
