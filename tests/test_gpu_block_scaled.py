"""Block-scaled 8-bit products against the format's definition and the formulas in 64 bits.

The rounding is exact arithmetic up to one rounding: bytes and scales are compared as they are.  Products: let t_k be the products of the rounded operands (exact in fp32).
fp32 results are sums in fp32: off by at most K 2^-24 sum|t|.  16-bit results come from an instruction that aligns neighbouring products at the largest of them and cuts what is
2^-15 of it: sixteen of them lose at most 16 * 2^-15 of their largest, and the sums of such groups, aligned at 2^-18 of the largest of an instruction's 64, as much again at most; the
result's rounding comes on top.  These bounds are far off for ordinary sums, so over many results the root mean square is held to what was measured of the instruction, 1.5e-5 of that of
the results (5e-5 allowed), beside that of a rounding.
"""
import math

import pytest
import torch

from basedxl_amd import _lib, BlockScaledWeight, block_scaled_matmul
from basedxl_amd.block_scaled import _round
from tests.side_streams import side_streams

pytestmark = pytest.mark.gpu

@pytest.fixture(params=["native", "python"], autouse=True)
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


def half_of(dtype):
    return torch.finfo(dtype).eps / 2


def held(x, how):
    """(rounded values, exponents of the scales), both 64-bit and of the shape of ``x``: the definition.  ``how``: "rows" (blocks along a row), "columns", "square"."""
    x = x.detach().cpu().double()
    if how == "columns":
        v, e = held(x.t(), "rows")
        return v.t(), e.t()
    rows, cols = x.shape
    finite = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs()
    e = torch.zeros_like(x)
    for c in range(0, cols, 128):
        for r in range(0, rows, 128 if how == "square" else rows or 1):
            part = finite[r:r + 128, c:c + 128] if how == "square" else finite[:, c:c + 128]
            most = part.amax() if how == "square" else part.amax(1, keepdim=True)
            k = torch.full_like(most, -127.0)
            for bit in (128.0, 64.0, 32.0, 16.0, 8.0, 4.0, 2.0, 1.0):      # (the smallest k with most <= 448 * 2^k, by halving)
                k = torch.where(most > 448 * torch.exp2(k + bit - 1), k + bit, k)
            k = torch.where(most > 0, k, torch.zeros_like(k))
            if how == "square":
                e[r:r + 128, c:c + 128] = k
            else:
                e[:, c:c + 128] = k.expand_as(part)
    v = x * torch.exp2(-e)
    top = torch.floor(torch.log2(torch.where(v.abs() > 0, v.abs(), torch.ones_like(v))))
    step = torch.exp2(top.clamp(min=-6) - 3)
    return torch.where(torch.isfinite(x), torch.round(v / step) * step * torch.exp2(e), torch.full_like(x, math.nan)), e


def seen(pair, rows, k):
    """The same of what the kernel wrote: values and exponents [rows, k], 64-bit on the host; and what lies behind k."""
    values, scales = pair
    exponents = scales.permute(1, 0, 2).reshape(rows, -1)[:, :values.shape[1] // 128].cpu().double() - 127
    exponents = exponents.repeat_interleave(128, 1)
    wide = values.cpu().view(torch.float8_e4m3fn).double() * torch.exp2(exponents)
    return wide[:, :k], exponents[:, :k], values[:, k:]


def same(got, want):
    return torch.equal(got.nan_to_num(nan=1e300), want.nan_to_num(nan=1e300)) and torch.equal(got.isnan(), want.isnan())


def stream(gen, rows, cols, dtype, scale=1.0):
    return (torch.randn(rows, cols, generator=gen) * torch.exp(torch.randn(cols, generator=gen)) * scale).to(dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 128), (3, 129), (127, 7), (128, 128), (129, 640), (200, 513), (5, 1030), (700, 40)])
def test_rounding(gpu_device, rows, cols, dtype):
    gen = torch.Generator().manual_seed(rows * 1031 + cols)
    x = stream(gen, rows, cols, dtype)
    if rows > 2 and cols > 5:
        x[1], x[:, 3] = 0.0, x[:, 3] * 0
        x[0, 0], x[2, 4], x[rows - 1, cols - 1] = math.inf, math.nan, -math.inf
    d = x.to(gpu_device)
    for square in (False, True):
        q, qt, total = _round(d, square, True, True, True)
        for pair, how, t in ((q, "rows", False), (qt, "columns", True)):
            v, e = held(x, "square" if square else how)
            v, e = (v.t(), e.t()) if t else (v, e)
            got, exps, behind = seen(pair, *v.shape)
            assert same(got, v), (square, how)
            assert torch.equal(exps, e), (square, how)
            assert not behind.any()
        want = x.double().sum(0)
        tol = half_of(dtype) * want.abs() + TINY[dtype] + (16 + rows // 128) * U * x.double().abs().sum(0)
        assert bool((((total.cpu().double() - want).abs() <= tol) | ~torch.isfinite(want)).all()) and torch.equal(total.cpu().isfinite(), torch.isfinite(want))
        # (one of them alone, and from rows inside larger ones, off 16 bytes)
        wide = torch.zeros(rows + 2, cols + 5, dtype=dtype, device=gpu_device)
        wide[1:-1, 3:-2] = d
        for along, across in ((True, False), (False, True)):
            one, other, _ = _round(wide[1:-1, 3:-2], square, along, across)
            mine, whole = (one, q) if along else (other, qt)
            assert torch.equal(mine[0], whole[0]) and torch.equal(seen(mine, mine[0].shape[0], 1)[1], seen(whole, mine[0].shape[0], 1)[1])


def test_rounding_at_every_border(gpu_device):
    """Every value of the format, the middles between neighbours and what lies next to them, at scales from the smallest to the largest."""
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    grid = torch.unique(codes[torch.isfinite(codes)])
    middles = (grid[1:] + grid[:-1]) / 2
    v = torch.cat([grid, middles, torch.nextafter(middles, torch.tensor(1e9)), torch.nextafter(middles, torch.tensor(-1e9))])
    v = torch.cat([v, torch.zeros(-len(v) % 127)]).view(-1, 127)
    v = torch.cat([torch.full((len(v), 1), 448.0), v], 1)                                # (every block has scale one)
    for e in (-140, -127, -126, -60, -1, 0, 1, 7, 60, 119):
        x = torch.ldexp(v, torch.tensor(e))
        got, exps, _ = seen(_round(x.to(gpu_device), False, True, False)[0], *v.shape)
        want, we = held(x, "rows")
        assert same(got, want) and torch.equal(exps, we) and bool((we == max(e, -127)).all())
    # the largest element at the border between two scales
    tops = torch.tensor([448.0, 448.00003, 447.99997, 224.0, 224.00002, 3.4028234e38, 1.17549435e-38, 1e-45, 0.0]).view(-1, 1) * torch.ones(1, 4)
    got, exps, _ = seen(_round(tops.to(gpu_device), False, True, False)[0], 9, 4)
    want, we = held(tops, "rows")
    assert same(got, want) and torch.equal(exps, we) and we[:5, 0].tolist() == [0, 1, 0, -1, 0] and we[8, 0] == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rounding_of_every_pattern(gpu_device, dtype):
    """All numbers of a 16-bit type, each in a block whose largest element is one of their own size or larger, along rows and along columns, by tiles and by the product's own rounding."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    order = torch.argsort(x.float().abs().nan_to_num(posinf=0.0, nan=0.0))
    for spread in (1, 37, 4099):
        v = x[order][torch.arange(65536) * spread % 65536].view(512, 128)
        d = v.to(gpu_device)
        q, qt, _ = _round(d, False, True, True)
        for pair, how, turn in ((q, "rows", False), (qt, "columns", True)):
            want, we = held(v, how)
            got, exps, _ = seen(pair, *(want.t() if turn else want).shape)
            assert same(got, want.t() if turn else want) and torch.equal(exps, we.t() if turn else we)
        eye = torch.eye(128, dtype=dtype, device=gpu_device)      # (held exactly: the product with it is the rounded block; what is not finite spoils its row, a sum of one)
        clean = v.clone()
        clean[~clean.isfinite()] = 0
        for r in range(0, 512, 16):
            got = block_scaled_matmul(clean[r:r + 16].to(gpu_device), eye)
            assert same(got.cpu().double(), held(clean[r:r + 16], "rows")[0].to(dtype).double())


def check_product(got, a, b, bias, what):
    """``a`` [M, K], ``b`` [K, N]: rounded operands in 64 bits."""
    M, K = a.shape
    want = a @ b + (0 if bias is None else bias.detach().cpu().double())
    size = a.abs() @ b.abs()
    if got.dtype == torch.float32:
        # (the 16-bit instruction takes rounded elements below its normal numbers as zeros: each loses less than 2^-126 of what it is multiplied with)
        tiny = lambda t: torch.where(t.abs() < 2.0 ** -126, 2.0 ** -126, 0.0).to(t)   # noqa: E731
        tol = (K + 2) * U * (size + want.abs()) + (lost := tiny(a) @ b.abs() + a.abs() @ tiny(b))
    else:
        pad = torch.nn.functional.pad
        an, bn = pad(a.abs(), (0, -K % 64)), pad(b.abs(), (0, 0, 0, -K % 64))
        groups = torch.zeros_like(want)
        for k in range(0, an.shape[1], 16):
            groups += torch.stack([an[:, k + i:k + i + 1] * bn[k + i] for i in range(16)]).amax(0)
        tol = 2 * 16 * 2.0 ** -15 * groups + (K / 32 + 8) * U * size
    tol = tol + half_of(got.dtype) * want.abs() * 1.001 + TINY[got.dtype] + 2.0 ** -126 * (K + 1)
    off = (got.detach().cpu().double() - want).abs()
    assert got.shape == want.shape and bool((off <= tol).all()), f"{what}: worst {float((off / tol).max())}"
    if want.numel() >= 1000:
        rms = lambda t: float(t.pow(2).mean().sqrt())   # noqa: E731
        most = 1e-6 if got.dtype == torch.float32 else 5e-5 + 0.75 * half_of(got.dtype)
        assert rms(off) <= most * rms(want) + (rms(lost) if got.dtype == torch.float32 else 0), f"{what}: rms {rms(off) / rms(want)}"


SIZES = [(1, 1, 1), (1, 5120, 130), (16, 2049, 47), (5, 4096, 16), (2, 128, 64), (3, 127, 129), (17, 130, 5), (64, 640, 128), (127, 384, 255), (129, 1000, 131), (260, 513, 320), (300, 1280, 640)]


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M, K, N", SIZES)
def test_product_and_gradients(gpu_device, M, K, N, dtype):
    gen = torch.Generator().manual_seed(M * 7 + K * 3 + N)
    a, b = stream(gen, M, K, dtype), stream(gen, K, N, dtype, 0.05)
    bias, dy = (0.1 * torch.randn(N, generator=gen)).to(dtype), stream(gen, M, N, dtype, 0.01)
    da, db, dbias, ddy = (t.to(gpu_device) for t in (a, b, bias, dy))
    ha, hb = held(a, "rows")[0], held(b, "square")[0]
    weight = BlockScaledWeight(db)
    assert torch.equal(weight.dequantized().cpu().double(), hb)
    y = block_scaled_matmul(da, db, bias=dbias)
    check_product(y, ha, hb, bias, "y")
    check_product(block_scaled_matmul(da, db), ha, hb, None, "y without bias")
    assert torch.equal(y, block_scaled_matmul(da, weight, bias=dbias))
    turned = db.t().contiguous().t()
    assert torch.equal(y, block_scaled_matmul(da, turned, bias=dbias)) and torch.equal(BlockScaledWeight(turned).values, weight.values)
    for right in (db, turned):
        leaves = [t.clone(memory_format=torch.preserve_format).requires_grad_() for t in (da, right, dbias)]
        out = block_scaled_matmul(leaves[0], leaves[1], bias=leaves[2])
        assert torch.equal(out, y)
        ga, gb, gbias = torch.autograd.grad(out, leaves, ddy)
        check_product(ga, held(dy, "rows")[0], hb.t(), None, "da")
        check_product(gb, held(a, "columns")[0].t(), held(dy, "columns")[0], None, "db")
        want = dy.double().sum(0)
        assert bool(((gbias.cpu().double() - want).abs() <= half_of(dtype) * want.abs() + TINY[dtype] + (16 + M // 128) * U * dy.double().abs().sum(0)).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("K, N", [(100, 4100), (2200, 45), (2200, 4104), (1024, 4096), (128, 5000)])
def test_few_rows(gpu_device, K, N, dtype):
    """Every number of rows that has a kernel of its own, from rows inside larger ones: a row's results do not depend on the others, whatever those hold."""
    gen = torch.Generator(device=gpu_device).manual_seed(K + N)
    wide = torch.randn(18, K + 9, generator=gen, device=gpu_device).to(dtype)
    b, bias = torch.randn(K, N, generator=gen, device=gpu_device).to(dtype), torch.randn(N, generator=gen, device=gpu_device).to(dtype)
    weight = BlockScaledWeight(b)
    x = wide[1:17, 3:K + 3]
    each = torch.cat([block_scaled_matmul(x[m:m + 1], weight, bias=bias) for m in range(16)])
    check_product(each, seen(_round(x.contiguous(), False, True, False)[0], 16, K)[0], weight.dequantized().cpu().double(), bias, "rows")
    x[2, K - 1] = math.nan
    for m in range(1, 17):
        y = block_scaled_matmul(x[:m], weight, bias=bias)
        keep = [r for r in range(m) if r != 2]
        assert torch.equal(y[keep], each[keep]) and (m < 3 or bool(y[2].isnan().all()))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("M, K, N", [(65, 2500, 70), (400, 700, 129), (300, 2500, 700), (500, 260, 1300), (520, 1100, 5130), (1030, 5000, 1290), (2100, 257, 2570), (4100, 600, 2500), (3900, 1300, 5000), (4900, 1300, 4700)])
def test_every_tile(gpu_device, M, K, N, dtype):
    """Sizes that the rule gives to each of its tiles, with rows, columns and k past their edges."""
    gen = torch.Generator(device=gpu_device).manual_seed(M)
    a, b = (torch.randn(M, K, generator=gen, device=gpu_device) * 3).to(dtype), torch.randn(K, N, generator=gen, device=gpu_device).to(dtype)
    bias = torch.randn(N, generator=gen, device=gpu_device).to(dtype)
    weight = BlockScaledWeight(b)
    y = block_scaled_matmul(a, weight, bias=bias)
    rows = sorted({0, 1, 31, 32, 63, 64, 127, 128, 129, 255, 256, 257, M // 2, M - 65, M - 2, M - 1} & set(range(M)))
    pick = torch.tensor(rows, device=gpu_device)
    wide = seen(_round(a[pick].contiguous(), False, True, False)[0], len(rows), K)[0]
    check_product(y[pick], wide, weight.dequantized().cpu().double(), bias, "rows")
    want = seen(_round(a, False, True, False)[0], M, K)[0].float().to(gpu_device) @ weight.dequantized()
    assert bool(((y.float() - want - bias.float()).abs() <= 2 * half_of(dtype) * want.abs() + 2e-3 * want.pow(2).mean().sqrt()).all())


def test_each_gradient_alone_and_other_shapes(gpu_device):
    gen = torch.Generator().manual_seed(5)
    a, b, bias, dy = stream(gen, 60, 200, torch.bfloat16), stream(gen, 200, 90, torch.bfloat16), stream(gen, 1, 90, torch.bfloat16)[0], stream(gen, 60, 90, torch.bfloat16)
    a, b, bias, dy = (t.to(gpu_device) for t in (a, b, bias, dy))
    leaves = [t.clone().requires_grad_() for t in (a, b, bias)]
    whole = torch.autograd.grad(block_scaled_matmul(leaves[0], leaves[1], bias=leaves[2]), leaves, dy)
    for i in range(3):
        args = [t.clone().requires_grad_(k == i) for k, t in enumerate((a, b, bias))]
        assert torch.equal(torch.autograd.grad(block_scaled_matmul(args[0], args[1], bias=args[2]), args[i], dy)[0], whole[i])
    y = block_scaled_matmul(a, b, bias=bias)
    assert torch.equal(block_scaled_matmul(a.view(3, 4, 5, 200), b, bias=bias).view(60, 90), y)
    assert torch.equal(block_scaled_matmul(a[7], b, bias=bias), y[7])
    wide = torch.zeros(60, 411, dtype=torch.bfloat16, device=gpu_device)
    wide[:, 11:211] = a
    assert torch.equal(block_scaled_matmul(wide[:, 11:211], b, bias=bias), y)
    assert torch.equal(block_scaled_matmul(a.t().contiguous().t(), b, bias=bias), y)
    assert torch.equal(block_scaled_matmul(a[:1].expand(9, 200), b), block_scaled_matmul(a[:1], b).expand(9, 90))
    x = a.view(3, 20, 200).clone().requires_grad_()
    (g,) = torch.autograd.grad(block_scaled_matmul(x, b), x, dy.view(3, 20, 90))
    assert torch.equal(g.view(60, 200), whole[0])
    (g,) = torch.autograd.grad(block_scaled_matmul(x, b).sum(), x)                         # (a gradient of the result that is expanded)
    assert torch.equal(g.view(60, 200), torch.autograd.grad(block_scaled_matmul(leaves[0], b), leaves[0], torch.ones_like(dy))[0])


def test_differences(gpu_device):
    """Small whole numbers are held exactly, so differences of the function along them are its gradient, exactly."""
    gen = torch.Generator().manual_seed(3)
    a, b, dy = (torch.randint(-7, 8, s, generator=gen).float().to(gpu_device) for s in ((5, 150), (150, 9), (5, 9)))
    bias = torch.zeros(9, device=gpu_device)
    for dtype in HALF:
        leaves = [t.to(dtype).requires_grad_() for t in (a, b, bias)]
        f = lambda *args: (block_scaled_matmul(args[0].to(dtype), args[1].to(dtype), bias=args[2].to(dtype)).double() * dy.double()).sum()   # noqa: E731
        grads = torch.autograd.grad(block_scaled_matmul(leaves[0], leaves[1], bias=leaves[2]), leaves, dy.to(dtype))
        for which, (r, c) in ((0, (0, 0)), (0, (4, 149)), (0, (2, 128)), (1, (0, 3)), (1, (127, 8)), (1, (149, 0)), (2, (4, None))):
            step = [a.clone(), b.clone(), bias.clone()]
            at = (r,) if c is None else (r, c)
            step[which][at] += 1
            up = f(*step)
            step[which][at] -= 2
            difference = float((up - f(*step)).detach()) / 2
            # (16-bit results of these sums are rounded: each of the results that changed by half a step)
            most = float(block_scaled_matmul(a, b).detach().abs().max() + 7) * 7 * 9 * half_of(dtype) if dtype != torch.float32 else 0.0
            assert abs(difference - float(grads[which][at])) <= most + half_of(dtype) * abs(difference), (dtype, which, at)


@pytest.mark.parametrize("dtype", HALF)
def test_values_that_are_not_finite_stay_where_they_are(gpu_device, dtype):
    gen = torch.Generator().manual_seed(9)
    a, b = stream(gen, 40, 300, dtype), stream(gen, 300, 140, dtype)
    clean = block_scaled_matmul(a.to(gpu_device), b.to(gpu_device))
    a[3, 299], a[17, 0], b[5, 139] = math.inf, math.nan, -math.inf
    y = block_scaled_matmul(a.to(gpu_device), b.to(gpu_device))
    want = torch.zeros(40, 140, dtype=torch.bool)
    want[3], want[17], want[:, 139] = True, True, True
    assert torch.equal(y.isnan().cpu(), want)
    untouched = ~want
    untouched[:, 128:] = False                                                             # (their block's scale may have been set by the element that is gone)
    assert torch.equal(y.cpu()[untouched], clean.cpu()[untouched])
    zero = torch.zeros(40, 300, dtype=dtype, device=gpu_device)
    assert not block_scaled_matmul(zero, clean.new_ones(300, 140)).any()


@pytest.mark.parametrize("ea, eb", [(100, -100), (-100, 90), (-140, 100), (60, 60), (-60, -60), (110, -120)])
def test_scales_far_apart(gpu_device, ea, eb):
    gen = torch.Generator().manual_seed(1)
    a, b = torch.randn(33, 260, generator=gen), torch.randn(260, 70, generator=gen)
    a, b = torch.ldexp(a, torch.tensor(ea)), torch.ldexp(b, torch.tensor(eb))
    check_product(block_scaled_matmul(a.to(gpu_device), b.to(gpu_device)), held(a, "rows")[0], held(b, "square")[0], None, "fp32")
    a16, b16 = a.bfloat16(), b.bfloat16()
    check_product(block_scaled_matmul(a16.to(gpu_device), b16.to(gpu_device)), held(a16, "rows")[0], held(b16, "square")[0], None, "bf16")


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("K", [16, 128, 300, 5000])
def test_large_products_that_cancel(gpu_device, K, dtype):
    """Two products of the largest size in every few neighbours, of which nothing is left: what small ones add up to is good to 2^-10 of the large ones in 16 bits, and exact in fp32."""
    gen = torch.Generator().manual_seed(K)
    a, b = torch.randint(1, 8, (5, K), generator=gen) * 2.0 ** -6, torch.randint(-7, 8, (K, 9), generator=gen) * 2.0 ** -3
    for at in range(0, K - 8, 37):
        a[:, at], a[:, at + 5] = 448.0, 448.0
        b[at], b[at + 5] = 1.0, -1.0
    a, b = a.to(dtype), b.to(dtype)
    ha, hb = held(a, "rows")[0], held(b, "square")[0]
    assert torch.equal(ha, a.double()) and torch.equal(hb, b.double())         # (whole numbers of up to three bits: held as they are)
    y = block_scaled_matmul(a.to(gpu_device), b.to(gpu_device))
    check_product(y, ha, hb, None, "y")
    if dtype == torch.float32:
        assert torch.equal(y.cpu().double(), ha @ hb)                          # (multiples of 2^-9, and sums of less than 2^15)


@pytest.mark.parametrize("dtype", HALF)
def test_the_largest_numbers(gpu_device, dtype):
    """The type's lowest value, as a mask has it: a finite number like others in 16 bits; in fp32, where it rounds to -2^128, infinite, and it alone."""
    gen = torch.Generator().manual_seed(4)
    a, b = stream(gen, 12, 260, dtype), (0.02 * torch.randn(260, 70, generator=gen)).to(dtype)
    b[7, 5] = 0.0
    clean = block_scaled_matmul(a.to(gpu_device), b.to(gpu_device))
    a[3, 7], a[6, 7], a[6, 200] = torch.finfo(dtype).min, 0.96 * torch.finfo(dtype).max, -0.9 * torch.finfo(dtype).max
    y = block_scaled_matmul(a.to(gpu_device), b.to(gpu_device))
    rest = [r for r in range(12) if r not in (3, 6)]
    assert torch.equal(y[rest], clean[rest])
    ha, hb = held(a, "rows")[0], held(b, "square")[0]
    if dtype == torch.float32:
        row, zero = y[3].cpu().double(), hb[7] == 0
        assert ha[3, 7] == -2.0 ** 128 and bool(row[zero].isnan().all()) and torch.equal(row[~zero], -math.inf * hb[7][~zero])
        ha, y = ha[[r for r in range(12) if r != 3]], y[[r for r in range(12) if r != 3]]
    check_product(y, ha, hb, None, "y")


def test_ordinary_calls_are_one_native_function(gpu_device):
    x, w, b = (torch.ones(s, device=gpu_device, dtype=torch.bfloat16) for s in ((4, 20, 64), (64, 32), (32,)))
    held = BlockScaledWeight(w)
    f = _lib.native().block_scaled
    for args in ((x, w, None, 0, 0, 0, b), (x, w.t().contiguous().t(), None, 0, 0, 0, None), (x, held.values, held.scales, 64, 32, _lib.DT_BF16, b), (x.clone().requires_grad_(), w, None, 0, 0, 0, b)):
        assert f(*args).shape == (4, 20, 32)
    for args in ((x, w.half(), None, 0, 0, 0, b), (x, w, None, 0, 0, 0, b[:31]), (x, held.values, held.scales, 63, 32, _lib.DT_BF16, b), (x, held.values, held.scales, 64, 33, _lib.DT_BF16, None),
                 (x, held.values[:1], held.scales, 64, 32, _lib.DT_BF16, b), (x, held.values, held.scales, 64, 32, _lib.DT_F16, b), (x.cpu(), w, None, 0, 0, 0, b), (x, w, None, 0, 0, 0), (x[:0], w, None, 0, 0, 0, b)):
        assert f(*args) is None


def test_nothing_to_do(gpu_device):
    e = lambda *s: torch.zeros(*s, device=gpu_device, requires_grad=True)   # noqa: E731
    for M, K, N in ((0, 8, 5), (4, 0, 5), (4, 8, 0), (0, 0, 0)):
        a, b, bias = e(M, K), e(K, N), torch.full((N,), 3.0, device=gpu_device, requires_grad=True)
        y = block_scaled_matmul(a, b, bias=bias)
        assert y.shape == (M, N) and bool((y == 3).all())
        with torch.no_grad():
            assert torch.equal(y, block_scaled_matmul(a, b, bias=bias)) and torch.equal(y, block_scaled_matmul(a, BlockScaledWeight(b), bias=bias))
        ga, gb, gbias = torch.autograd.grad(y, (a, b, bias), torch.ones_like(y))
        assert ga.shape == a.shape and gb.shape == b.shape and not ga.any() and not gb.any() and bool((gbias == M).all())


def test_refusals(gpu_device):
    x = torch.zeros(4, 8, device=gpu_device)
    w = torch.zeros(8, 6, device=gpu_device)
    for f, error, text in ((lambda: block_scaled_matmul(x, w.half()), TypeError, "but b"), (lambda: block_scaled_matmul(x, w.t()), ValueError, "columns"),
                           (lambda: block_scaled_matmul(x, w[None]), ValueError, "2-D"), (lambda: block_scaled_matmul(x.double(), w.double()), TypeError, "dtype"),
                           (lambda: block_scaled_matmul(x, w.cpu()), RuntimeError, "AMD GPU"), (lambda: block_scaled_matmul(x, w, bias=x[0]), ValueError, "bias"),
                           (lambda: block_scaled_matmul(x, w, bias=w[0].half()), ValueError, "bias"), (lambda: block_scaled_matmul(x[0, 0], w), ValueError, "dimension"),
                           (lambda: block_scaled_matmul(x.half(), BlockScaledWeight(w)), TypeError, "but b"), (lambda: BlockScaledWeight(x[0]), ValueError, "2-D"),
                           (lambda: block_scaled_matmul(x.requires_grad_(), BlockScaledWeight(w)), RuntimeError, "weight itself")):
        with pytest.raises(error, match=text):
            f()
    a = torch.ones(4, 8, device=gpu_device, requires_grad=True)
    (g,) = torch.autograd.grad(block_scaled_matmul(a, w).sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(torch.ones(4, 8, device=gpu_device), torch.ones(4, 8, device=gpu_device))
        with pytest.raises(NotImplementedError):
            block_scaled_matmul(dual, w)


def test_recorded_replayed_and_on_other_streams(gpu_device):
    gen = torch.Generator(device=gpu_device).manual_seed(2)
    a, b = torch.randn(150, 700, device=gpu_device, generator=gen).bfloat16(), torch.randn(700, 333, device=gpu_device, generator=gen).bfloat16()
    weight = BlockScaledWeight(b)
    graphs = []
    for right in (b, weight):
        block_scaled_matmul(a, right)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = block_scaled_matmul(a, right)
        graphs.append((graph, y, right))
    side = side_streams()[0]
    for _ in range(4):
        a.normal_(generator=gen)
        eager = [block_scaled_matmul(a, right) for _, _, right in graphs]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[0][0].replay()
            other = block_scaled_matmul(a, weight)
        graphs[1][0].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, e) for (_, y, _), e in zip(graphs, eager)) and torch.equal(other, eager[1])
