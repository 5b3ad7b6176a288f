"""The norms around a residual add against the formulas in 64 bits.

Tolerances, element by element, from the arithmetic: u = 2^-24 is fp32's half step, half of a type's step its results' rounding.  A lane adds at most ``depth`` numbers one behind the
other (a row's elements over sixteen lanes or more, then the lanes), so a mean is off by depth u mean|v|, and what a norm gives by
e = rstd (depth u mean|v| + 2 u (|v| + |mean|)) + (depth / 2 + 4) u |v hat|, the last term being rstd's.  y is held against the norm of s as it was returned.  Errors go through the
formulas of the backward pass term by term; a sum over rows adds at most ``deep`` numbers one behind the other.
"""
import math

import pytest
import torch

from basedxl_amd import _lib, add_layer_norm, gated_add_norm
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
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
TYPES = list(TINY)


def half_of(dtype):
    return torch.finfo(dtype).eps / 2


def within(got, want, tol, what):
    assert got.shape == want.shape, what
    tol = tol + half_of(got.dtype) * want.abs() * 1.001 + TINY[got.dtype]
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, the worst {float((off / tol).nan_to_num(nan=math.inf).max()):.2f} of the tolerance"


def normed(v, kind, eps):
    """(v hat, its error, 1 / deviation, depth)"""
    depth = -(-v.shape[-1] // 16) + 24
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)
    hat = (v - mean) * rstd
    off = depth * U * v.abs().mean(-1, keepdim=True) if kind == "layer" else 0.0
    return hat, rstd * (off + 2 * U * (v.abs() + mean.abs())) + (depth / 2 + 4) * U * hat.abs(), rstd, depth


def through(q, tolq, hat, e, rstd, depth, kind):
    """A norm's gradient rstd (q - [mean q] - hat mean(q hat)) and its error, q off by tolq, hat by e."""
    m = lambda t: t.mean(-1, keepdim=True)   # noqa: E731
    c1, c2 = (m(q) if kind == "layer" else torch.zeros_like(rstd)), m(q * hat)
    d1 = (depth * U * m(q.abs()) + m(tolq)) if kind == "layer" else 0.0
    d2 = depth * U * m((q * hat).abs()) + m(q.abs() * e + tolq * (hat.abs() + e))
    want = rstd * (q - c1 - hat * c2)
    return want, rstd * (tolq + 4 * U * (q.abs() + c1.abs() + (hat * c2).abs()) + d1 + hat.abs() * d2 + e * c2.abs()) + (depth / 2 + 4) * U * want.abs()


PARTS = ("weight", "bias", "gate", "scale", "post_weight", "post_bias")
# which parameters there are: "c" one row, "s" one for each sample
HOWS = {
    "bare": dict(),
    "affine": dict(weight="c", bias="c", alpha=0.5),
    "gated": dict(weight="c", gate="c", alpha=-1.25),
    "conditioned": dict(weight="s", bias="s", gate="s"),
    "both_norms": dict(weight="c", bias="c", post=True, post_weight="c", gate="c"),
    "everything": dict(weight="c", bias="s", gate="s", scale="s", post=True, post_weight="c", post_bias="c"),
    "scaled": dict(weight="c", scale="c", norm="rms"),
    "rms_both": dict(weight="c", post=True, post_weight="c", gate="s", norm="rms"),
    "rms_bare": dict(post=True, norm="rms"),
    "rms_everything": dict(weight="s", bias="c", gate="c", scale="c", post=True, post_weight="c", post_bias="c", norm="rms"),
}
SIZES = [(1, 1, 1), (1, 3, 2), (2, 2, 7), (2, 1, 1280), (3, 5, 64), (1, 77, 130), (5, 33, 256), (2, 10, 257), (4, 65, 640), (3, 40, 1280), (2, 5, 1537), (1, 4, 2049), (2, 3, 3001),
         (1, 3, 6145), (2, 2, 8193), (50, 3, 96), (1, 3000, 24)]


def make(how, samples, tokens, cols, dtype, wdtype, device, seed):
    gen = torch.Generator().manual_seed(seed)

    def stream():
        return (torch.randn(samples, tokens, cols, generator=gen) * torch.exp(0.3 * torch.randn(cols, generator=gen)) + 0.5 * torch.randn(cols, generator=gen)).to(dtype).to(device)
    t = {"x": stream(), "residual": stream(), "dy": stream(), "ds": stream()}
    for name in PARTS:
        if name in how:
            shape = (samples, 1, cols) if how[name] == "s" else (cols,)
            mean = {"weight": 1.0, "gate": 0.5, "scale": 1.0, "post_weight": 1.0}.get(name, 0.0)
            t[name] = (mean + 0.2 * torch.randn(shape, generator=gen)).to(wdtype).to(device)
    return t


def call(t, how, eps):
    return gated_add_norm(t["x"], t["residual"], t.get("weight"), t.get("bias"), gate=t.get("gate"), residual_scale=t.get("scale", how.get("alpha", 1.0)),
                          post_norm=how.get("post", False), post_weight=t.get("post_weight"), post_bias=t.get("post_bias"), norm=how.get("norm", "layer"), eps=eps)


def check(t, how, eps, y, s, grads, ds_given=True):
    kind = how.get("norm", "layer")
    d = {k: v.detach().double() for k, v in t.items()}
    one = torch.ones_like(d["x"][..., :1])
    w, b, g = d.get("weight", one), d.get("bias", 0 * one), d.get("gate", one)
    a = d.get("scale", one * how.get("alpha", 1.0))
    w1, b1 = d.get("post_weight", one), d.get("post_bias", 0 * one)
    if how.get("post"):
        xhat, e1, rstd1, depth1 = normed(d["x"], kind, eps)
    else:
        xhat, e1 = d["x"], torch.zeros_like(d["x"])
    want = a * d["residual"] + g * (xhat * w1 + b1)
    within(s, want, (g * w1).abs() * e1 + 6 * U * ((a * d["residual"]).abs() + (g * w1 * xhat).abs() + (g * b1).abs()), "s")
    shat, e2, rstd2, depth2 = normed(s.detach().double(), kind, eps)
    within(y, shat * w + b, w.abs() * e2 + 4 * U * ((shat * w).abs() + b.abs()), "y")
    if grads is None:
        return
    dy, ds = d["dy"], d["ds"] if ds_given else torch.zeros_like(d["ds"])
    D, tolD = through(dy * w, U * (dy * w).abs(), shat, e2, rstd2, depth2, kind)
    D, tolD = D + ds, tolD + 2 * U * ((D + ds).abs() + ds.abs())
    within(grads["residual"], a * D, a.abs() * tolD + U * (a * D).abs(), "dresidual")
    q, tolq = D * g * w1, (g * w1).abs() * tolD + 3 * U * (D * g * w1).abs()
    if how.get("post"):
        want, tol = through(q, tolq, xhat, e1, rstd1, depth1, kind)
    else:
        want, tol = q, tolq
    within(grads["x"], want, tol, "dx")
    deep = 64 + d["x"].shape[:-1].numel() // 8

    def summed(name, terms, tols):
        """terms over the rows that share an element"""
        if name not in t:
            return
        over = (lambda v: v.sum(1, keepdim=True)) if t[name].dim() == 3 else (lambda v: v.sum((0, 1)))
        within(grads[name], over(terms), over(tols) + deep * U * over(terms.abs()), "d" + name)
    p, e = xhat * w1, e1 * w1.abs()
    # (of the gate's gradient the two sums are taken apart and put together with their factors)
    summed("gate", D * (p + b1), tolD * (p.abs() + e + b1.abs()) + D.abs() * e + deep * U * D.abs() * (p.abs() + b1.abs()))
    summed("scale", D * d["residual"], tolD * d["residual"].abs())
    summed("post_weight", D * g * xhat, g.abs() * (tolD * (xhat.abs() + e1) + D.abs() * e1) + deep * U * (D * g * xhat).abs())
    summed("post_bias", D * g, g.abs() * tolD + deep * U * (D * g).abs())
    summed("weight", dy * shat, dy.abs() * e2)
    summed("bias", dy, 0 * dy)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", HOWS)
@pytest.mark.parametrize("samples, tokens, cols", SIZES)
def test_forward_and_backward(gpu_device, samples, tokens, cols, name, dtype):
    how, eps = HOWS[name], 1e-3
    for wdtype in {dtype, torch.float32}:
        t = make(how, samples, tokens, cols, dtype, wdtype, gpu_device, samples * 7 + tokens * 3 + cols)
        y, s = call(t, how, eps)
        check(t, how, eps, y, s, None)
        leaves = {k: v.clone().requires_grad_() for k, v in t.items() if k not in ("dy", "ds")}
        y1, s1 = call(leaves, how, eps)
        assert torch.equal(y1, y) and torch.equal(s1, s)
        grads = dict(zip(leaves, torch.autograd.grad((y1, s1), list(leaves.values()), (t["dy"], t["ds"]))))
        check(t, how, eps, y, s, grads)
        assert all(v.dtype == t[k].dtype for k, v in grads.items())


@pytest.mark.parametrize("name", HOWS)
def test_each_gradient_alone(gpu_device, name):
    how = HOWS[name]
    t = make(how, 3, 20, 300, torch.bfloat16, torch.bfloat16, gpu_device, 4)
    names = [k for k in t if k not in ("dy", "ds")]
    leaves = {k: t[k].clone().requires_grad_() for k in names}
    whole = dict(zip(names, torch.autograd.grad(call(leaves, how, 1e-5), list(leaves.values()), (t["dy"], t["ds"]))))
    for k in names:
        args = {n: t[n].clone().requires_grad_(n == k) for n in names}
        assert torch.equal(torch.autograd.grad(call(args, how, 1e-5), args[k], (t["dy"], t["ds"]))[0], whole[k]), k
    # through one result alone
    y, s = call(leaves, how, 1e-5)
    only_y = dict(zip(names, torch.autograd.grad(y, list(leaves.values()), t["dy"])))
    check(t, how, 1e-5, y, s, only_y, ds_given=False)
    y, s = call(leaves, how, 1e-5)
    only_s = torch.autograd.grad(s, [leaves["x"], leaves["residual"]], t["ds"])
    quiet = dict(t, dy=torch.zeros_like(t["dy"]))
    y, s = call(leaves, how, 1e-5)
    both = torch.autograd.grad((y, s), [leaves["x"], leaves["residual"]], (quiet["dy"], t["ds"]))
    assert all(torch.equal(p, q) for p, q in zip(only_s, both))


def test_it_is_add_layer_norm_where_nothing_is_gated(gpu_device):
    t = make(HOWS["affine"], 2, 50, 640, torch.float16, torch.float16, gpu_device, 8)
    y, s = gated_add_norm(t["x"], t["residual"], t["weight"], t["bias"])
    want, total = add_layer_norm(t["x"], t["residual"], t["weight"], t["bias"])
    assert torch.equal(s, total) and float((y.float() - want.float()).abs().max()) <= 2 * half_of(torch.float16) * float(want.abs().max())


@pytest.mark.parametrize("name", ["conditioned", "both_norms", "everything", "rms_everything"])
def test_differences(gpu_device, name):
    """Central differences of the operator itself, in fp32, of two step widths put together so that the third derivative drops out.  A value of the function
    is off by the roundings of its results, at most 16 u of each, and what is left of the expansion by h^4 of its size."""
    how, eps = HOWS[name], 1e-2
    t = make(how, 2, 3, 12, torch.float32, torch.float32, gpu_device, 3)
    names = [k for k in t if k not in ("dy", "ds")]
    leaves = {k: t[k].clone().requires_grad_() for k in names}
    y, s = call(leaves, how, eps)
    grads = dict(zip(names, torch.autograd.grad((y, s), list(leaves.values()), (t["dy"], t["ds"]))))
    f = lambda args: float((call(args, how, eps)[0].double() * t["dy"].double()).sum() + (call(args, how, eps)[1].double() * t["ds"].double()).sum())   # noqa: E731
    size = float(((y.abs() * t["dy"].abs()).sum() + (s.abs() * t["ds"].abs()).sum()).detach())
    for k in names:
        flat = grads[k].flatten()
        for i in {0, flat.numel() // 2, flat.numel() - 1}:
            slopes = []
            for h in (2.0 ** -5, 2.0 ** -6):
                values = []
                for step in (h, -h):
                    args = {n: v.clone() for n, v in t.items()}
                    args[k].view(-1)[i] += step
                    values.append(f(args))
                slopes.append((values[0] - values[1]) / (2 * h))
            difference = (4 * slopes[1] - slopes[0]) / 3
            assert abs(difference - float(flat[i])) <= 2 * 16 * U * size * 2 ** 6 + 2.0 ** -18 * size, (k, i)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [1, 640, 457, 2500, 9000])
def test_strides(gpu_device, cols, dtype):
    how = HOWS["everything"]
    t = make(how, 3, 7, cols, dtype, dtype, gpu_device, cols)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items() if k not in ("dy", "ds")}
    whole = call(t, how, 1e-5)
    grads = torch.autograd.grad(call(leaves, how, 1e-5), list(leaves.values()), (t["dy"], t["ds"]))
    for first in (1, 4):
        wide = {k: torch.zeros(*v.shape[:-1], cols + 9, dtype=v.dtype, device=gpu_device) for k, v in t.items()}
        for k, v in t.items():
            wide[k][..., first:first + cols] = v
        views = {k: v[..., first:first + cols] for k, v in wide.items()}
        assert all(torch.equal(p, q) for p, q in zip(call(views, how, 1e-5), whole))
        again = {k: v.detach().requires_grad_() for k, v in views.items() if k not in ("dy", "ds")}
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(call(again, how, 1e-5), list(again.values()), (views["dy"], views["ds"])), grads))
    # leading axes in another order, two and four axes, one row, expanded operands
    turned = dict(t, x=t["x"].transpose(0, 1).contiguous().transpose(0, 1))
    assert all(torch.equal(p, q) for p, q in zip(call(turned, how, 1e-5), whole))
    four = {k: v.unsqueeze(1) if v.dim() == 3 else v for k, v in t.items()}
    assert all(torch.equal(p.squeeze(1), q) for p, q in zip(call(four, how, 1e-5), whole))
    c = lambda v: v[0] if v.dim() == 3 else v   # noqa: E731  (one sample's tokens; its parameters as one row)
    single = {k: c(v) for k, v in t.items()}
    assert all(torch.equal(p, q[0]) for p, q in zip(call(single, how, 1e-5), whole))
    still = dict(t, residual=t["residual"][:1, :1].expand(3, 7, cols))
    assert all(torch.equal(p, q) for p, q in zip(call(still, how, 1e-5), call(dict(t, residual=still["residual"].contiguous()), how, 1e-5)))
    # a row each: gates of the shape of x
    rows = {k: (v.reshape(21, cols) if v.shape == t["x"].shape else v.expand(3, 7, cols).reshape(21, cols).contiguous() if v.dim() == 3 else v) for k, v in t.items()}
    assert all(torch.equal(p.view(3, 7, cols), q) for p, q in zip(call(rows, how, 1e-5), whole))
    leaves = {k: v.clone().requires_grad_() for k, v in rows.items() if k not in ("dy", "ds")}
    mine = torch.autograd.grad(call(leaves, how, 1e-5), list(leaves.values()), (rows["dy"], rows["ds"]))
    assert torch.equal(mine[0].view(3, 7, cols), grads[0]) and mine[list(leaves).index("gate")].shape == (21, cols)


@pytest.mark.parametrize("name", ["conditioned", "both_norms", "everything", "rms_everything"])
@pytest.mark.parametrize("samples, tokens, cols", [(3, 7, 5), (4, 64, 640), (8, 33, 1000), (2, 9, 7000)])
def test_gradients_of_rows_that_are_copied(gpu_device, samples, tokens, cols, name):
    """x and the residual in orders that no rows describe (a channel-first image's tokens, samples behind tokens, one row for all tokens): the gradients of copies made beforehand.
    A workspace of five rows of sums for each of up to 256 groups fits in what such a copy occupies."""
    how = HOWS[name]
    t = make(how, samples, tokens, cols, torch.float32, torch.float32, gpu_device, cols)
    forms = {"columns": lambda v: v.transpose(1, 2).contiguous().transpose(1, 2), "turned": lambda v: v.transpose(0, 1).contiguous().transpose(0, 1),
             "expanded": lambda v: v[:, :1].expand(v.shape)}
    for of_x, of_residual in (("columns", "turned"), ("turned", "expanded"), ("expanded", "columns")):
        given = dict(t, x=forms[of_x](t["x"]), residual=forms[of_residual](t["residual"]))
        grads = []
        for contiguous in (True, False):
            leaves = {k: (v.contiguous() if contiguous else v).detach().requires_grad_() for k, v in given.items() if k not in ("dy", "ds")}
            for _ in range(3):      # (again on memory that the last one gave back)
                grads.append(torch.autograd.grad(call(leaves, how, 1e-5), list(leaves.values()), (t["dy"], t["ds"])))
        for other in grads[1:]:
            assert all(torch.equal(p, q) for p, q in zip(other, grads[0])), (of_x, of_residual)


@pytest.mark.parametrize("name", ["conditioned", "everything"])
@pytest.mark.parametrize("samples, tokens, cols, dtype", [(65537, 1, 3, torch.float32), (70001, 2, 7, torch.bfloat16), (5000, 3, 6147, torch.float16)])
def test_more_groups_than_a_grid_has_rows(gpu_device, samples, tokens, cols, dtype, name):
    """Rows that no registers hold, with parameters for each of many samples."""
    how = HOWS[name]
    t = make(how, samples, tokens, cols, dtype, dtype, gpu_device, cols)
    leaves = {k: v.clone().requires_grad_() for k, v in t.items() if k not in ("dy", "ds")}
    y, s = call(leaves, how, 1e-3)
    grads = dict(zip(leaves, torch.autograd.grad((y, s), list(leaves.values()), (t["dy"], t["ds"]))))
    check(t, how, 1e-3, y, s, grads)


@pytest.mark.parametrize("cols", [5, 640, 7000])
@pytest.mark.parametrize("name", ["conditioned", "both_norms", "everything"])
def test_gradients_of_the_streams_alone(gpu_device, cols, name):
    """Parameters for every token that are not trained: the same gradients of x and the residual, without memory for sums that nobody wants."""
    how, rows = HOWS[name], 2000
    t = make(how, rows, 1, cols, torch.bfloat16, torch.bfloat16, gpu_device, cols)
    both = []
    for trained in (True, False):
        leaves = {k: v.clone().requires_grad_(trained or k in ("x", "residual")) for k, v in t.items() if k not in ("dy", "ds")}
        out = call(leaves, how, 1e-5)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        requested = lambda which: torch.cuda.memory_stats()["requested_bytes.all." + which]   # noqa: E731  (what was asked for: a block may be up to 1 MiB larger)
        before = requested("current")
        both.append(torch.autograd.grad(out, (leaves["x"], leaves["residual"]), (t["dy"], t["ds"])))
        if not trained:
            assert requested("peak") - before == 2 * rows * cols * 2 + 16      # (the two results, and the least workspace)
    assert all(torch.equal(p, q) for p, q in zip(*both))


@pytest.mark.parametrize("samples", [1, 4])
@pytest.mark.parametrize("wdtype", [torch.bfloat16, torch.float32])
def test_parts_of_a_conditioning(gpu_device, samples, wdtype):
    """Parameters of a sample as parts of one wide row, of one sample too: the same as parameters of their own, without a copy, and so are the gradients."""
    gen = torch.Generator(device=gpu_device).manual_seed(samples)
    draw = lambda *shape: torch.randn(*shape, generator=gen, device=gpu_device)   # noqa: E731
    x, residual, dy, ds = (draw(samples, 9, 200).bfloat16() for _ in range(4))
    wide = draw(samples, 1, 3 * 200).to(wdtype).requires_grad_()
    how = dict(norm="rms", eps=1e-5)
    weight, bias, gate = wide.chunk(3, dim=-1)
    native = _lib.native().gated_add_norm(x, residual, weight, bias, gate, 1.0, None, None, False, 1, 1e-5)
    assert native is not None
    y, s = gated_add_norm(x, residual, weight, bias, gate=gate, **how)
    own = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_() for t in (weight, bias, gate)]
    y2, s2 = gated_add_norm(x, residual, own[0], own[1], gate=own[2], **how)
    assert all(torch.equal(p, q) for p, q in ((native[0], y2), (native[1], s2), (y, y2), (s, s2)))
    whole = torch.autograd.grad((y, s), wide, (dy, ds))[0]
    parts = torch.autograd.grad((y2, s2), own, (dy, ds))
    assert torch.equal(whole, torch.cat(parts, -1)) and all(g.shape == (samples, 1, 200) for g in parts)
    with torch.no_grad():
        # one gate for all samples, spread over them: read as it would be written out
        spread = gate[:1].expand(samples, 1, 200)
        assert all(torch.equal(p, q) for p, q in zip(gated_add_norm(x, residual, gate=spread, **how), gated_add_norm(x, residual, gate=spread.contiguous(), **how)))


def test_scalars_and_mixed_types(gpu_device):
    t = make(HOWS["affine"], 2, 30, 128, torch.bfloat16, torch.float32, gpu_device, 6)
    gate, scale = torch.tensor(0.75, device=gpu_device, requires_grad=True), torch.tensor(1.5, device=gpu_device, requires_grad=True)
    weight = t["weight"].bfloat16().requires_grad_()
    y, s = gated_add_norm(t["x"], t["residual"], weight, t["bias"], gate=gate, residual_scale=scale)
    y2, s2 = gated_add_norm(t["x"], t["residual"], weight.float(), t["bias"], gate=torch.full((128,), 0.75, device=gpu_device), residual_scale=1.5)
    assert torch.equal(y, y2) and torch.equal(s, s2)
    gg, gs, gw = torch.autograd.grad((y, s), (gate, scale, weight), (t["dy"], t["ds"]))
    assert gg.shape == () and gs.shape == () and gw.dtype == torch.bfloat16
    rows = {k: v.clone().requires_grad_() for k, v in dict(gate=torch.full((128,), 0.75, device=gpu_device), scale=torch.full((128,), 1.5, device=gpu_device)).items()}
    out = gated_add_norm(t["x"], t["residual"], weight.float(), t["bias"], gate=rows["gate"], residual_scale=rows["scale"])
    fg, fs = torch.autograd.grad(out, list(rows.values()), (t["dy"], t["ds"]))
    assert abs(float(gg) - float(fg.double().sum())) <= 130 * U * float(fg.abs().sum()) and abs(float(gs) - float(fs.double().sum())) <= 130 * U * float(fs.abs().sum())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [5, 640, 1001, 9000])
def test_rows_that_are_not_finite_stay_alone(gpu_device, cols, dtype):
    how = HOWS["both_norms"]
    t = make(how, 1, 12, cols, dtype, dtype, gpu_device, 2)
    clean = call(t, how, 1e-5)
    t["x"][0, 3, cols - 1], t["residual"][0, 7, 0], t["x"][0, 9] = math.inf, math.nan, 0.0
    y, s = call(t, how, 1e-5)
    touched = torch.tensor([3, 7, 9], device=gpu_device)
    keep = torch.ones(12, dtype=torch.bool, device=gpu_device)
    keep[touched] = False
    assert torch.equal(y[0][keep], clean[0][0][keep]) and torch.equal(s[0][keep], clean[1][0][keep])
    assert bool(y[0, 3].isnan().all() and y[0, 7].isnan().all() and y[0, 9].isfinite().all())


def test_ordinary_calls_are_one_native_function(gpu_device):
    x, c, g = torch.ones(3, 4, 64, device=gpu_device), torch.ones(64, device=gpu_device), torch.ones(3, 1, 64, device=gpu_device)
    f = _lib.native().gated_add_norm
    for args in ((x, x, c, c, g, 1.0, None, None, False, 0, 1e-5), (x, x, None, None, None, g, c, c, True, 1, 1e-5), (x.clone().requires_grad_(), x, g, g, c, 0.5, None, None, False, 1, 0.0)):
        y, s = f(*args)
        assert y.shape == s.shape == x.shape
    for args in ((x, x, c, c, g[:2], 1.0, None, None, False, 0, 1e-5), (x, x, c.half(), c, g, 1.0, None, None, False, 0, 1e-5), (x, x, c, c, g, 1.0, c, None, False, 0, 1e-5),
                 (x, x, c, c, g, 1.0, None, None, False, 2, 1e-5), (x, x, c, c, g, 1.0, None, None, False, 0, -1.0), (x, x, c, c, g, math.inf, None, None, False, 0, 1e-5),
                 (x, x, c, c, g, 1.0, g, None, True, 0, 1e-5), (x, x[:2], c, c, g, 1.0, None, None, False, 0, 1e-5), (x, x, c, c, g, 1.0, None, None, False, 0)):
        assert f(*args) is None


def test_nothing_to_do(gpu_device):
    for samples, tokens, cols in ((0, 4, 8), (3, 0, 8), (3, 4, 0)):
        how = HOWS["everything"]
        t = make(how, samples, tokens, cols, torch.float32, torch.float32, gpu_device, 1)
        leaves = {k: v.clone().requires_grad_() for k, v in t.items() if k not in ("dy", "ds")}
        y, s = call(leaves, how, 1e-5)
        assert y.shape == s.shape == t["x"].shape
        grads = torch.autograd.grad((y, s), list(leaves.values()), (t["dy"], t["ds"]))
        assert all(g.shape == leaves[k].shape and not g.any() for g, k in zip(grads, leaves))


def test_refusals(gpu_device):
    x = torch.zeros(3, 4, 8, device=gpu_device)
    w = torch.ones(8, device=gpu_device)
    for change, error, text in (
            (dict(residual=x[:2]), ValueError, "residual"), (dict(residual=x.half()), ValueError, "residual"), (dict(weight=w[:7]), ValueError, "weight"),
            (dict(weight=w.half()), TypeError, "weight"), (dict(weight=w.cpu()), ValueError, "weight is on"), (dict(gate=torch.ones(3, 8, device=gpu_device)), ValueError, "gate"),
            (dict(gate=torch.ones(3, 4, 8, device=gpu_device)), ValueError, "gate"), (dict(gate=torch.ones(2, 1, 8, device=gpu_device)), ValueError, "gate"),
            (dict(post_weight=torch.ones(3, 1, 8, device=gpu_device), post_norm=True), ValueError, "post_weight"), (dict(post_weight=w), ValueError, "post_norm"),
            (dict(norm="batch"), ValueError, "norm"), (dict(eps=-1.0), ValueError, "eps"), (dict(eps=math.nan), ValueError, "eps"), (dict(residual_scale=math.inf), ValueError, "finite"),
            (dict(residual_scale=w[:3]), ValueError, "residual_scale")):
        args = dict(residual=x, weight=w)
        args.update(change)
        residual, weight = args.pop("residual"), args.pop("weight")
        with pytest.raises(error, match=text):
            gated_add_norm(x, residual, weight, **args)
    with pytest.raises(TypeError, match="dtype"):
        gated_add_norm(x.double(), x.double())
    a = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(gated_add_norm(a, x, w, gate=w)[0].sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            gated_add_norm(torch.autograd.forward_ad.make_dual(x, x), x)


def test_recorded_replayed_and_on_other_streams(gpu_device):
    """Two recorded training passes whose workspaces are their own, replayed side by side between eager work."""
    how = HOWS["everything"]
    t = make(how, 4, 100, 640, torch.bfloat16, torch.bfloat16, gpu_device, 5)
    inputs = {k: v for k, v in t.items() if k not in ("dy", "ds")}

    def step():
        leaves = {k: v.detach().requires_grad_() for k, v in inputs.items()}
        y, s = call(leaves, how, 1e-5)
        return [y.detach(), s.detach(), *torch.autograd.grad((y, s), list(leaves.values()), (t["dy"], t["ds"]))]
    graphs = []
    for _ in range(2):
        side = side_streams()[0]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    gen = torch.Generator(device=gpu_device).manual_seed(1)
    streams = side_streams()
    for _ in range(4):
        for v in t.values():
            v.normal_(generator=gen)
        eager = step()
        for (graph, _), stream in zip(graphs, streams):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(p, q) for p, q in zip(out, eager))
