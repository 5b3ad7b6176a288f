"""The gradients' norm and clipping against the formulas in 64 bits.

Tolerances: the sums are fp64, so the norm is off by its rounding to fp32, u = 2^-24 of it (and 2^-40 for 2^-53 times any number of elements here); a
result by the factor's rounding and the product's, u each, and the rounding to its type.
"""
import math

import pytest
import torch

from basedxl_amd import _lib, clip_grad_norm_, clip_gradients, gradient_norm
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
KINDS = [1.0, 2.0, math.inf]
LISTS = {
    "one": [(1,)],
    "short": [(3,), (7,), (1,), (5, 3), (8,), (9,)],
    "with_empty": [(0,), (17,), (4, 0), (33,), (0,)],
    "all_empty": [(0,), (0, 5)],
    "chunk_edges": [(4095,), (4096,), (4097,), (8192,), (4096 * 3 + 1,)],
    "many": [(1 + i % 37,) for i in range(301)],
    "chunks_of_other_sizes": [(4096 * 2100 + 5,), (77,), (4096 * 300,)],
    "more_parts_than_merged": [(1 + i % 9,) for i in range(2700)],
    "large": [(4097, 8195), (129,), (1000, 1000)],
}


def make(shapes, dtypes, device, seed=0, scale=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return [(torch.randn(s, generator=gen, device=device) * scale).to(dtypes[i % len(dtypes)]) for i, s in enumerate(shapes)]


def norm_of(gradients, kind):
    flat = torch.cat([g.double().flatten() for g in gradients])
    return torch.linalg.vector_norm(flat, kind) if flat.numel() else flat.new_zeros(())


def check_norm(got, want):
    assert got.dtype == torch.float32 and got.dim() == 0
    assert abs(float(got) - float(want)) <= float(want) * U * (1 + 2.0 ** -15) + 2.0 ** -149


def check_scaled(got, gradient, want_norm, max_norm):
    factor = min(1.0, max_norm / (float(want_norm) + 1e-6))
    want = gradient.double() * factor
    tol = want.abs() * ((HALF[got.dtype] + 2 * U) * (1 + 2.0 ** -8)) + TINY[got.dtype]
    assert got.shape == gradient.shape and bool(((got.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.float16,), (torch.bfloat16,), (torch.bfloat16, torch.float32, torch.float16)])
@pytest.mark.parametrize("name", LISTS)
def test_norm_and_clipping(gpu_device, name, dtypes, kind):
    gradients = make(LISTS[name], dtypes, gpu_device)
    want = norm_of(gradients, kind)
    check_norm(gradient_norm(gradients, kind), want)
    for max_norm in (0.37 * float(want), 2 * float(want) + 1, 0.0):
        same, wide = [torch.full_like(g, 7.0) for g in gradients], [torch.full_like(g, 7.0, dtype=torch.float32) for g in gradients]
        kept = [g.clone() for g in gradients]
        for out in (same, wide):
            check_norm(clip_gradients(gradients, max_norm, norm_type=kind, out=out), want)
            for o, g, k in zip(out, gradients, kept):
                check_scaled(o, g, want, max_norm)
                assert torch.equal(g, k)
        check_norm(clip_gradients(kept, max_norm, norm_type=kind), want)
        for k, o in zip(kept, same):
            assert torch.equal(k, o)


@pytest.mark.parametrize("scale", [1e30, 1e-30, 1e-42])
def test_squares_beyond_fp32(gpu_device, scale):
    gradients = make([(1000,), (333,)], (torch.float32,), gpu_device, scale=scale)
    want = norm_of(gradients, 2.0)
    check_norm(gradient_norm(gradients), want)
    clip_gradients(into := [g.clone() for g in gradients], 0.5 * scale)
    for o, g in zip(into, gradients):
        check_scaled(o, g, want, 0.5 * scale)


@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.bfloat16, torch.float32, torch.float16)])
@pytest.mark.parametrize("sizes", [[(1000,), (333,)], [(1 + i % 9,) for i in range(2700)]])        # (the factor made by every workgroup, and by a kernel of its own)
@pytest.mark.parametrize("max_norm", [2.0, 1e-3, 1e-20, 3e-38, 1e-60])
def test_factors_below_the_normal_numbers(gpu_device, max_norm, sizes, dtypes):
    """Gradients as large as their type holds: the factor is far below fp32's normal numbers, and the results are not."""
    gradients = [(g.float().tanh() * (6e4 if g.dtype == torch.float16 else 3e38)).to(g.dtype) for g in make(sizes, dtypes, gpu_device)]
    want = norm_of(gradients, 2.0)
    for out in ([torch.empty_like(g) for g in gradients], [torch.empty_like(g, dtype=torch.float32) for g in gradients], None):
        into = [g.clone() for g in gradients] if out is None else gradients
        norm = clip_gradients(into, max_norm, out=out)
        assert float(norm) == math.inf if float(want) > 3.5e38 else abs(float(norm) - float(want)) <= float(want) * U
        for o, g in zip(into if out is None else out, gradients):
            check_scaled(o, g, want, max_norm)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("where", [0, 4099, 9999])
def test_values_that_are_not_finite(gpu_device, where, dtype, kind):
    gradients = make([(10000,), (50,)], (dtype,), gpu_device)
    gradients[0][where] = math.nan
    out = [torch.empty_like(g) for g in gradients]
    assert math.isnan(clip_gradients(gradients, 1.0, norm_type=kind, out=out)) and all(bool(o.isnan().all()) for o in out)
    gradients[0][where] = -math.inf
    assert float(clip_gradients(gradients, 1.0, norm_type=kind, out=out)) == math.inf
    assert bool(out[0][where].isnan()) and float(out[0].nan_to_num(0.0).abs().max()) == 0.0 and float(out[1].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", HALF)
def test_orders_and_alignments(gpu_device, dtype):
    flat = make([(9001,)], (dtype,), gpu_device)[0]
    parts = list(flat.split([1, 4, 7, 4101, 130, 9001 - 4243]))                       # off 16 bytes, side by side
    nhwc = make([(6, 5, 3, 3)], (dtype,), gpu_device, 1)[0].contiguous(memory_format=torch.channels_last)
    turned = make([(33, 20)], (dtype,), gpu_device, 2)[0].t()
    columns = make([(40, 30)], (dtype,), gpu_device, 3)[0]
    gradients = parts + [nhwc, turned, columns[:, :11], columns[:, 13:]]
    kept, aside = [g.clone() for g in gradients], columns[:, 11:13].clone()
    want = norm_of(gradients, 2.0)
    out = [torch.empty_strided(g.shape, g.stride(), dtype=torch.float32, device=gpu_device) for g in gradients[:-2]] + [torch.empty(g.shape, device=gpu_device) for g in gradients[-2:]]
    out[-3] = torch.empty(20, 33, device=gpu_device)                                   # (another order than its gradient's)
    check_norm(clip_gradients(gradients, 1.5, out=out), want)
    for o, g in zip(out, gradients):
        check_scaled(o, g, want, 1.5)
    before = [g._version for g in gradients]
    check_norm(clip_gradients(gradients, 1.5), want)
    assert all(g._version > v for g, v in zip(gradients, before))
    for g, k in zip(gradients, kept):
        check_scaled(g, k, want, 1.5)
    assert torch.equal(columns[:, 11:13], aside)


def test_what_lies_beside_is_left_alone(gpu_device):
    for n in (1, 5, 4096, 4103):
        buffer = torch.full((n + 32,), 3.0, device=gpu_device)
        clip_gradients([buffer[13:13 + n]], 1e-3)
        assert bool((buffer[:13] == 3).all() and (buffer[13 + n:] == 3).all() and (buffer[13:13 + n] < 1).all())


def test_refusals(gpu_device):
    g, h = torch.ones(8, device=gpu_device), torch.ones(8, device=gpu_device)
    with pytest.raises(_lib.CascmmError, match="shares memory"):
        clip_gradients([g, g], 1.0)
    with pytest.raises(_lib.CascmmError, match="shares memory"):
        clip_gradients([g, h], 1.0, out=[h, g])
    with pytest.raises(ValueError, match="shares memory"):
        c = torch.ones(8, 8, device=gpu_device)
        clip_gradients([c[:, :3], c[:, :5]], 1.0)
    with pytest.raises(ValueError, match="share memory"):
        clip_gradients([torch.ones(1, device=gpu_device).expand(8)], 1.0)
    with pytest.raises(ValueError, match="results"):
        clip_gradients([g, h], 1.0, out=[g])
    with pytest.raises(ValueError, match="out"):
        clip_gradients([g], 1.0, out=[torch.ones(9, device=gpu_device)])
    with pytest.raises(ValueError, match="out"):
        clip_gradients([g], 1.0, out=[torch.ones(8, device=gpu_device, dtype=torch.bfloat16)])
    with pytest.raises(ValueError, match="max_norm"):
        clip_gradients([g], -1.0)
    with pytest.raises(TypeError, match="dense"):
        gradient_norm([torch.ones(8, device=gpu_device, dtype=torch.float64)])
    with pytest.raises(TypeError, match="dense"):
        gradient_norm([torch.eye(3, device=gpu_device).to_sparse()])
    with pytest.raises(RuntimeError, match="AMD GPU"):
        gradient_norm([g, torch.ones(3)])
    assert bool((g == 1).all() and (h == 1).all())
    assert torch.equal(gradient_norm([g, g]), gradient_norm([g, h]))                   # (a norm reads only)


def test_columns_of_one_buffer(gpu_device):
    """Views whose elements lie between each other are no overlap; views that share elements are one wherever they begin, and then nothing is written."""
    c, far = torch.randn(40, 30, device=gpu_device), torch.randn(40, 30, device=gpu_device)
    kept, views = c.clone(), [c[:, :7], c[:, 7:8], c[:, 8::2], c[:, 9::2]]
    want = norm_of([kept], 2.0)
    check_norm(clip_gradients(views, 0.5), want)
    check_scaled(c, kept, want, 0.5)
    c.copy_(kept)
    for gradients, out in (([c[:, :3], c[:, 2:5]], None), ([far[:, 1:3], far], [c[:, 1:3], c]), ([far, far[:, 1:3]], [c, c[:, 1:3]]), ([far[:, :5], c[:, 4:9]], [c[:, :5], far[:, 4:9]]),
                           ([far[:, :5], c], [c[:, 3:8], torch.empty_like(c)]), ([far[:, :5], c.bfloat16()[:, :2]], [c[:, ::7], c[:, 6:8]]), ([far[:6, :3]], [c.as_strided((6, 3), (1, 1))])):
        with pytest.raises(ValueError, match="share"):
            clip_gradients(gradients, 1e-3, out=out)
        assert torch.equal(c, kept)


def test_ordinary_calls_are_one_native_function(gpu_device):
    g, h = torch.ones(8, 3, device=gpu_device), torch.ones(8, 3, device=gpu_device, dtype=torch.bfloat16)
    f = _lib.native().clip_gradients
    assert f([g, h], None, 2, 0.0).shape == () and f([g, h], [g, h], 0, 1.0).shape == () and f([g.t(), h], [torch.ones_like(g).t(), torch.ones_like(g)], 2, 1.0).shape == ()
    for args in (([], None, 2, 0.0), ([g, g], [g, g], 2, 1.0), ([g], [g[:4]], 2, 1.0), ([g], [h], 2, 1.0), ([g], [g], 3, 1.0), ([g], [g], 2, -1.0), ([g.cpu()], None, 2, 0.0), ([g[:, :2]], None, 2, 0.0),
                 ([g], [g.t().contiguous().t()], 2, 1.0), ((g,), None, 2, 0.0), ([g], [g, g], 2, 1.0), ([g.double()], None, 2, 0.0), ([g], [None], 2, 1.0)):
        assert f(*args) is None


def test_parameters(gpu_device):
    model = torch.nn.Sequential(torch.nn.Linear(37, 50), torch.nn.Linear(50, 3)).to(gpu_device)
    model(torch.randn(8, 37, device=gpu_device)).square().sum().backward()
    model[0].bias.grad = None
    kept = {n: p.grad.clone() for n, p in model.named_parameters() if p.grad is not None}
    want = norm_of(kept.values(), 2.0)
    check_norm(clip_grad_norm_(model.parameters(), 0.01), want)
    for n, p in model.named_parameters():
        if n in kept:
            check_scaled(p.grad, kept[n], want, 0.01)
    model[1].bias.grad[1] = math.nan
    before = model[1].weight.grad.clone()
    with pytest.raises(RuntimeError, match="non-finite"):
        clip_grad_norm_(model.parameters(), 0.01, error_if_nonfinite=True)
    assert torch.equal(model[1].weight.grad, before)


def test_recorded_and_replayed(gpu_device):
    """Two graphs of the same gradients, replayed between eager calls: every replay gives what an eager call gives."""
    shapes = [(50, 70), (4096 * 700,), (3,)]
    gradients, outs = make(shapes, (torch.float32, torch.bfloat16), gpu_device), []
    graphs = []
    side = side_streams()[0]
    for kind in (2.0, math.inf):
        out = [torch.zeros_like(g) for g in gradients]
        clip_gradients(gradients, 0.5, norm_type=kind, out=out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = clip_gradients(gradients, 0.5, norm_type=kind, out=out)
        graphs.append((graph, kind, norm, out))
    for turn in range(4):
        for g, fresh in zip(gradients, make(shapes, (torch.float32, torch.bfloat16), gpu_device, 10 + turn, 0.1 + turn)):
            g.copy_(fresh)
        eager = {}
        for _, kind, _, _ in graphs:
            into = [torch.empty_like(g) for g in gradients]
            eager[kind] = (clip_gradients(gradients, 0.5, norm_type=kind, out=into), into)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for graph, *_ in graphs:
                graph.replay()
        torch.cuda.synchronize()
        for _, kind, norm, out in graphs:
            assert torch.equal(norm, eager[kind][0]) and all(torch.equal(o, e) for o, e in zip(out, eager[kind][1]))


def test_other_stream_and_same_bits(gpu_device):
    gradients = make([(4097, 8195), (129,)], (torch.bfloat16,), gpu_device)
    first = gradient_norm(gradients)
    side = side_streams()[0]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [gradient_norm(gradients) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(first, a) for a in again)
