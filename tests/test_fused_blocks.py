"""Layer norms and epilogues in module trees: the patchers, the modules and the blocks that use them.  The blocks are compared with the
same calls written out, bit by bit: what a kernel computes is the other files' matter."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from basedxl_amd import (BasedXLChainedFeedForward, BasedXLFusedKV, BasedXLLayerNorm, BasedXLLowPConv1x1, BasedXLLowPGEGLU, BasedXLLowPLinear, add_layer_norm,
                         cascaded_lowp_matmul, cascaded_lowp_matmul_epilogue, chain_feed_forward_layers, layer_norm, patch_layer_norms, patch_linear_layers)
from basedxl_amd.unet import BasedXLUnet, patch_unet
from basedxl_amd.unet_skeleton import BasicTransformerBlock, SDXLUNetSkeleton, TimestepEmbedding, fuse_epilogues, fuse_geglu_layers, fuse_kv_projections, last_layer, synthetic_inputs
from basedxl_amd.utils import BasedXLConfig

SMALL = dict(channels=(64, 128, 256), head_dim=32, depths=(1, 2), cross_dim=96, add_time_dim=32)


# ---- without a GPU ----
def test_norm_patcher_keeps_parameters_and_leaves_other_norms_alone():
    model = nn.ModuleDict({"a": nn.LayerNorm(8, eps=1e-3), "b": nn.LayerNorm((2, 8)), "c": nn.Sequential(nn.LayerNorm(4, elementwise_affine=False), nn.GroupNorm(2, 8))})
    weight, names = model["a"].weight, sorted(n for n, _ in model.named_parameters())
    patch_layer_norms(model)
    assert isinstance(model["a"], BasedXLLayerNorm) and model["a"].weight is weight and model["a"].eps == 1e-3
    assert isinstance(model["b"], nn.LayerNorm) and isinstance(model["c"][0], BasedXLLayerNorm) and isinstance(model["c"][1], nn.GroupNorm)
    assert model["c"][0].weight is None and sorted(n for n, _ in model.named_parameters()) == names
    with pytest.raises(ValueError, match="last axis"):
        BasedXLLayerNorm(nn.LayerNorm((2, 8)))
    with pytest.raises(ValueError, match="8 columns"):
        model["a"](torch.zeros(2, 7))


def test_norm_patcher_leaves_subclasses_alone():
    class Scaled(nn.LayerNorm):
        def forward(self, x):
            return 2 * super().forward(x)

    model = nn.Sequential(Scaled(8), nn.LayerNorm(8))
    patch_layer_norms(model)
    assert type(model[0]) is Scaled and isinstance(model[1], BasedXLLayerNorm)


def test_norm_patcher_leaves_norms_with_hooks_alone():
    block, seen = BasicTransformerBlock(32, 2, 24), []
    block.norm2.register_forward_hook(lambda m, args, y: seen.append(m))
    block.norm3.register_forward_pre_hook(lambda m, args: seen.append(m))
    norm2, norm3 = block.norm2, block.norm3
    patch_layer_norms(block)
    assert isinstance(block.norm1, BasedXLLayerNorm) and block.norm2 is norm2 and block.norm3 is norm3
    block.norm1 = nn.Identity()
    block(torch.randn(2, 5, 32), torch.randn(2, 3, 24))
    assert seen == [norm2, norm3]
    model = nn.ModuleList([nn.LayerNorm(4), nn.LayerNorm(4)])
    model[0].register_full_backward_hook(lambda m, gi, go: None)
    patch_layer_norms(model)
    assert type(model[0]) is nn.LayerNorm and isinstance(model[1], BasedXLLayerNorm)


def test_linear_wrapper_checks_its_activation():
    with pytest.raises(ValueError, match="activation"):
        BasedXLLowPLinear(nn.Linear(4, 4), activation="tanh")
    assert BasedXLLowPLinear(nn.Linear(4, 4)).activation is None and BasedXLLowPLinear(nn.Linear(4, 4), activation="gelu").activation == "gelu"


def test_the_config_fuses_only_when_asked():
    plain = patch_unet(SDXLUNetSkeleton(**SMALL), BasedXLConfig(fp16_acc_matmul=True))
    assert not any(getattr(m, "fused_epilogues", False) or isinstance(m, BasedXLLayerNorm) for m in plain.modules())
    model = patch_unet(SDXLUNetSkeleton(**SMALL), BasedXLConfig(fp16_acc_matmul=True, fuse_epilogues=True, fuse_norms=True))
    kinds = [m for m in model.modules() if isinstance(m, (BasicTransformerBlock, TimestepEmbedding))]
    assert kinds and all(m.fused_epilogues for m in kinds)
    assert model.time_embedding.linear_1.activation == "silu" and model.time_embedding.linear_2.activation is None
    assert not any(type(m) is nn.LayerNorm for m in model.modules())
    off = patch_unet(SDXLUNetSkeleton(**SMALL), BasedXLConfig(fuse_epilogues=True, fuse_norms=True))
    assert not any(getattr(m, "fused_epilogues", False) or isinstance(m, BasedXLLayerNorm) for m in off.modules())
    # nothing routed: nothing to hold an epilogue
    assert not any(getattr(m, "fused_epilogues", False) for m in fuse_epilogues(SDXLUNetSkeleton(**SMALL)).modules())


def test_an_unrouted_block_adds_its_residuals_itself():
    torch.manual_seed(0)
    block = BasicTransformerBlock(32, 2, 24)
    x, ctx = torch.randn(2, 5, 32), torch.randn(2, 3, 24)
    want = block(x, ctx)
    block.fused_epilogues = True
    assert torch.equal(block(x, ctx), want)
    block.train()
    for attn in (block.attn1, block.attn2):
        attn.to_out[1] = nn.Dropout(0.5)      # (an active dropout stands between the layer and the add)
    torch.manual_seed(1)
    got = block(x, ctx)
    block.fused_epilogues = False
    torch.manual_seed(1)
    assert torch.equal(got, block(x, ctx))


def test_custom_ops_shapes_without_a_gpu():
    from basedxl_amd.compiled import add_layer_norm_op, cascade_linear_epilogue, layer_norm_op
    x, w = torch.empty(2, 3, 16, device="meta"), torch.empty(16, 8, device="meta")
    assert cascade_linear_epilogue(x, w, None, None, torch.empty(2, 3, 8, device="meta"), "gelu", "bf16", 2, "tri", None).shape == (2, 3, 8)
    assert layer_norm_op(x, None, None, 1e-5).shape == x.shape and [t.shape for t in add_layer_norm_op(x, x, None, None, 1e-5)] == [x.shape, x.shape]


# ---- on the GPU ----
def linear(device, i, o, dtype, **kw):
    return BasedXLLowPLinear(nn.Linear(i, o).to(device=device, dtype=dtype), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, kw", [(torch.float32, {}), (torch.float32, dict(prepared=True)), (torch.float32, dict(lowp="fp16", terms=3)),
                                       (torch.float32, dict(lowp="fp8", terms=3)), (torch.float32, dict(lowp="fp8", terms=3, prepared=True)),
                                       (torch.float16, {}), (torch.bfloat16, dict(prepared=False))])
@pytest.mark.parametrize("rows, i, o", [(2, 64, 96), (300, 128, 320), (77, 50, 30)])
def test_linear_wrapper_with_an_epilogue(gpu_device, dtype, kw, rows, i, o):
    torch.manual_seed(3)
    layer = linear(gpu_device, i, o, dtype, **kw)
    x, r = torch.randn(rows, i, device=gpu_device, dtype=dtype), torch.randn(rows, o, device=gpu_device, dtype=dtype)
    with torch.no_grad():
        z = layer(x)
        layer.activation = "gelu"
        y, yr = layer(x), layer(x, r)
    u = torch.finfo(dtype).eps / 2
    # (z as the plain layer rounds it: off by a half step of it, slope 1.13, and one more of the result)
    for got, want in ((y, F.gelu(z.double())), (yr, F.gelu(z.double()) + r.double())):
        tol = 2.0 ** -20 * (1 + z.double().abs()) if dtype == torch.float32 else 1.13 * u * z.double().abs() + 2.0 ** -20
        assert bool(((got.double() - want).abs() <= tol + u * want.abs() + 2.0 ** -24).all())


@pytest.mark.gpu
def test_gradients_pass_a_linear_wrapper_with_an_epilogue(gpu_device):
    torch.manual_seed(4)
    for kw in (dict(prepared=False), dict(prepared=True)):
        layer = linear(gpu_device, 64, 96, torch.float16, **kw)
        x, r = (torch.randn(33, n, device=gpu_device, dtype=torch.float16).requires_grad_() for n in (64, 96))
        dy = torch.randn(33, 96, device=gpu_device, dtype=torch.float16)
        gx, gr = torch.autograd.grad(layer(x, r), (x, r), dy)
        wx, wr = torch.autograd.grad(cascaded_lowp_matmul_epilogue(x, layer.weight, bias=layer.bias, residual=r), (x, r), dy)
        assert torch.equal(gx, wx) and torch.equal(gr, wr)


def block_of(device, dtype, norms, epilogues, seed=5):
    torch.manual_seed(seed)
    block = BasicTransformerBlock(128, 4, 96).to(device=device, dtype=dtype).requires_grad_(False)
    for p in block.parameters():
        p.normal_(0, 0.1)
    patch_linear_layers(block)
    if epilogues:
        fuse_epilogues(block)
    if norms:
        patch_layer_norms(block)
    return block


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_blocks_make_the_calls_they_stand_for(gpu_device, dtype):
    x, ctx = torch.randn(2, 70, 128, device=gpu_device).to(dtype), torch.randn(2, 11, 96, device=gpu_device).to(dtype)

    def attend(a, h, c):
        q, k, v = a.to_q(h), a.to_k(c), a.to_v(c)
        heads = lambda t: t.reshape(2, -1, 4, 32).transpose(1, 2)   # noqa: E731
        return F.scaled_dot_product_attention(heads(q), heads(k), heads(v)).transpose(1, 2).reshape(2, 70, 128)

    def gated(f, h):
        value, gate = f.net[0].proj(h).chunk(2, dim=-1)
        return value * F.gelu(gate)

    # epilogues and norms
    b = block_of(gpu_device, dtype, True, True)
    n = lambda m, t: layer_norm(t, m.weight, m.bias, eps=m.eps)   # noqa: E731
    want = b.attn1.to_out[0](attend(b.attn1, n(b.norm1, x), n(b.norm1, x)), x)
    want = b.attn2.to_out[0](attend(b.attn2, n(b.norm2, want), ctx), want)
    want = b.ff.net[2](gated(b.ff, n(b.norm3, want)), want)
    assert torch.equal(b(x, ctx), want)
    # epilogues alone
    b = block_of(gpu_device, dtype, False, True)
    want = b.attn1.to_out[0](attend(b.attn1, b.norm1(x), b.norm1(x)), x)
    want = b.attn2.to_out[0](attend(b.attn2, b.norm2(want), ctx), want)
    want = b.ff.net[2](gated(b.ff, b.norm3(want)), want)
    assert torch.equal(b(x, ctx), want)
    # norms alone: the adds in front of them
    b = block_of(gpu_device, dtype, True, False)
    h, s = add_layer_norm(b.attn1.to_out[0](attend(b.attn1, n(b.norm1, x), n(b.norm1, x))), x, b.norm2.weight, b.norm2.bias, eps=b.norm2.eps)
    h, s = add_layer_norm(b.attn2.to_out[0](attend(b.attn2, h, ctx)), s, b.norm3.weight, b.norm3.bias, eps=b.norm3.eps)
    assert torch.equal(b(x, ctx), s + b.ff.net[2](gated(b.ff, h)))


@pytest.mark.gpu
def test_embedding_with_its_activation_in_the_epilogue(gpu_device):
    torch.manual_seed(6)
    e = TimestepEmbedding(64, 128).to(gpu_device).requires_grad_(False)
    patch_linear_layers(e)
    x = torch.randn(2, 64, device=gpu_device)
    fused = fuse_epilogues(copy.deepcopy(e))
    want = fused.linear_2(cascaded_lowp_matmul_epilogue(x, e.linear_1.weight, bias=e.linear_1.bias, activation="silu"))
    assert torch.equal(fused(x), want)
    assert float((fused(x) - e(x)).norm() / e(x).norm()) < 1e-5
    assert torch.equal(e.linear_1(x), cascaded_lowp_matmul(x, e.linear_1.weight, bias=e.linear_1.bias))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_fused_block_traces_under_torch_compile(gpu_device, dtype):
    b = block_of(gpu_device, dtype, True, True)
    x, ctx = torch.randn(2, 70, 128, device=gpu_device).to(dtype), torch.randn(2, 11, 96, device=gpu_device).to(dtype)
    split = block_of(gpu_device, dtype, True, False)
    with torch.no_grad():
        for m in (b, split):
            want = m(x, ctx)
            assert torch.equal(torch.compile(m, backend="aot_eager", fullgraph=True)(x, ctx), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, bound", [(torch.float32, 1e-3), (torch.float16, 3e-2)])
def test_small_unet_with_and_without(gpu_device, dtype, bound):
    """The same function, rounded elsewhere: fp32 layers are off by 1e-5 (two bf16 terms), fp16 ones by 2^-11, and some thirty of them follow each other."""
    base = SDXLUNetSkeleton(**SMALL, device=gpu_device).to(dtype)
    inputs = synthetic_inputs(base, batch=2, latent=16, device=gpu_device, dtype=dtype)
    with torch.no_grad():
        want = BasedXLUnet(copy.deepcopy(base), BasedXLConfig(dtype=dtype, fp16_acc_matmul=True))(*inputs).double()
        for flags in (dict(fuse_epilogues=True), dict(fuse_norms=True), dict(fuse_epilogues=True, fuse_norms=True, fuse_geglu=True), dict(fuse_epilogues=True, chain_ffn=True)):
            got = BasedXLUnet(copy.deepcopy(base), BasedXLConfig(dtype=dtype, fp16_acc_matmul=True, **flags))(*inputs).double()
            assert float((got - want).norm() / want.norm()) <= bound, flags


# ---- gradients through module trees ----
# Products of fp32 operands by two bf16 terms leave out 3 2^-16 of |a| @ |b|, by three fp16 terms 2^-24, by three fp8 terms 2^-9 of it (tests/test_gpu_matmul_epilogue.py)
LOST = {(torch.float32, "bf16"): 3 * 2.0 ** -16, (torch.float32, "fp16"): 2.0 ** -24, (torch.float32, "fp8"): 2.0 ** -9, (torch.float16, "fp16"): 0.0, (torch.bfloat16, "bf16"): 0.0}
LAYERS = [(torch.float32, {}), (torch.float32, dict(prepared=True)), (torch.float32, dict(lowp="fp16", terms=3)), (torch.float32, dict(lowp="fp8", terms=3)),
          (torch.float32, dict(lowp="fp8", terms=3, prepared=True)), (torch.float16, {}), (torch.bfloat16, dict(prepared=False)), (torch.bfloat16, {})]


def product_tolerance(dy, w, dtype, lowp):
    """(dy @ w.T in 64 bits, how far a product of one cascade may be off)."""
    want, S = dy.double() @ w.double().t(), dy.double().abs() @ w.double().abs().t()
    u = torch.finfo(dtype).eps / 2
    return want, ((w.shape[1] + 4) * 2.0 ** -24 + LOST[dtype, lowp]) * S + u * want.abs() + torch.finfo(dtype).smallest_normal


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, kw", LAYERS)
@pytest.mark.parametrize("rows, i, o", [(2, 64, 96), (300, 128, 320), (77, 50, 30), (1, 1, 1)])
def test_gradients_pass_a_linear_wrapper(gpu_device, dtype, kw, rows, i, o):
    torch.manual_seed(7)
    layer = linear(gpu_device, i, o, dtype, **kw)
    x, dy = torch.randn(2, rows, i, device=gpu_device, dtype=dtype), torch.randn(2, rows, o, device=gpu_device, dtype=dtype)
    with torch.no_grad():
        want = layer(x)
    leaf = x.clone().requires_grad_()
    y = layer(leaf)
    assert torch.equal(y, want)          # (the same kernels, prepared weights among them)
    (g,) = torch.autograd.grad(y, leaf, dy, create_graph=True)
    dx, tol = product_tolerance(dy, layer.weight, dtype, layer.lowp)
    assert bool(((g.detach().double() - dx).abs() <= tol).all())
    with pytest.raises(RuntimeError):    # (once differentiable)
        g.sum().backward()
    # a gradient that is one value for all, and no graph where none is wanted
    (g,) = torch.autograd.grad(layer(leaf).sum(), leaf)
    assert torch.equal(g, torch.autograd.grad(layer(leaf), leaf, torch.ones_like(dy))[0])
    with torch.no_grad():
        assert layer(leaf).grad_fn is None
    assert layer(x).grad_fn is None
    # weights written to between the two ways are noticed
    y = layer(leaf)
    layer.weight.mul_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, kw", LAYERS)
@pytest.mark.parametrize("rows, i, inner", [(130, 128, 64), (20, 50, 30)])
def test_gradients_pass_a_gated_wrapper(gpu_device, dtype, kw, rows, i, inner):
    torch.manual_seed(8)
    layer = BasedXLLowPGEGLU(nn.Linear(i, 2 * inner).to(device=gpu_device, dtype=dtype), **kw)
    x, dy = torch.randn(rows, i, device=gpu_device, dtype=dtype), torch.randn(rows, inner, device=gpu_device, dtype=dtype)
    with torch.no_grad():
        want = layer(x)
    leaf = x.clone().requires_grad_()
    y = layer(leaf)
    assert torch.equal(y, want)
    (g,) = torch.autograd.grad(y, leaf, dy)
    e = x.double().requires_grad_()
    value, gate = (e @ layer.weight.double() + layer.bias.double()).chunk(2, dim=-1)
    (dx,) = torch.autograd.grad(value * F.gelu(gate), e, dy.double())
    # In the mean square: h, dh and the result are rounded once each (half a step at most), dh follows h with slopes up to 1.13 in the value and 0.8 of the value
    # in the gate; the products leave out `lost` of |a| @ |b|, which adds up over K as they do, twice: four of the larger
    assert float((g.double() - dx).norm() / dx.norm()) <= 4 * max(torch.finfo(dtype).eps / 2, LOST[dtype, layer.lowp], 2.0 ** -22)


@pytest.mark.gpu
def test_gradients_pass_a_chained_feed_forward(gpu_device):
    torch.manual_seed(9)
    proj, out = nn.Linear(320, 2560).to(gpu_device), nn.Linear(1280, 320).to(gpu_device)
    for prepared in (False, True):
        ff = BasedXLChainedFeedForward(proj, out, prepared=prepared)
        for rows in (8192, 100):    # (with the chain, and layer by layer)
            x, dy = torch.randn(rows, 320, device=gpu_device), torch.randn(rows, 320, device=gpu_device)
            with torch.no_grad():
                want = ff(x)
            chained, leaf = ff.chained_calls, x.clone().requires_grad_()
            y = ff(leaf)
            assert torch.equal(y, want) and (ff.chained_calls > chained) == (rows == 8192)
            (g,) = torch.autograd.grad(y, leaf, dy)
            (wg,) = torch.autograd.grad(ff.linear(ff.geglu(leaf)), leaf, dy)
            assert torch.equal(g, wg)
            e = x.double().requires_grad_()
            value, gate = F.linear(e, proj.weight.double(), proj.bias.double()).chunk(2, dim=-1)
            (dx,) = torch.autograd.grad(F.linear(value * F.gelu(gate), out.weight.double()), e, dy.double())
            assert float((g.double() - dx).norm() / dx.norm()) <= 6 * 3 * 2.0 ** -16   # (three products of the cascade, the first one's error with slopes up to 1.13)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_gradients_pass_a_pointwise_convolution(gpu_device, dtype):
    torch.manual_seed(10)
    conv = BasedXLLowPConv1x1(nn.Conv2d(64, 96, 1).to(device=gpu_device, dtype=dtype))
    for layout in (torch.contiguous_format, torch.channels_last):
        x = torch.randn(3, 64, 9, 7, device=gpu_device, dtype=dtype).contiguous(memory_format=layout)
        dy = torch.randn(3, 96, 9, 7, device=gpu_device, dtype=dtype)
        with torch.no_grad():
            want = conv(x)
        leaf = x.clone().requires_grad_()
        y = conv(leaf)
        assert torch.equal(y, want)
        for d in (dy, dy.contiguous(memory_format=torch.channels_last)):
            (g,) = torch.autograd.grad(conv(leaf), leaf, d)
            dx, tol = product_tolerance(dy.permute(0, 2, 3, 1), conv.weight.t(), dtype, conv.lowp)
            assert g.shape == x.shape and bool(((g.permute(0, 2, 3, 1).double() - dx).abs() <= tol).all())


@pytest.mark.gpu
def test_a_kept_key_and_value_are_constants(gpu_device):
    torch.manual_seed(11)
    kv = BasedXLFusedKV(nn.Linear(64, 32).to(gpu_device), nn.Linear(64, 32).to(gpu_device), cache=True)
    s = torch.randn(10, 64, device=gpu_device, requires_grad=True)
    k, v = kv(s)
    (g,) = torch.autograd.grad((k.sum() + 2 * v.sum()), s)
    dx, tol = product_tolerance(torch.cat([torch.ones(10, 32), 2 * torch.ones(10, 32)], 1).to(gpu_device), kv.to_kv.weight, torch.float32, "bf16")
    assert bool(((g.double() - dx).abs() <= tol).all())
    k2, v2 = kv(s)
    assert torch.equal(k2, k) and torch.equal(v2, v) and not k2.requires_grad
    k3, _ = kv(s, recompute=True)
    assert torch.equal(k3, k) and k3.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("kw, bound", [({}, 2e-3), (dict(lowp="fp16", terms=3), 2e-5)])
@pytest.mark.parametrize("what", ["linear", "epilogues", "norms", "both", "fused", "chained"])
def test_gradients_of_a_whole_block(gpu_device, what, kw, bound):
    """dx, the context's gradient and the norms' of a transformer block in fp32, against torch in 64 bits.  In the mean square a product by two bf16
    terms leaves out at most 3 2^-16 = 4.6e-5 of itself, some ten of them follow each other either way, and norms and softmax at most quadruple an error: 2e-3;
    three fp16 terms hold fp32's own accuracy, some thirty sums of 128 and more numbers in fp32, 2^-24 (128)^1/2 each: 2e-5."""
    torch.manual_seed(12)
    base = BasicTransformerBlock(128, 4, 96).to(gpu_device)
    for p in base.parameters():
        p.data.normal_(0, 0.1)
    for n in (base.norm1, base.norm2, base.norm3):
        n.weight.data += 1
    block = copy.deepcopy(base)
    if what == "chained":
        chain_feed_forward_layers(block, **kw)
    if what == "fused":
        fuse_kv_projections(block, fuse_q=True, **kw)
        fuse_geglu_layers(block, **kw)
    patch_linear_layers(block, **kw)
    if what in ("epilogues", "both", "fused", "chained"):
        fuse_epilogues(block)
    if what in ("norms", "both", "fused", "chained"):
        patch_layer_norms(block)
    x, ctx, dy = torch.randn(2, 70, 128, device=gpu_device), torch.randn(2, 11, 96, device=gpu_device), torch.randn(2, 70, 128, device=gpu_device)
    norms = ["norm1", "norm2", "norm3"]

    def grads(b, x, ctx, dy):
        leaves = [x.detach().clone().requires_grad_(), ctx.detach().clone().requires_grad_()]
        params = [p for n in norms for p in (getattr(b, n).weight, getattr(b, n).bias)]
        y = b(leaves[0], leaves[1])
        return [y.detach(), *torch.autograd.grad(y, leaves + params, dy)]

    got = grads(block, x, ctx, dy)
    want = grads(base.double().cpu(), x.double().cpu(), ctx.double().cpu(), dy.double().cpu())
    for name, g, w in zip(["y", "x", "context", *[n + "." + p for n in norms for p in ("weight", "bias")]], got, want):
        assert float((g.cpu().double() - w).norm() / w.norm()) <= bound, name


@pytest.mark.gpu
def test_sums_of_two_dtypes_are_promoted_as_torch_does(gpu_device):
    """Under autocast the Linear layers of a block whose norms alone are patched give fp16, the residual stream stays fp32."""
    torch.manual_seed(13)
    base = BasicTransformerBlock(128, 4, 96).to(gpu_device).requires_grad_(False)
    block = patch_layer_norms(copy.deepcopy(base))
    x, ctx = torch.randn(2, 70, 128, device=gpu_device), torch.randn(2, 11, 96, device=gpu_device)
    with torch.no_grad(), torch.autocast("cuda", torch.float16):
        want, got = base(x, ctx), block(x, ctx)
    assert got.dtype == want.dtype == torch.float32
    # (the norms differ by fp32's half steps, which now and then turn a rounding to fp16 around: single half steps of it, far less in the mean square)
    assert float((got - want).norm() / want.norm()) <= 2.0 ** -11
    # an epilogue with a residual of another dtype
    layer = linear(gpu_device, 64, 96, torch.float16)
    a, r = torch.randn(5, 64, device=gpu_device).half(), torch.randn(5, 96, device=gpu_device)
    assert torch.equal(last_layer(layer, a, r), r + layer(a)) and last_layer(layer, a, r).dtype == torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_recorded_gradients_of_modules(gpu_device, dtype):
    """Forward and backward through routed modules in a graph, replayed between eager work of their own."""
    torch.manual_seed(14)
    first, gated, conv = linear(gpu_device, 64, 96, dtype), BasedXLLowPGEGLU(nn.Linear(96, 128).to(device=gpu_device, dtype=dtype)), \
        BasedXLLowPConv1x1(nn.Conv2d(64, 32, 1).to(device=gpu_device, dtype=dtype))
    norm = BasedXLLayerNorm(nn.LayerNorm(64).to(device=gpu_device, dtype=dtype))

    def step(x, dy, w, b):
        norm.weight, norm.bias = w, b
        h = gated(first(norm(x)))
        y = conv(h.view(2, 5, 10, 64).permute(0, 3, 1, 2))
        return (y, *torch.autograd.grad(y, (x, w, b), dy))

    def inputs(seed):
        gen = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(gpu_device)   # noqa: E731
        return [r(100, 64).requires_grad_(), r(2, 32, 5, 10), r(64).requires_grad_(), r(64).requires_grad_()]

    norm.weight = norm.bias = None
    side, ins = torch.cuda.Stream(), inputs(0)
    ins = [nn.Parameter(t.detach()) if t.requires_grad else t for t in ins]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*ins)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*ins)
    for seed in range(1, 5):
        fresh = inputs(seed)
        with torch.no_grad():
            for t, f in zip(ins, fresh):
                t.copy_(f)
        graph.replay()
        got = [t.detach().clone() for t in outs]
        want = step(*[nn.Parameter(f.detach()) if f.requires_grad else f for f in fresh])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
