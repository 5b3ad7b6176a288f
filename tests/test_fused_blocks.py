"""Layer norms and epilogues in module trees: the patchers, the modules and the blocks that use them.  The blocks are compared with the
same calls written out, bit by bit: what a kernel computes is the other files' matter."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from basedxl_amd import (BasedXLLayerNorm, BasedXLLowPLinear, add_layer_norm, cascaded_lowp_matmul, cascaded_lowp_matmul_epilogue, layer_norm, patch_layer_norms,
                         patch_linear_layers)
from basedxl_amd.unet import BasedXLUnet, patch_unet
from basedxl_amd.unet_skeleton import BasicTransformerBlock, SDXLUNetSkeleton, TimestepEmbedding, fuse_epilogues, synthetic_inputs
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
