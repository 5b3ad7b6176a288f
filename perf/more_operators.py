"""Three more operators around the package's products, as timed cases: a product in 8 bits, the norms on both sides of a
block's residual add, and the clipping of gradients by their common norm.

Each in its plain form (elementary torch operations in 32 bits) and, with ``own`` set, as a user's program calls it:

* ``product``: ``block_scaled_matmul(a, b, bias=)``.  Both operands are rounded to 8-bit floating point (e4m3) with one
  power of two as the scale of every block of 128.  A block is 128 consecutive k of one row of ``a``, and 128 x 128 elements
  of ``b``; its scale 2^e is the smallest with max|x| <= 448 * 2^e over the block's finite elements (from 2^-127 on; 1 where
  the block has no finite element but zeros); infinities and NaN become NaN.  The blocks at the ends are shorter.  Products
  and sums of the rounded operands are those of 32 bits.  The gradients are products of the same kind: da = dy b^T with the
  same rounded b, dy in blocks of 128 along n; db = a^T dy with both in blocks of 128 along the rows; dbias sums dy itself.
* ``norm``: ``gated_add_norm(x, residual, weight, bias, gate=, residual_scale=, post_norm=, post_weight=, norm=)``:
  s = residual_scale * residual + gate * post(x), rounded to the tensors' type, and y = norm(s) * weight + bias of that s.
  ``post``: nothing, or the same kind of norm with a weight of its own.  The kinds: "layer" and "rms".
* ``clip``: ``clip_gradients(gradients, max_norm, norm_type=, out=)``: the norm of all gradients taken together, and every
  gradient times min(1, max_norm / (norm + 1e-6)), into ``out``.

Activations are N(0, 1) with a spread of scales and means over the columns, as a residual stream has them; weights of
products N(0, 0.02), of norms around one.
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5


def _named(name, case):
    return case if name is None else {"name": name, **case}


def _product(rows, k, n, *, dtype="bf16", train=False, kept=False, bias=True, name=None):
    """``kept``: the weight is held rounded between calls, as a serving program holds it."""
    return _named(name, {"kind": "product", "rows": rows, "k": k, "n": n, "dtype": dtype, "train": train, "kept": kept, "bias": bias})


def _norm(samples, rows, cols, *, dtype="bf16", train=False, norm="layer", post=False, gate="none", scaled=False, modulated=False, name=None):
    """``samples`` of ``rows`` tokens each; ``gate``: "none", "channel" (one for all tokens) or "sample" (one for each
    sample); ``scaled``: the residual has a scale of its own in each channel; ``modulated``: weight and bias are given for each sample."""
    return _named(name, {"kind": "norm", "samples": samples, "rows": rows, "cols": cols, "dtype": dtype, "train": train, "norm": norm, "post": post,
                         "gate": gate, "scaled": scaled, "modulated": modulated})


def _clip(blocks, width, *, dtype="fp32", out="same", norm="2", max_norm=1.0, name=None):
    """The gradients of ``blocks`` transformer blocks of ``width`` channels."""
    return _named(name, {"kind": "clip", "blocks": blocks, "width": width, "dtype": dtype, "out": out, "norm": norm, "max_norm": max_norm})


def listed():
    return [
        # one token through a down-projection, weight kept: latency and the weight's bytes
        _product(1, 5120, 1280, kept=True, name="product_token_bf16"),
        # a text encoder's 2 x 77 tokens through its up-projection
        _product(154, 1280, 5120, dtype="fp16", kept=True, name="product_text_fp16"),
        # the wide projection of a feed-forward block at the 32 x 32 stage, guided batch of two
        _product(2048, 1280, 10240, kept=True, name="product_ffn_bf16"),
        # the same block's projection while it is trained, tokens of eight images
        _product(8192, 1280, 5120, train=True, name="product_train_bf16"),
        # no dimension a multiple of anything, fp32, trained
        _product(333, 457, 211, dtype="fp32", train=True, name="product_train_ragged_fp32"),
        # two pooled rows: nothing but latency
        _norm(2, 1, 1280, dtype="fp16", gate="sample", modulated=True, name="norm_pooled_fp16"),
        # a block with norms on both sides at the 64 x 64 stage, guided batch of two, a gate in each channel
        _norm(2, 4096, 640, dtype="bf16", norm="rms", post=True, gate="channel", name="norm_tokens_rms_bf16"),
        # a training batch at the 32 x 32 stage, gated and modulated by its conditioning: bytes, and sums over each sample's tokens
        _norm(32, 1024, 1280, dtype="bf16", train=True, gate="sample", modulated=True, name="norm_train_sample_bf16"),
        # odd columns and rows, fp32, everything that can be learned
        _norm(3, 777, 457, dtype="fp32", train=True, post=True, gate="channel", scaled=True, name="norm_train_ragged_fp32"),
        # a small adapter's gradients: launches
        _clip(3, 32, max_norm=0.1, name="clip_adapter_fp32"),
        # half a dozen odd-sized blocks in bf16, accumulated into fp32 gradients
        _clip(6, 645, dtype="bf16", out="fp32", name="clip_blocks_bf16"),
        # forty blocks at the 32 x 32 stage's width: bytes
        _clip(40, 1280, name="clip_stage_fp32"),
    ]


#: multiply-adds of the largest listed products (16-bit, and fp32), elements of the largest listed norm and gradients
_MOST_MACS = {"fp32": 8192 * 1280 * 1280, "fp16": 3 * 8192 * 1280 * 5120, "bf16": 3 * 8192 * 1280 * 5120}
_MOST_ELEMENTS = 32 * 1024 * 1280
_MOST_GRADIENTS = 40 * 12 * 1280 * 1280


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Layer widths: mostly multiples of 64, some of 8, some anything."""
    x, r = _log(rng, lo, hi), rng.random()
    unit = 64 if r < 0.6 else 8 if r < 0.8 else 1
    return max(unit, (x + unit // 2) // unit * unit)


def draw(rng):
    kind = rng.choice(("product", "product", "norm", "norm", "clip"))
    dtype = rng.choice(("fp32", "fp16", "bf16"))
    train = rng.random() < 0.5
    if kind == "product":
        k, n, rows = _width(rng, 64, 5120), _width(rng, 64, 10240), _log(rng, 1, 8192)
        rows = max(1, min(rows, int(0.9 * _MOST_MACS[dtype]) // ((3 if train else 1) * k * n)))
        return _product(rows, k, n, dtype=dtype, train=train, kept=not train and rng.random() < 0.7, bias=rng.random() < 0.7)
    if kind == "norm":
        cols, samples, rows = _width(rng, 64, 2560), _log(rng, 1, 32), _log(rng, 1, 4096)
        most = _MOST_ELEMENTS // (2 if dtype == "fp32" else 1)
        rows = max(1, min(rows, int(0.9 * most) // (samples * cols)))
        return _norm(samples, rows, cols, dtype=dtype, train=train, norm=rng.choice(("layer", "rms")), post=rng.random() < 0.5,
                     gate=rng.choice(("none", "channel", "sample")), scaled=rng.random() < 0.3, modulated=rng.random() < 0.3)
    width = _width(rng, 32, 1280)
    blocks = max(1, min(_log(rng, 1, 40), int(0.9 * _MOST_GRADIENTS) // (12 * width * width)))
    return _clip(blocks, width, dtype=dtype, out=rng.choice(("same", "fp32")), norm=rng.choice(("2", "2", "inf")),
                 max_norm=rng.choice((0.1, 1.0, 1e6)))


def _gradient_shapes(case):
    w = case["width"]
    return [s for _ in range(case["blocks"]) for s in ((w, w), (w, w), (w, w), (w, w), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,), (w,))]


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "product":
        rows, k, n = case["rows"], case["k"], case["n"]
        bias = n if case["bias"] else 0
        read = size * (rows * k + bias + rows * n) + (1 if case["kept"] else size) * k * n
        if case["train"]:   # (the result's gradient in; those of a, b and the bias out)
            read += size * (rows * n + rows * k + k * n + bias)
        return {"bytes": read, "flops": 2 * (3 if case["train"] else 1) * rows * k * n}
    if case["kind"] == "norm":
        tokens, cols, samples = case["samples"] * case["rows"], case["cols"], case["samples"]
        learned = cols * ((1 if case["post"] else 0) + {"none": 0, "channel": 1, "sample": samples}[case["gate"]] + (1 if case["scaled"] else 0)
                          + 2 * (samples if case["modulated"] else 1))
        streams = 4 + (4 if case["train"] else 0)      # (x, residual, s, y; dy, ds, dx, dresidual)
        return {"bytes": size * (streams * tokens * cols + (2 if case["train"] else 1) * learned), "flops": (48 if case["train"] else 14) * tokens * cols}
    count = sum(math.prod(s) for s in _gradient_shapes(case))
    return {"bytes": (size + (4 if case["out"] == "fp32" else size)) * count, "flops": 3 * count}


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * std + mean).to(dtype)

    def stream(*shape):
        spread = torch.exp(0.5 * torch.randn(shape[-1], device="cuda", generator=gen))
        means = 0.5 * torch.randn(shape[-1], device="cuda", generator=gen)
        return (torch.randn(*shape, device="cuda", generator=gen) * spread + means).to(dtype)

    state = dict(case)
    if case["kind"] == "product":
        rows, k, n = case["rows"], case["k"], case["n"]
        state["leaves"] = {"a": stream(rows, k), "b": normal(k, n, std=0.02)}
        if case["bias"]:
            state["leaves"]["bias"] = normal(n, std=0.02)
        if case["train"]:
            state["dy"] = normal(rows, n, std=1e-3)
    elif case["kind"] == "norm":
        samples, rows, cols = case["samples"], case["rows"], case["cols"]
        leaves = state["leaves"] = {"x": stream(samples, rows, cols), "residual": stream(samples, rows, cols)}
        weights = (samples, 1, cols) if case["modulated"] else (cols,)
        leaves["weight"], leaves["bias"] = normal(*weights, std=0.1, mean=1.0), normal(*weights, std=0.1)
        if case["gate"] != "none":
            leaves["gate"] = normal(*((samples, 1, cols) if case["gate"] == "sample" else (cols,)), std=0.3, mean=0.5)
        if case["scaled"]:
            leaves["scale"] = normal(cols, std=0.1, mean=1.0)
        if case["post"]:
            leaves["post_weight"] = normal(cols, std=0.1, mean=1.0)
        if case["train"]:
            state["dy"], state["ds"] = normal(samples, rows, cols), normal(samples, rows, cols)
    else:
        shapes = _gradient_shapes(case)
        flat = normal(sum(math.prod(s) for s in shapes), std=1e-3)
        state["gradients"], at = [], 0
        for s in shapes:
            state["gradients"].append(flat[at:at + math.prod(s)].view(s).clone())
            at += math.prod(s)
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if case["kind"] == "clip":
        # (one buffer of all of them, as a program holds them that exchanges or steps them together)
        state["bucket"] = torch.empty(sum(g.numel() for g in state["gradients"]), dtype=torch.float32 if case["out"] == "fp32" else _DTYPES[case["dtype"]], device="cuda")
        state["into"] = [part.view_as(g) for part, g in zip(state["bucket"].split([g.numel() for g in state["gradients"]]), state["gradients"])]
    elif case["train"]:
        for leaf in state["leaves"].values():
            leaf.requires_grad_(True)
    if own and case["kind"] == "product" and case["kept"]:
        from basedxl_amd import BlockScaledWeight
        state["held"] = BlockScaledWeight(state["leaves"]["b"])
    return state


# ---- plain forms ----
def _rounded(x, block_rows, block_cols):
    """``x`` [r, c] in 32 bits, rounded block by block: the values that the 8 bits and their scales stand for."""
    r, c = x.shape
    padded = torch.zeros(-(-r // block_rows) * block_rows, -(-c // block_cols) * block_cols, device=x.device)
    padded[:r, :c] = x
    tiles = padded.view(padded.shape[0] // block_rows, block_rows, padded.shape[1] // block_cols, block_cols)
    finite = torch.where(tiles.abs() < float("inf"), tiles.abs(), torch.zeros_like(tiles))
    most = finite.amax((1, 3), keepdim=True)
    mantissa, exponent = torch.frexp(most)              # most = mantissa 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(min=-127)
    e = torch.where(most > 0, e, torch.zeros_like(e))
    scaled = torch.ldexp(torch.ldexp(tiles, -(e // 2)), -(e - e // 2))
    scaled = torch.where(tiles.abs() < float("inf"), scaled, torch.full_like(scaled, float("nan")))
    held = scaled.to(torch.float8_e4m3fn).float()
    return torch.ldexp(torch.ldexp(held, e // 2), e - e // 2).reshape(padded.shape)[:r, :c]


def _plain_product(state):
    leaf = {name: t.detach() for name, t in state["leaves"].items()}
    dtype = leaf["a"].dtype
    a, b = leaf["a"].float(), leaf["b"].float()
    held = _rounded(b, 128, 128)
    y = _rounded(a, 1, 128) @ held
    if "bias" in leaf:
        y = y + leaf["bias"].float()
    out = {"y": y.to(dtype)}
    if state["train"]:
        dy = state["dy"].float()
        out["da"] = (_rounded(dy, 1, 128) @ held.t().contiguous()).to(dtype)
        out["db"] = (_rounded(a, 128, 1).t().contiguous() @ _rounded(dy, 128, 1)).to(dtype)
        if "bias" in leaf:
            out["dbias"] = dy.sum(0).to(dtype)
    return out


def _plain_statistics(x, kind):
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    rstd = torch.rsqrt(((x - mean) * (x - mean)).mean(-1, keepdim=True) + _EPS)
    return (x - mean) * rstd, rstd


def _plain_norm_gradient(g, xhat, rstd, kind):
    d = g - xhat * (g * xhat).mean(-1, keepdim=True)
    return rstd * (d - g.mean(-1, keepdim=True) if kind == "layer" else d)


def _plain_norm(state):
    stored = {name: t.detach() for name, t in state["leaves"].items()}
    dtype, kind = stored["x"].dtype, state["norm"]
    leaf = {name: t.float() for name, t in stored.items()}
    p = leaf["x"]
    if state["post"]:
        xhat, rstd = _plain_statistics(p, kind)
        p = xhat * leaf["post_weight"]
    gated = p * leaf["gate"] if "gate" in leaf else p
    s = (gated + (leaf["residual"] * leaf["scale"] if "scale" in leaf else leaf["residual"])).to(dtype)
    shat, srstd = _plain_statistics(s.float(), kind)
    out = {"s": s, "y": (shat * leaf["weight"] + leaf["bias"]).to(dtype)}
    if not state["train"]:
        return out

    def summed(t, name):
        """over the tokens that share an element of ``name``"""
        return (t.sum(1, keepdim=True) if leaf[name].dim() == 3 else t.sum((0, 1))).to(dtype)

    dy = state["dy"].float()
    out["dweight"], out["dbias"] = summed(dy * shat, "weight"), summed(dy, "bias")
    ds = state["ds"].float() + _plain_norm_gradient(dy * leaf["weight"], shat, srstd, kind)
    out["dresidual"] = (ds * leaf["scale"] if "scale" in leaf else ds).to(dtype)
    if "scale" in leaf:
        out["dscale"] = summed(ds * leaf["residual"], "scale")
    if "gate" in leaf:
        out["dgate"] = summed(ds * p, "gate")
    dp = ds * leaf["gate"] if "gate" in leaf else ds
    if state["post"]:
        out["dpost_weight"] = summed(dp * xhat, "post_weight")
        dp = _plain_norm_gradient(dp * leaf["post_weight"], xhat, rstd, kind)
    out["dx"] = dp.to(dtype)
    return out


def _plain_clip(state):
    if state["norm"] == "inf":
        norm = torch.stack([g.abs().amax().float() for g in state["gradients"]]).amax()
    else:   # (long sums: in 64 bits)
        norm = torch.stack([(g.double() * g.double()).sum() for g in state["gradients"]]).sum().sqrt()
    factor = (state["max_norm"] / (norm.double() + 1e-6)).clamp(max=1.0).float()
    for g, into in zip(state["gradients"], state["into"]):
        into.copy_(g.float() * factor)
    return {"norm": norm.float(), "gradients": state["bucket"]}


# ---- the package's calls ----
def _own_product(state):
    from basedxl_amd import block_scaled_matmul
    leaf = state["leaves"]
    y = block_scaled_matmul(leaf["a"], state.get("held", leaf["b"]), bias=leaf.get("bias"))
    if not state["train"]:
        return {"y": y}
    names = [name for name in ("a", "b", "bias") if name in leaf]
    grads = torch.autograd.grad(y, [leaf[name] for name in names], state["dy"])
    return {"y": y.detach(), **{"d" + name: g for name, g in zip(names, grads)}}


def _own_norm(state):
    from basedxl_amd import gated_add_norm
    leaf = state["leaves"]
    y, s = gated_add_norm(leaf["x"], leaf["residual"], leaf["weight"], leaf["bias"], gate=leaf.get("gate"), residual_scale=leaf.get("scale", 1.0),
                          post_norm=state["post"], post_weight=leaf.get("post_weight"), norm=state["norm"], eps=_EPS)
    if not state["train"]:
        return {"s": s, "y": y}
    grads = torch.autograd.grad((y, s), list(leaf.values()), (state["dy"], state["ds"]))
    return {"s": s.detach(), "y": y.detach(), **{"d" + name: g for name, g in zip(leaf, grads)}}


def _own_clip(state):
    from basedxl_amd import clip_gradients
    norm = clip_gradients(state["gradients"], state["max_norm"], norm_type=float(state["norm"]), out=state["into"])
    return {"norm": norm, "gradients": state["bucket"]}


def run(state):
    return (globals()[("_own_" if own else "_plain_") + state["kind"]])(state)


# ---- the definitions, in 64 bits ----
def _held_exactly(x, axis):
    """``x`` in 64 bits, rounded in blocks of 128 along ``axis`` (0, 1, or None: both), from the definition of the format: three
    bits behind the leading one down to 2^-6, steps of 2^-9 below."""
    x = x.double()
    if axis == 0:
        return _held_exactly(x.t(), 1).t()
    out = torch.empty_like(x)
    for at in range(0, x.shape[1], 128):
        part = x[:, at:at + 128]
        most = torch.where(torch.isfinite(part), part, 0.0).abs().amax(1, keepdim=True)
        if axis is None:
            most = torch.cat([rows.amax(0, keepdim=True).expand_as(rows) for rows in most.split(128)])
        e = torch.ceil(torch.log2(torch.where(most > 0, most, 448.0) / 448))
        e = torch.where(most > 448 * torch.exp2(e), e + 1, e)
        e = torch.where(most <= 448 * torch.exp2(e - 1), e - 1, e).clamp(min=-127)
        e = torch.where(most > 0, e, 0.0)
        v = part * torch.exp2(-e)
        floor = torch.floor(torch.log2(torch.where(v != 0, v, 1.0).abs()))
        step = torch.exp2(floor.clamp(min=-6) - 3)
        out[:, at:at + 128] = torch.where(torch.isfinite(part), torch.round(v / step) * step * torch.exp2(e), float("nan"))
    return out


def exact(case, seed):
    state = _inputs(case, seed)
    F = torch.nn.functional
    if case["kind"] == "clip":
        together = torch.cat([g.flatten() for g in state["gradients"]]).double()
        norm = torch.linalg.vector_norm(together, float(case["norm"]))
        return {"norm": norm, "gradients": together.mul_(min(1.0, case["max_norm"] / (float(norm) + 1e-6)))}
    if case["kind"] == "product":
        leaf = state["leaves"]
        held = _held_exactly(leaf["b"], None)
        out = {"y": F.linear(_held_exactly(leaf["a"], 1), held.t(), leaf["bias"].double() if "bias" in leaf else None)}
        if case["train"]:
            out["da"] = F.linear(_held_exactly(state["dy"], 1), held)
            out["db"] = torch.mm(_held_exactly(leaf["a"], 0).t(), _held_exactly(state["dy"], 0))
            if "bias" in leaf:
                out["dbias"] = state["dy"].double().sum(0)
        return out
    dtype, leaf = _DTYPES[case["dtype"]], {name: t.double().requires_grad_(case["train"]) for name, t in state["leaves"].items()}

    def normed(t):
        if case["norm"] == "layer":
            return F.layer_norm(t, (case["cols"],), None, None, _EPS)
        return F.rms_norm(t, (case["cols"],), None, _EPS)

    branch = normed(leaf["x"]) * leaf["post_weight"] if case["post"] else leaf["x"]
    total = leaf["residual"] * leaf.get("scale", 1.0) + branch * leaf.get("gate", 1.0)
    stored = total.detach().to(dtype).double().requires_grad_(case["train"])      # (the stored sum: rounded once, its gradient passes through)
    y = normed(stored) * leaf["weight"] + leaf["bias"]
    out = {"s": stored.detach(), "y": y.detach()}
    if case["train"]:
        ds, out["dweight"], out["dbias"] = torch.autograd.grad(y, (stored, leaf["weight"], leaf["bias"]), state["dy"].double())
        names = [name for name in leaf if name not in ("weight", "bias")]
        for name, grad in zip(names, torch.autograd.grad(total, [leaf[name] for name in names], ds + state["ds"].double())):
            out["d" + name] = grad
    return out
