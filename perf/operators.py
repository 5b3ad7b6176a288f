"""The operators around a product that a transformer block's forward and backward pass is made of, as timed cases.

Three operators of the package, in their plain form (elementary torch operations in 32 bits) and, with ``own`` set, as a
user's program calls them:

* ``norm``: ``layer_norm(x, weight, bias)``;
* ``add_norm``: ``add_layer_norm(x, residual, weight, bias)``, the residual stream's sum and its norm.  The norm is
  taken of the sum as it is stored (rounded to the tensors' type), which is what the block goes on with;
* ``linear``: ``cascaded_lowp_matmul_epilogue(a, b, bias=, activation=, residual=)``: activation(a b + bias) + residual.

A case is ``{kind, train, dtype, rows, k, n, activation, residual, prepared}``.  ``rows``: tokens; norms have ``k``
columns (``n`` is 0), products ``k`` inputs and ``n`` outputs.  ``train``: the gradients of all floating inputs too, for a
given gradient of the result.  fp32 products run with three fp16 terms (fp32's own accuracy), 16-bit ones as one term of
their own format.  ``prepared``: the weight is kept re-laid between calls, as a serving program keeps it.

Activations are N(0, 1) with a spread of scales and means over the columns, as a residual stream has them; weights of
products N(0, 0.02), of norms around one.
"""
import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5


def _case(kind, rows, k, n=0, *, dtype="fp32", train=False, activation="none", residual=False, prepared=False, name=None):
    c = {"kind": kind, "train": train, "dtype": dtype, "rows": rows, "k": k, "n": n, "activation": activation, "residual": residual, "prepared": prepared}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # two rows (the guided batch's pooled conditioning): nothing but latency
        _case("norm", 2, 1280, name="norm_pooled_fp32"),
        # the norms of a transformer block at the 64 x 64 stage, guided batch of two, in the dtype UNets are run in
        _case("norm", 8192, 640, dtype="fp16", name="norm_tokens_fp16"),
        # residual add and norm at the 32 x 32 stage of an 832 x 1216 image (2 x 26 x 38 tokens)
        _case("add_norm", 1976, 1280, dtype="bf16", name="add_norm_bucket_bf16"),
        # the same norm while its weights are trained, in fp32
        _case("norm", 8192, 640, train=True, name="norm_train_fp32"),
        # a training batch of 64 images at the 32 x 32 stage: bytes, and a long reduction for the weights' gradients
        _case("norm", 65536, 1280, dtype="bf16", train=True, name="norm_train_large_bf16"),
        # no dimension a multiple of anything, the residual stream's gradient coming in from both sides
        _case("add_norm", 2333, 457, train=True, name="add_norm_train_ragged_fp32"),
        # time embedding's first layer with its activation, on the guided batch
        _case("linear", 2, 320, 1280, activation="silu", name="embedding_silu_fp32"),
        # up-projection of a text encoder's feed-forward block on 2 x 77 tokens, weight kept re-laid
        _case("linear", 154, 1280, 5120, dtype="fp16", activation="gelu", prepared=True, name="text_up_gelu_fp16"),
        # attention's output projection at the 32 x 32 stage, added to the residual stream: the most frequent layer of a step
        _case("linear", 2048, 1280, 1280, dtype="fp16", residual=True, prepared=True, name="proj_out_residual_fp16"),
        # the down-projection of the feed-forward block with fp32's accuracy
        _case("linear", 2048, 5120, 1280, residual=True, name="ffn_down_residual_fp32"),
        # a feed-forward block's first layer while it is trained (64 x 64 stage)
        _case("linear", 8192, 640, 2560, dtype="bf16", activation="gelu", train=True, name="ffn_up_train_bf16"),
        # a ragged layer in training, with everything an epilogue can hold
        _case("linear", 333, 456, 211, dtype="fp16", activation="silu", residual=True, train=True, name="ragged_train_fp16"),
    ]


#: elements of the largest listed norm, multiply-adds of the largest listed products (16-bit, and fp32)
_MOST_ELEMENTS = 65536 * 1280
_MOST_MACS = {"fp32": 2048 * 5120 * 1280, "fp16": 3 * 8192 * 640 * 2560, "bf16": 3 * 8192 * 640 * 2560}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Layer widths: mostly multiples of 64, some of 8, some anything."""
    x, r = _log(rng, lo, hi), rng.random()
    unit = 64 if r < 0.6 else 8 if r < 0.8 else 1
    return max(unit, (x + unit // 2) // unit * unit)


def draw(rng):
    kind = rng.choice(("norm", "add_norm", "linear", "linear"))
    dtype = rng.choice(("fp32", "fp16", "bf16"))
    train = rng.random() < 0.5
    if kind != "linear":
        k = _width(rng, 64, 2560)
        rows = _log(rng, 1, 65536)
        most = _MOST_ELEMENTS // (2 if dtype == "fp32" else 1) // (2 if kind == "add_norm" else 1)
        return _case(kind, max(1, min(rows, most // k)), k, dtype=dtype, train=train)
    k, n = _width(rng, 64, 5120), _width(rng, 64, 5120)
    rows = _log(rng, 1, 8192)
    passes = 3 if train else 1
    rows = max(1, min(rows, int(0.9 * _MOST_MACS[dtype]) // (passes * k * n)))
    return _case(kind, rows, k, n, dtype=dtype, train=train, activation=rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu")),
                 residual=rng.random() < 0.5, prepared=not train and dtype != "fp32" and rng.random() < 0.5)


def work(case):
    rows, k, n = case["rows"], case["k"], case["n"]
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] != "linear":
        streams = {("norm", False): 2, ("norm", True): 4, ("add_norm", False): 4, ("add_norm", True): 7}[case["kind"], case["train"]]
        weights = 4 if case["train"] else 2      # (weight and bias; their gradients)
        return {"bytes": size * (streams * rows * k + weights * k), "flops": (26 if case["train"] else 8) * rows * k}
    values = rows * k + k * n + n + rows * n + (rows * n if case["residual"] else 0)
    passes = 1
    if case["train"]:   # (the result's gradient in; the gradients of a, b and bias out; the residual's is the result's)
        passes = 3
        values += rows * n + rows * k + k * n + n
    return {"bytes": size * values, "flops": 2 * passes * rows * k * n}


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, rows, k, n = _DTYPES[case["dtype"]], case["rows"], case["k"], case["n"]

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * std + mean).to(dtype)

    def stream(width):
        spread = torch.exp(0.5 * torch.randn(width, device="cuda", generator=gen))
        means = 0.5 * torch.randn(width, device="cuda", generator=gen)
        return (torch.randn(rows, width, device="cuda", generator=gen) * spread + means).to(dtype)

    state = {key: case[key] for key in ("kind", "train", "activation", "dtype")}
    width = n if case["kind"] == "linear" else k
    if case["kind"] == "linear":
        state["leaves"] = {"a": normal(rows, k), "b": normal(k, n, std=0.02), "bias": normal(n, std=0.02)}
        if case["residual"]:
            state["leaves"]["residual"] = stream(n)
    else:
        state["leaves"] = {"x": stream(k), "weight": normal(k, std=0.1, mean=1.0), "bias": normal(k, std=0.1)}
        if case["kind"] == "add_norm":
            state["leaves"]["residual"] = stream(k)
    if case["train"]:
        state["dy"] = normal(rows, width)
        if case["kind"] == "add_norm":
            state["ds"] = normal(rows, width)
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    if case["train"]:
        for leaf in state["leaves"].values():
            leaf.requires_grad_(True)
    if own and case["prepared"]:
        from basedxl_amd import PreparedWeight
        state["kept"] = PreparedWeight(state["leaves"]["b"])
    return state


# ---- plain forms ----
def _activate(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    if name == "gelu_tanh":
        t = torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return torch.ones_like(z)


def _plain_norm(state):
    leaf = {name: t.detach() for name, t in state["leaves"].items()}
    dtype = leaf["x"].dtype
    x = leaf["x"].float()
    out = {}
    if state["kind"] == "add_norm":
        s = (x + leaf["residual"].float()).to(dtype)
        out["sum"] = s
        x = s.float()
    w = leaf["weight"].float()
    centred = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + _EPS)
    xhat = centred * rstd
    out["y"] = (xhat * w + leaf["bias"].float()).to(dtype)
    if state["train"]:
        dy = state["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
        if state["kind"] == "add_norm":
            dx = dx + state["ds"].float()
            out["dresidual"] = dx.to(dtype)
        out["dx"] = dx.to(dtype)
        out["dweight"] = (dy * xhat).sum(0).to(dtype)
        out["dbias"] = dy.sum(0).to(dtype)
    return out


def _plain_linear(state):
    leaf = {name: t.detach() for name, t in state["leaves"].items()}
    dtype = leaf["a"].dtype
    a, b = leaf["a"].float(), leaf["b"].float()
    z = a @ b + leaf["bias"].float()
    y = _activate(z, state["activation"])
    if "residual" in leaf:
        y = y + leaf["residual"].float()
    out = {"y": y.to(dtype)}
    if state["train"]:
        dy = state["dy"].float()
        dz = dy * _slope(z, state["activation"])
        out["da"] = (dz @ b.t().contiguous()).to(dtype)
        out["db"] = (a.t().contiguous() @ dz).to(dtype)
        out["dbias"] = dz.sum(0).to(dtype)
        if "residual" in leaf:
            out["dresidual"] = state["dy"]
    return out


# ---- the package's calls ----
def _own_norm(state):
    from basedxl_amd import add_layer_norm, layer_norm
    leaf = state["leaves"]
    if state["kind"] == "norm":
        y = layer_norm(leaf["x"], leaf["weight"], leaf["bias"], eps=_EPS)
        if not state["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (leaf["x"], leaf["weight"], leaf["bias"]), state["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    y, s = add_layer_norm(leaf["x"], leaf["residual"], leaf["weight"], leaf["bias"], eps=_EPS)
    if not state["train"]:
        return {"sum": s, "y": y}
    dx, dr, dw, db = torch.autograd.grad((y, s), (leaf["x"], leaf["residual"], leaf["weight"], leaf["bias"]), (state["dy"], state["ds"]))
    return {"sum": s.detach(), "y": y.detach(), "dresidual": dr, "dx": dx, "dweight": dw, "dbias": db}


def _own_linear(state):
    from basedxl_amd import cascaded_lowp_matmul_epilogue
    leaf = state["leaves"]
    options = {"lowp": "fp16", "terms": 3} if state["dtype"] == "fp32" else {}
    activation = None if state["activation"] == "none" else state["activation"]
    y = cascaded_lowp_matmul_epilogue(leaf["a"], state.get("kept", leaf["b"]), bias=leaf["bias"], activation=activation, residual=leaf.get("residual"), **options)
    if not state["train"]:
        return {"y": y}
    wrt = tuple(leaf[name] for name in ("a", "b", "bias", "residual") if name in leaf)
    grads = torch.autograd.grad(y, wrt, state["dy"])
    out = {"y": y.detach(), "da": grads[0], "db": grads[1], "dbias": grads[2]}
    if "residual" in leaf:
        out["dresidual"] = grads[3]
    return out


def run(state):
    if own:
        return _own_linear(state) if state["kind"] == "linear" else _own_norm(state)
    return _plain_linear(state) if state["kind"] == "linear" else _plain_norm(state)


# ---- the definition, in 64 bits: torch's own functions and its autograd ----
def exact(case, seed):
    state = _inputs(case, seed)
    dtype = _DTYPES[case["dtype"]]
    leaf = {name: t.double().requires_grad_(case["train"]) for name, t in state["leaves"].items()}
    F = torch.nn.functional
    if case["kind"] == "linear":
        f = {"none": lambda z: z, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}[case["activation"]]
        y = f(F.linear(leaf["a"], leaf["b"].t(), leaf["bias"]))
        if case["residual"]:
            y = y + leaf["residual"]
        out = {"y": y.detach()}
        if case["train"]:
            names = [name for name in ("a", "b", "bias", "residual") if name in leaf]
            for name, grad in zip(names, torch.autograd.grad(y, [leaf[name] for name in names], state["dy"].double())):
                out["d" + name] = grad
        return out
    if case["kind"] == "norm":
        x, out = leaf["x"], {}
    else:   # (the stored sum: rounded once, its gradient passes through)
        stored = (state["leaves"]["x"].float() + state["leaves"]["residual"].float()).to(dtype).double()
        x = stored.requires_grad_(case["train"])
        out = {"sum": stored.detach()}
    y = F.layer_norm(x, (case["k"],), leaf["weight"], leaf["bias"], _EPS)
    out["y"] = y.detach()
    if case["train"]:
        dx, dw, db = torch.autograd.grad(y, (x, leaf["weight"], leaf["bias"]), state["dy"].double())
        if case["kind"] == "add_norm":
            dx = dx + state["ds"].double()
            out["dresidual"] = dx
        out.update(dx=dx, dweight=dw, dbias=db)
    return out
