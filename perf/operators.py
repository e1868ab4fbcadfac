"""What is measured of the gated feed-forward block and of the norms around a block: the cases, their inputs, the
operators in plain torch and the values that they should have.

* ``ffn``   y = W_down (act(W_gate x + b_gate) * (W_up x + b_up)) + b_down over the rows of x, inference ("forward") or
  with every gradient ("train");
* ``norm``  stream = residual_scale * residual + gate * post_norm(x),  normed = pre_norm(stream): what stands between
  two blocks of a pre-norm / sandwich-norm stack, inference or with every gradient.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_ACTIVATIONS = ("silu", "gelu", "gelu_tanh", "relu", "sigmoid")


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def _ffn(name, rows, width, hidden, dtype, direction, activation="silu", bias=False, pad=0):
    return {"name": name, "op": "ffn", "rows": rows, "width": width, "hidden": hidden, "dtype": dtype,
            "direction": direction, "activation": activation, "bias": bias, "pad": pad}


def _norm(name, batch, length, width, dtype, direction, stream, post, pre, gate, scale=1.0, params=None):
    return {"name": name, "op": "norm", "batch": batch, "length": length, "width": width, "dtype": dtype,
            "direction": direction, "stream": stream, "post": post, "pre": pre, "gate": gate, "scale": scale,
            "params": params or dtype}


def listed():
    return [
        # one token of one sequence through a large layer: the weights are read once, nothing else counts
        _ffn("ffn_one_token", 1, 4096, 11264, "bf16", "forward"),
        # a handful of sequences, one token each, in half precision; rows that are slices of a wider buffer
        _ffn("ffn_few_tokens", 13, 2048, 5632, "f16", "forward", "gelu_tanh", pad=64),
        # the decoder's 8 x 256 object queries at the decoder layer's default hidden width, with biases, in the
        # framework's own precision
        _ffn("ffn_queries_train", 2048, 288, 2048, "f32", "train", "gelu", bias=True),
        # the encoder's 8 x 1024 seed points at the model's hidden width: small matrices, many rows
        _ffn("ffn_seeds_train", 8192, 288, 256, "bf16", "train", "silu", bias=True),
        # sizes that are no multiple of anything, as pruned or concatenated features have them
        _ffn("ffn_odd_train", 1003, 777, 2051, "f16", "train", "relu", bias=True, pad=3),
        # a prompt of 2048 tokens through a large layer
        _ffn("ffn_prompt", 2048, 4096, 11264, "bf16", "forward"),
        # a training step's share of a large layer: 8192 tokens
        _ffn("ffn_large_train", 8192, 4096, 11264, "bf16", "train"),
        # four sequences, one token each: a launch's latency
        _norm("norm_few_tokens", 4, 1, 4096, "bf16", "forward", "f32", "rms", "rms", None),
        # the decoder's queries with a gate per scene and channel
        _norm("norm_queries_train", 8, 256, 288, "f32", "train", "f32", "layer", "layer", "sample", 0.8),
        # odd width and length, a gate for every element, parameters kept in 32 bits
        _norm("norm_odd_train", 3, 1001, 1537, "f16", "train", "f16", "layer", "rms", "element", 1.25, "f32"),
        # a prompt: no norm after the block, half-width stream
        _norm("norm_prompt", 4, 2048, 8192, "bf16", "forward", "bf16", None, "rms", "channel"),
        # a training step's share of a large layer, the residual stream kept in 32 bits
        _norm("norm_large_train", 8, 2048, 4096, "bf16", "train", "f32", "rms", "rms", "channel"),
    ]


def _spread(rng, low, high):
    """A size whose logarithm is spread evenly; every other one is a multiple of 16 where it is large enough."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5 and n >= 16:
        n -= n % 16
    return max(low, min(high, n))


def draw(rng):
    direction = rng.choice(["forward", "train"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if rng.random() < 0.55:
        # the matrix rate of 32-bit inputs is a sixteenth of the 16-bit one: its sizes end earlier
        wide = dtype != "f32"
        return {"op": "ffn", "rows": _spread(rng, 1, 8192 if wide else 4096),
                "width": _spread(rng, 24, 4096 if wide else 1536), "hidden": _spread(rng, 24, 11264 if wide else 4096),
                "dtype": dtype, "direction": direction, "activation": rng.choice(_ACTIVATIONS),
                "bias": rng.random() < 0.5, "pad": rng.choice([0, 0, 5, 32])}
    width = _spread(rng, 16, 8192)
    rows = _spread(rng, 1, max(1, min(16384, (1 << 26) // width)))
    batch = rng.choice([1, 2, 3, 8, 16])
    post, pre = rng.choice([("rms", "rms"), ("layer", "layer"), (None, "rms"), ("rms", None), ("layer", "rms"), (None, "layer")])
    return {"op": "norm", "batch": batch, "length": max(1, rows // batch), "width": width, "dtype": dtype,
            "direction": direction, "stream": rng.choice([dtype, "f32"]), "post": post, "pre": pre,
            "gate": rng.choice([None, "channel", "sample", "element"]), "scale": rng.choice([1.0, 0.8, 1.25]),
            "params": rng.choice([dtype, "f32"])}


def work(case):
    size = _SIZE[case["dtype"]]
    train = case["direction"] == "train"
    if case["op"] == "ffn":
        m, e, f = case["rows"], case["width"], case["hidden"]
        weights = (3 * e * f + (2 * f + e if case["bias"] else 0)) * size
        rows = m * e * size
        # forward: x, weights in, y out; train: dy in, d_x and the weights' gradients out as well
        return {"bytes": (2 * weights + 4 * rows) if train else (weights + 2 * rows),
                "flops": (18 if train else 6) * m * e * f}
    n = case["batch"] * case["length"]
    c, stream, params = case["width"], _SIZE[case["stream"]], _SIZE[case["params"]]
    vectors = {None: 0, "rms": 1, "layer": 2}
    small = (vectors[case["post"]] + vectors[case["pre"]]) * c * params
    small += {None: 0, "channel": c, "sample": case["batch"] * c, "element": n * c}[case["gate"]] * size
    normed = size if case["pre"] else 0
    once = n * c * (size + 2 * stream + normed)            # x, residual in; stream, normed out
    if not train:
        return {"bytes": once + small, "flops": 12 * n * c}
    # d_stream, d_normed in; d_x, d_residual and the parameters' gradients out
    return {"bytes": once + n * c * (2 * stream + normed + size) + 2 * small, "flops": 36 * n * c}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _normal(gen, shape, scale=1.0, shift=0.0, dtype=torch.float32):
    return (torch.randn(shape, device="cuda", generator=gen) * scale + shift).to(dtype)


def _padded(t, pad):
    """The same values as rows of a buffer that is ``pad`` elements wider."""
    if not pad:
        return t
    buf = torch.zeros(t.shape[0], t.shape[1] + pad, device=t.device, dtype=t.dtype)
    buf[:, :t.shape[1]] = t
    return buf[:, :t.shape[1]]


def _norm_module(gen, kind, width, dtype):
    if kind is None:
        return None
    cls = torch.nn.RMSNorm if kind == "rms" else torch.nn.LayerNorm
    module = cls(width, eps=1e-6 if kind == "rms" else 1e-5, device="cuda", dtype=dtype)
    with torch.no_grad():
        module.weight.copy_(_normal(gen, width, 0.2, 1.0))
        if kind == "layer":
            module.bias.copy_(_normal(gen, width, 0.1))
    return module


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = _DTYPES[case["dtype"]]
    train = case["direction"] == "train"
    if case["op"] == "ffn":
        m, e, f = case["rows"], case["width"], case["hidden"]
        leaves = {"x": _padded(_normal(gen, (m, e), dtype=dtype), case["pad"]),
                  "w_gate": _normal(gen, (f, e), e ** -0.5, dtype=dtype),
                  "w_up": _normal(gen, (f, e), e ** -0.5, dtype=dtype),
                  "w_down": _normal(gen, (e, f), f ** -0.5, dtype=dtype)}
        if case["bias"]:
            leaves.update(b_gate=_normal(gen, f, 0.2, dtype=dtype), b_up=_normal(gen, f, 0.2, dtype=dtype),
                          b_down=_normal(gen, e, 0.2, dtype=dtype))
        state = {"case": case, "leaves": leaves}
        if train:
            state["d_y"] = _normal(gen, (m, e), 0.1, dtype=dtype)
    else:
        b, l, c = case["batch"], case["length"], case["width"]
        stream, params = _DTYPES[case["stream"]], _DTYPES[case["params"]]
        # a residual stream is larger than what a block adds to it, and some of its channels stand out
        loud = 1.0 + 7.0 * (torch.rand(c, device="cuda", generator=gen) < 0.01)
        leaves = {"x": _normal(gen, (b, l, c), 0.7, 0.1, dtype),
                  "residual": (_normal(gen, (b, l, c), 2.0, 0.3) * loud).to(stream)}
        shape = {None: None, "channel": (c,), "sample": (b, c), "element": (b, l, c)}[case["gate"]]
        if shape is not None:
            leaves["gate"] = _normal(gen, shape, 0.4, 0.5, dtype)
        state = {"case": case, "leaves": leaves, "post": _norm_module(gen, case["post"], c, params),
                 "pre": _norm_module(gen, case["pre"], c, params)}
        for which in ("post", "pre"):
            module = state[which]
            if module is not None:
                module.requires_grad_(train)
                leaves[which + "_weight"] = module.weight
                if case[which] == "layer":
                    leaves[which + "_bias"] = module.bias
        if train:
            state["d_stream"] = _normal(gen, (b, l, c), 0.1, dtype=stream)
            if case["pre"]:
                state["d_normed"] = _normal(gen, (b, l, c), 0.1, dtype=dtype)
    for t in leaves.values():
        t.requires_grad_(train)
    return state


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    forward = _forward_own if own else _forward_plain
    leaves = state["leaves"]
    if state["case"]["direction"] == "forward":
        with torch.no_grad():
            return _rounded(state, forward(state, leaves if own else _wide(leaves)))
    given = leaves if own else {k: t.requires_grad_(True) for k, t in _wide(leaves).items()}
    out = forward(state, given)
    gradients = [state["d_" + k] if own else state["d_" + k].float() for k in out]
    back = torch.autograd.grad(list(out.values()), list(given.values()), gradients)
    return _rounded(state, {**out, **{"d_" + k: g for k, g in zip(given, back)}})


def _wide(leaves):
    return {k: t.detach().float() for k, t in leaves.items()}


def _rounded(state, out):
    """Every output in its own type (the framework's have it already)."""
    leaves = state["leaves"]
    types = {"y": leaves["x"].dtype, "normed": leaves["x"].dtype}
    if "residual" in leaves:
        types["stream"] = leaves["residual"].dtype
    types.update({"d_" + k: t.dtype for k, t in leaves.items()})
    return {k: t.detach().to(types[k]) for k, t in out.items()}


def _forward_own(state, t):
    case = state["case"]
    if case["op"] == "ffn":
        from butd_detr_amd.gated_ffn import gated_ffn
        return {"y": gated_ffn(t["x"], t["w_gate"], t["w_up"], t["w_down"], t.get("b_gate"), t.get("b_up"),
                               t.get("b_down"), activation=case["activation"])}
    from butd_detr_amd.residual_norm import residual_norm
    stream, normed = residual_norm(t["x"], t["residual"], post_norm=state["post"], gate=t.get("gate"),
                                   residual_scale=case["scale"], pre_norm=state["pre"])
    return {"stream": stream} if normed is None else {"stream": stream, "normed": normed}


def _activate(a, kind):
    if kind == "silu":
        return a * torch.sigmoid(a)
    if kind == "gelu":
        return 0.5 * a * (1.0 + torch.erf(a * math.sqrt(0.5)))
    if kind == "gelu_tanh":
        return 0.5 * a * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (a + 0.044715 * a * a * a)))
    if kind == "relu":
        return a * (a > 0)
    return torch.sigmoid(a)


def _normalize(v, kind, weight, bias, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * weight
    return v if bias is None else v + bias


def _forward_plain(state, t):
    case = state["case"]
    if case["op"] == "ffn":
        a, b = t["x"] @ t["w_gate"].t(), t["x"] @ t["w_up"].t()
        if case["bias"]:
            a, b = a + t["b_gate"], b + t["b_up"]
        y = (_activate(a, case["activation"]) * b) @ t["w_down"].t()
        return {"y": y + t["b_down"] if case["bias"] else y}
    v = t["x"]
    if case["post"]:
        v = _normalize(v, case["post"], t["post_weight"], t.get("post_bias"), state["post"].eps)
    if case["gate"]:
        v = v * (t["gate"][:, None, :] if case["gate"] == "sample" else t["gate"])
    stream = case["scale"] * t["residual"] + v
    if not case["pre"]:
        return {"stream": stream}
    return {"stream": stream, "normed": _normalize(stream, case["pre"], t["pre_weight"], t.get("pre_bias"), state["pre"].eps)}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, its derivatives by hand
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    t = {k: v.detach().double() for k, v in state["leaves"].items()}
    for k in ("d_y", "d_stream", "d_normed"):
        if k in state:
            t[k] = state[k].double()
    return _exact_ffn(case, t) if case["op"] == "ffn" else _exact_norm(case, state, t)


def _act_and_slope(a, kind):
    if kind == "relu":
        live = (a > 0).double()
        return a * live, live
    if kind in ("silu", "sigmoid"):
        s = 1.0 / (1.0 + torch.exp(-a))
        return (s, s * (1.0 - s)) if kind == "sigmoid" else (a * s, s * (1.0 + a * (1.0 - s)))
    if kind == "gelu":
        cdf = 0.5 * torch.erfc(-a / math.sqrt(2.0))
        return a * cdf, cdf + a * torch.exp(-0.5 * a * a) / math.sqrt(2.0 * math.pi)
    k = math.sqrt(2.0 / math.pi)
    th = torch.tanh(k * (a + 0.044715 * a ** 3))
    return 0.5 * a * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * a * (1.0 - th * th) * k * (1.0 + 3.0 * 0.044715 * a * a)


def _exact_ffn(case, t):
    zero = torch.zeros((), device="cuda", dtype=torch.float64)
    a = torch.addmm(t["b_gate"] if case["bias"] else zero, t["x"], t["w_gate"].t())
    b = torch.addmm(t["b_up"] if case["bias"] else zero, t["x"], t["w_up"].t())
    act, slope = _act_and_slope(a, case["activation"])
    h = act * b
    out = {"y": torch.addmm(t["b_down"] if case["bias"] else zero, h, t["w_down"].t())}
    if case["direction"] == "forward":
        return out
    d_h = t["d_y"] @ t["w_down"]
    d_a, d_b = d_h * b * slope, d_h * act
    out["d_x"] = d_a @ t["w_gate"] + d_b @ t["w_up"]
    out["d_w_gate"], out["d_w_up"], out["d_w_down"] = d_a.t() @ t["x"], d_b.t() @ t["x"], t["d_y"].t() @ h
    if case["bias"]:
        out["d_b_gate"], out["d_b_up"], out["d_b_down"] = d_a.sum(0), d_b.sum(0), t["d_y"].sum(0)
    return out


def _unit(v, kind, eps):
    """Normalised values and 1 / deviation of every row."""
    if kind == "layer":
        v = v - v.sum(-1, keepdim=True) / v.shape[-1]
    inverse = ((v ** 2).sum(-1, keepdim=True) / v.shape[-1] + eps) ** -0.5
    return v * inverse, inverse


def _unit_backward(g, unit, inverse, kind):
    n = g.shape[-1]
    back = g - unit * ((g * unit).sum(-1, keepdim=True) / n)
    if kind == "layer":
        back = back - g.sum(-1, keepdim=True) / n
    return back * inverse


def _exact_norm(case, state, t):
    post, pre = case["post"], case["pre"]
    branch = t["x"]
    if post:
        unit, inverse = _unit(t["x"], post, state["post"].eps)
        branch = unit * t["post_weight"] + t.get("post_bias", 0.0)
    gate = {None: lambda: 1.0, "sample": lambda: t["gate"][:, None, :]}.get(case["gate"], lambda: t["gate"])()
    stream = case["scale"] * t["residual"] + gate * branch
    out = {"stream": stream}
    if pre:
        unit2, inverse2 = _unit(stream, pre, state["pre"].eps)
        out["normed"] = unit2 * t["pre_weight"] + t.get("pre_bias", 0.0)
    if case["direction"] == "forward":
        return out
    d = t["d_stream"]
    if pre:
        d = d + _unit_backward(t["d_normed"] * t["pre_weight"], unit2, inverse2, pre)
    d_branch = d * gate
    grads = {"x": _unit_backward(d_branch * t["post_weight"], unit, inverse, post) if post else d_branch,
             "residual": case["scale"] * d}
    if case["gate"]:
        axes = {"channel": (0, 1), "sample": (1,)}.get(case["gate"])
        grads["gate"] = d * branch if axes is None else (d * branch).sum(axes)
    if post:
        grads["post_weight"] = (d_branch * unit).sum((0, 1))
        if post == "layer":
            grads["post_bias"] = d_branch.sum((0, 1))
    if pre:
        grads["pre_weight"] = (t["d_normed"] * unit2).sum((0, 1))
        if pre == "layer":
            grads["pre_bias"] = t["d_normed"].sum((0, 1))
    return {**out, **{"d_" + k: grads[k] for k in state["leaves"]}}
