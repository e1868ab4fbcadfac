"""-m gpu: norms before and after a block with its gate and residual scale (include/butd_residual_norm.h) against the
formulas in 64 bits.

Tolerances are elementwise bounds carried through the formulas.  Every output is rounded once to its type (u = ``eps / 2`` of
itself).  Inside, 32 bits: an element-wise step is off by at most 2^-23 of its value; a sum over a row of c elements (eight in
a thread, then a tree over lanes and waves: at most 8 + 6 + 16 additions in a chain) by 32 * 2^-24 of the sum of magnitudes,
taken here as E = 2^-18 to cover the statistics' division and square root; a column sum over r rows by (r + 32) 2^-24 of its
magnitudes."""
import itertools

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

E = 2.0 ** -18
TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
         (torch.float16, torch.float16), (torch.float16, torch.float32)]
KINDS = [("rms", "rms"), ("layer", "layer"), (None, "rms"), ("rms", None), ("layer", "rms"), (None, "layer"), (None, None)]


def norm_of(kind, cols, dtype, affine=True, bias=True):
    if kind is None:
        return None
    m = (nn.RMSNorm(cols, eps=1e-6, elementwise_affine=affine) if kind == "rms"
         else nn.LayerNorm(cols, eps=1e-5, elementwise_affine=affine, bias=bias))
    with torch.no_grad():
        for p in m.parameters():
            p.copy_(torch.randn(cols) * 0.2 + (1.0 if p is m.weight else 0.0))
    return m.to("cuda", dtype)


def inputs(batch, length, cols, dtype, stream, post, pre, gate, params=None, seed=0):
    torch.manual_seed(1000 * seed + batch + 7 * length + 31 * cols)
    n = lambda *s: torch.randn(*s, device="cuda")                                                  # noqa: E731
    t = {"x": (n(batch, length, cols) * 0.7 + 0.1).to(dtype), "residual": (n(batch, length, cols) * 2 + 0.3).to(stream)}
    if gate:
        shape = {"channel": (cols,), "sample": (batch, cols), "element": (batch, length, cols)}[gate]
        t["gate"] = (n(*shape) * 0.4 + 0.5).to(dtype)
    norms = {"post": norm_of(post, cols, params or dtype), "pre": norm_of(pre, cols, params or dtype)}
    d = {"stream": (n(batch, length, cols) * 0.3).to(stream)}
    if pre:
        d["normed"] = (n(batch, length, cols) * 0.3).to(dtype)
    return t, norms, d


def unit(v, ev, kind, eps):
    """(normalised, its error, 1 / deviation, its relative error): v is known to +- ev"""
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    size = v.abs().mean(-1, keepdim=True)
    ec = ev + ev.mean(-1, keepdim=True) + (E * size if kind == "layer" else 0.0) + 2.0 ** -23 * (v.abs() + mean.abs())
    c = v - mean
    var = (c * c).mean(-1, keepdim=True) + eps
    rstd = var.rsqrt()
    er = E + (c.abs() * ec + ec * ec).mean(-1, keepdim=True) / var
    n = c * rstd
    return n, ec * rstd + n.abs() * er + ec * rstd * er, rstd, er


def unit_back(g, eg, n, en, rstd, er, kind):
    """gradient through ``unit``: rstd (g - mean(g) - n mean(g n))"""
    m1, a1 = (g * n).mean(-1, keepdim=True), (g * n).abs().mean(-1, keepdim=True)
    e1 = E * a1 + (eg * n.abs() + g.abs() * en + eg * en).mean(-1, keepdim=True)
    m0 = g.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(m1)
    e0 = E * g.abs().mean(-1, keepdim=True) + eg.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(m1)
    v = g - m0 - n * m1
    size = g.abs() + m0.abs() + (n * m1).abs()
    ev = eg + e0 + n.abs() * e1 + en * (m1.abs() + e1) + 2.0 ** -22 * size
    return rstd * v, rstd * (ev + er * (v.abs() + ev))


def reference(t, norms, d, scale, residual=True):
    """{output: (value, bound)} in 64 bits; an output's own rounding is added in ``check``"""
    v = {k: p.detach().double() for k, p in t.items()}
    x = v["x"]
    cols, rows = x.shape[-1], x[..., 0].numel()
    w = lambda m, name: (getattr(m, name, None) if m is not None else None)                        # noqa: E731
    val = lambda p, other: other if p is None else p.detach().double()                             # noqa: E731
    post, pre = norms["post"], norms["pre"]
    kind = lambda m: None if m is None else "layer" if isinstance(m, nn.LayerNorm) else "rms"      # noqa: E731
    w1, b1, w2, b2 = val(w(post, "weight"), 1.0), val(w(post, "bias"), 0.0), val(w(pre, "weight"), 1.0), val(w(pre, "bias"), 0.0)
    zero = torch.zeros_like(x)
    if post is not None:
        n1, en1, r1, er1 = unit(x, zero, kind(post), post.eps)
    else:
        n1, en1 = x, zero
    gate = v.get("gate")
    g = 1.0 if gate is None else gate[:, None] if gate.dim() == 2 else gate
    ga = abs(g)
    t1 = n1 * w1 + b1
    et = en1 * abs(w1) + 2.0 ** -22 * (abs(n1 * w1) + abs(b1))
    res = scale * v["residual"] if residual else zero
    s = res + g * t1
    es = ga * et + 2.0 ** -22 * (res.abs() + (g * t1).abs())
    out = {"stream": (s, es)}
    ds, eds = (d["stream"].double() if "stream" in d else zero), zero
    if pre is not None:
        n2, en2, r2, er2 = unit(s, es, kind(pre), pre.eps)
        out["normed"] = (n2 * w2 + b2, en2 * abs(w2) + 2.0 ** -22 * (abs(n2 * w2) + abs(b2)))
        if "normed" in d:
            dn = d["normed"].double()
            back, eback = unit_back(dn * w2, 2.0 ** -23 * (dn * w2).abs(), n2, en2, r2, er2, kind(pre))
            eds = eback + 2.0 ** -23 * (ds.abs() + back.abs())
            ds = ds + back
        else:
            dn = zero
    axes = tuple(range(x.dim() - 1))
    col = lambda p, ep, ax: (p.sum(ax), ep.sum(ax) + (rows + 32) * 2.0 ** -24 * p.abs().sum(ax))   # noqa: E731
    out["d_residual"] = (scale * ds, abs(scale) * eds + 2.0 ** -23 * abs(scale) * ds.abs())
    dg = ds * t1
    edg = eds * t1.abs() + ds.abs() * et + eds * et + 2.0 ** -23 * dg.abs()
    if gate is not None:
        out["d_gate"] = (dg, edg) if gate.dim() == 3 else col(dg, edg, axes if gate.dim() == 1 else (1,))
    dt, edt = ds * g, eds * ga + 2.0 ** -23 * (ds * g).abs()
    if post is None:
        out["d_x"] = (dt, edt)
    else:
        out["d_x"] = unit_back(dt * w1, edt * abs(w1) + 2.0 ** -23 * (dt * w1).abs(), n1, en1, r1, er1, kind(post))
        p = dt * n1
        out["d_post_weight"] = col(p, edt * n1.abs() + dt.abs() * en1 + edt * en1 + 2.0 ** -23 * p.abs(), axes)
        out["d_post_bias"] = col(dt, edt, axes)
    if pre is not None:
        p = dn * n2
        out["d_pre_weight"] = col(p, dn.abs() * en2 + 2.0 ** -23 * p.abs(), axes)
        out["d_pre_bias"] = col(dn, zero, axes)
    return out


def run(t, norms, d, scale, residual=True, train=True, only=None):
    from butd_detr_amd.residual_norm import residual_norm
    leaves = {k: p.detach().requires_grad_(train) for k, p in t.items() if residual or k != "residual"}
    for which, m in norms.items():
        if m is not None:
            m.requires_grad_(train)
            for name, p in m.named_parameters():
                leaves[f"{which}_{name}"] = p
    stream, normed = residual_norm(leaves["x"], leaves.get("residual"), post_norm=norms["post"], gate=leaves.get("gate"),
                                   residual_scale=scale, pre_norm=norms["pre"])
    out = {"stream": stream} | ({} if normed is None else {"normed": normed})
    if not train:
        return out
    arriving = [k for k in out if k in d and out[k].requires_grad]
    names = [k for k in leaves if only is None or k in only]
    grads = torch.autograd.grad([out[k] for k in arriving], [leaves[k] for k in names], [d[k] for k in arriving], allow_unused=True)
    return {k: v.detach() for k, v in out.items()} | {"d_" + k: g for k, g in zip(names, grads) if g is not None}


def check(got, want, what):
    for k, v in got.items():
        value, bound = want[k]
        assert v.shape == value.shape, (what, k, v.shape, value.shape)
        u = torch.finfo(v.dtype).eps / 2
        tiny = 2.0 ** -25 if v.dtype == torch.float16 else 0.0
        off = (v.double() - value).abs() - (bound * (1 + 2.0 ** -10) + u * (value.abs() + bound) + tiny)
        assert not torch.isnan(v).any() and float(off.max()) <= 0, (what, k, float(off.max()), float(bound.max()))


# widths: within one thread, odd, the layers' 288, either side of every workgroup size, the widest
WIDTHS = [1, 7, 16, 288, 511, 512, 513, 1024, 1537, 2050, 4096, 4100, 8191, 8192]


@pytest.mark.parametrize("dtype, stream", TYPES)
@pytest.mark.parametrize("cols", WIDTHS)
def test_widths(cols, dtype, stream):
    for i, ((post, pre), gate) in enumerate(zip(KINDS, ["channel", "sample", None, "element", "sample", "channel", "element"])):
        t, norms, d = inputs(3, 5, cols, dtype, stream, post, pre, gate, params=torch.float32 if i % 2 else None)
        want = reference(t, norms, d, 0.75)
        check(run(t, norms, d, 0.75), want, (cols, dtype, stream, post, pre, gate))
        check(run(t, norms, d, 0.75, train=False), want, (cols, dtype, stream, post, pre, gate, "inference"))


# lengths around the rows of a workgroup: whole samples in one, samples cut into several, one row a sample
@pytest.mark.parametrize("batch, length", [(1, 1), (5, 1), (1, 9), (300, 2), (7, 3), (2, 700), (4, 2500), (3, 1001), (2500, 5)])
@pytest.mark.parametrize("gate", [None, "channel", "sample", "element"])
@pytest.mark.parametrize("cols", [24, 600])
def test_row_shares(cols, gate, batch, length):
    t, norms, d = inputs(batch, length, cols, torch.bfloat16, torch.float32, "layer", "rms", gate)
    check(run(t, norms, d, 1.25), reference(t, norms, d, 1.25), (cols, gate, batch, length))


@pytest.mark.parametrize("dtype, stream", TYPES[:3])
@pytest.mark.parametrize("post, pre", KINDS)
def test_without_residual_and_with_one_gradient(post, pre, dtype, stream):
    stream = dtype
    t, norms, d = inputs(2, 40, 72, dtype, stream, post, pre, "channel")
    want = reference(t, norms, d, 1.0, residual=False)
    check(run(t, norms, d, 1.0, residual=False), {k: v for k, v in want.items() if k != "d_residual"}, (post, pre, dtype))
    for k in list(d):
        one = {k: d[k]}
        check(run(t, norms, one, 0.5), reference(t, norms, one, 0.5), (post, pre, dtype, k))
    if pre:      # a norm alone: the stream is x itself
        from butd_detr_amd.residual_norm import residual_norm
        x = t["x"].detach().requires_grad_(True)
        s, n = residual_norm(x, pre_norm=norms["pre"])
        assert s is x
        bare = {"x": t["x"], "residual": torch.zeros_like(t["x"])}
        only = {"normed": d["normed"]}
        want = reference(bare, {"post": None, "pre": norms["pre"]}, only, 1.0)
        (g,) = torch.autograd.grad(n, x, d["normed"])
        check({"normed": n.detach(), "d_x": g}, want, "norm alone")
    if post is None and pre is None:
        from butd_detr_amd.residual_norm import residual_norm
        assert residual_norm(t["x"])[0] is t["x"]


def test_norms_without_parameters_and_partial_gradients():
    t, _, d = inputs(2, 30, 264, torch.bfloat16, torch.float32, "rms", "layer", "sample")
    for post, pre in [(norm_of("rms", 264, None, affine=False), norm_of("layer", 264, None, affine=False)),
                      (norm_of("layer", 264, torch.bfloat16, bias=False), norm_of("layer", 264, torch.float32, bias=False))]:
        norms = {"post": post, "pre": pre}
        want = reference(t, norms, d, 1.0)
        check(run(t, norms, d, 1.0), want, "no parameters")
        for only in (["x"], ["residual"], ["gate"], ["x", "gate"]):
            check(run(t, norms, d, 1.0, only=only), want, only)


def test_default_epsilon_and_constant_rows():
    """RMSNorm(eps=None) is the type's eps; a row of one value has deviation 0: eps alone carries the LayerNorm"""
    from butd_detr_amd.residual_norm import residual_norm
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        m = nn.RMSNorm(40, device="cuda", dtype=dtype)
        x = torch.randn(3, 40, device="cuda").to(dtype)
        x[1] = 0
        got = residual_norm(x, pre_norm=m)[1].double()
        want = x.double() * ((x.double() ** 2).mean(-1, keepdim=True) + torch.finfo(dtype).eps).rsqrt()
        assert float(((got - want).abs() - want.abs() * (torch.finfo(dtype).eps / 2 + E)).max()) <= 0
        x = torch.full((2, 40), 3.0, device="cuda", dtype=dtype)
        ln = nn.LayerNorm(40, device="cuda", dtype=dtype)
        assert float(residual_norm(x, pre_norm=ln)[1].abs().max()) == 0.0


def test_infinities_and_nan_stay_in_their_rows():
    for cols in (72, 1537):
        t, norms, d = inputs(1, 9, cols, torch.float32, torch.float32, "layer", "rms", "channel")
        clean = run(t, norms, d, 1.0)
        t["x"] = t["x"].clone()
        t["x"][0, 2, 3], t["x"][0, 5] = float("inf"), float("nan")
        got = run(t, norms, d, 1.0)
        rest = [r for r in range(9) if r not in (2, 5)]
        for k in ("stream", "normed", "d_x", "d_residual"):
            assert torch.equal(got[k][0, rest], clean[k][0, rest]), k
            assert torch.isnan(got[k][0, 5]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_and_misaligned_addresses(dtype):
    t, norms, d = inputs(2, 11, 72, dtype, dtype, "layer", "layer", "sample")
    want = reference(t, norms, d, 1.0)

    def shifted(v, offset):                                  # contiguous, off the 16-byte grid
        buf = torch.empty(v.numel() + offset, dtype=v.dtype, device="cuda")
        buf[offset:] = v.reshape(-1)
        return buf[offset:].view(v.shape)
    for offset in (1, 3):
        check(run({k: shifted(v, offset) for k, v in t.items()}, norms, {k: shifted(v, offset) for k, v in d.items()}, 1.0), want, offset)
    strided = {k: v.transpose(0, -1).contiguous().transpose(0, -1) for k, v in t.items()}
    check(run(strided, norms, {k: v.transpose(0, 1).contiguous().transpose(0, 1) for k, v in d.items()}, 1.0), want, "strided")
    s = dict(t, gate=t["gate"][:, None])                     # (batch, 1, cols)
    got = run(s, norms, d, 1.0)
    got["d_gate"] = got["d_gate"][:, 0]
    check(got, want, "(batch, 1, cols)")
    flat = {k: v.reshape(-1, 72) for k, v in t.items() if k != "gate"}
    w = reference({"x": t["x"], "residual": t["residual"]}, norms, d, 1.0)
    got = run(flat, norms, {k: v.reshape(-1, 72) for k, v in d.items()}, 1.0)
    check({k: v.reshape(w[k][0].shape) for k, v in got.items()}, w, "two dimensions")


def test_no_rows():
    t, norms, d = inputs(0, 4, 72, torch.bfloat16, torch.float32, "layer", "rms", "channel")
    got = run(t, norms, d, 1.0)
    for k in ("d_gate", "d_post_weight", "d_post_bias", "d_pre_weight"):
        assert float(got[k].abs().sum()) == 0.0, k
    assert got["normed"].shape == (0, 4, 72) and got["d_x"].shape == (0, 4, 72)
    t, norms, d = inputs(3, 0, 72, torch.float32, torch.float32, "layer", "rms", "sample")
    got = run(t, norms, d, 1.0)
    assert got["d_gate"].shape == (3, 72) and float(got["d_gate"].abs().sum()) == 0.0


def test_gradient_against_differences():
    """L = <stream, ds> + <normed, dn> along random directions, as the gated block's test takes it"""
    t, norms, d = inputs(2, 9, 40, torch.float32, torch.float32, "layer", "rms", "sample")
    got = run(t, norms, d, 0.8)
    eps = 2.0 ** -7
    for name in t:
        v = torch.randn(t[name].shape, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
        v /= v.norm()

        def moved(e, moved_name=name, direction=v):
            return dict(t, **{moved_name: t[moved_name].double() + e * direction.double()})

        def loss64(e):
            r = reference(moved(e), norms, d, 0.8)
            return sum(float((r[k][0] * d[k].double()).sum()) for k in d)

        def loss(e):
            s = {k: p.float() for k, p in moved(e).items()}
            out, r = run(s, norms, d, 0.8, train=False), reference(s, norms, d, 0.8)
            return (sum(float((out[k].double() * d[k].double()).sum()) for k in d),
                    sum(float(((r[k][1] + 2.0 ** -24 * r[k][0].abs()) * d[k].double().abs()).sum()) for k in d))
        full, half = ((loss64(e) - loss64(-e)) / (2 * e) for e in (eps, eps / 2))
        (up, e1), (down, e2) = loss(eps), loss(-eps)
        slope = float((got["d_" + name].double() * v.double()).sum())
        rounded = 2.0 ** -24 * float((got["d_" + name].double().abs() * (t[name].double().abs() + eps)).sum())
        assert abs(slope - (up - down) / (2 * eps)) <= 2 * abs(full - half) + (e1 + e2 + 2 * rounded) / (2 * eps) + 1e-5 * abs(slope), name


def test_reproducible_on_streams_and_replayed():
    sets = [inputs(4, 300, 600, torch.bfloat16, torch.float32, "rms", "layer", "sample", seed=s) for s in range(3)]
    norms = sets[0][1]
    first = run(sets[0][0], norms, sets[0][2], 0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(sets[0][0], norms, sets[0][2], 0.9)
    here = run(sets[0][0], norms, sets[0][2], 0.9)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for k in first:
        assert torch.equal(first[k], other[k]) and torch.equal(first[k], here[k]), k
    t = {k: v.clone() for k, v in sets[0][0].items()}
    d = {k: v.clone() for k, v in sets[0][2].items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(t, norms, d, 0.9)
    for turn in range(4):
        new_t, _, new_d = sets[turn % 3]
        with torch.no_grad():
            for k in t:
                t[k].copy_(new_t[k])
            for k in d:
                d[k].copy_(new_d[k])
        graph.replay()
        want = run(new_t, norms, new_d, 0.9)
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(captured[k], want[k]), (turn, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [(1, 1), (2, 300)])
def test_a_stack_of_gated_blocks(rows, dtype):
    """Two sandwich blocks as a model runs them -- the stream in 32 bits, each block's normed input from the previous one's
    kernel -- forward and gradients, against the same modules in 64 bits.  In units of the norm: seven roundings to the
    tensors' type lie on the longest path of the forward pass (the normed inputs, h and y of two blocks and the last norm),
    twice that of a gradient; norms and products hand on relative errors at about one, so 3 x the square root of their number
    x u x the four paths that meet bounds them."""
    from butd_detr_amd import attention_blocks as ab
    from butd_detr_amd.gated_ffn import GatedFeedForward
    torch.manual_seed(4)
    cols, hidden = 288, 512
    ffns = [GatedFeedForward(cols, hidden, a).cuda().to(dtype) for a in ("silu", "gelu")]
    norms = [norm_of(k, cols, torch.float32) for k in ("rms", "layer", "rms", "rms", "layer")]
    gate = torch.rand(rows[0], cols, device="cuda").to(dtype)
    x = torch.randn(*rows, cols, device="cuda")
    probe = torch.randn(*rows, cols, device="cuda")

    def stack(x, gate, ffns, norms, first):
        stream, normed = ab.gated_ffn_block(ffns[0], x, normed=first, post_norm=norms[1], gate=gate, next_norm=norms[2])
        return ab.gated_ffn_block(ffns[1], stream, normed=normed, post_norm=norms[3], gate=gate, residual_scale=0.7, next_norm=norms[4])

    prev = ab.get_backend()
    try:
        grads, outs = [], []
        for backend in ("hip", "torch"):
            ab.set_backend(backend)
            if backend == "torch":                           # the same values in 64 bits
                import copy
                f = [copy.deepcopy(m).double() for m in ffns]
                n = [copy.deepcopy(m).double() for m in norms]
                xs, gs, p = x.double(), gate.double(), probe.double()
            else:
                f, n, xs, gs, p = ffns, norms, x, gate, probe
            xs, gs = xs.detach().requires_grad_(True), gs.detach().requires_grad_(True)
            first = ab.residual_norm(xs, pre_norm=n[0])[1]
            first = first.to(dtype) if backend == "hip" else first
            stream, normed = stack(xs, gs, f, n, first)
            leaves = [xs, gs] + [q for m in f for q in m.parameters()]
            grads.append(torch.autograd.grad([stream, normed], leaves, [p.to(stream.dtype), p.to(normed.dtype)]))
            outs.append([stream.detach(), normed.detach()])
    finally:
        ab.set_backend(prev)
    assert outs[0][0].dtype == torch.float32 and outs[0][1].dtype == dtype
    u = max(torch.finfo(dtype).eps / 2, 2.0 ** -20)          # (32 bits: the sums' own errors, 2^-20 of the norm)
    for got, want, count in list(zip(*outs, [7, 7])) + [(g, w, 14) for g, w in zip(*grads)]:
        assert float((got.double() - want).norm() / want.norm()) <= 4 * 3 * count ** 0.5 * u


@pytest.mark.parametrize("batch, length", [(5, 1), (300, 2), (2, 700), (3, 1001)])
@pytest.mark.parametrize("gate", ["channel", "sample", "element"])
@pytest.mark.parametrize("cols", [9, 25, 601, 4097])
def test_row_shares_of_odd_widths(cols, gate, batch, length):
    """the last unit of a row overlaps its neighbour's"""
    for dtype, stream in ((torch.float32, torch.float32), (torch.float16, torch.float16)):
        t, norms, d = inputs(batch, length, cols, dtype, stream, "layer", "layer", gate)
        check(run(t, norms, d, 1.25), reference(t, norms, d, 1.25), (cols, gate, batch, length, dtype))


def _rows(t, d, a, b):
    cut = lambda m: {k: (v[:, a:b].contiguous() if v.dim() == 3 else v) for k, v in m.items()}     # noqa: E731
    return cut(t), cut(d)


@pytest.mark.parametrize("rows, cols", [((1 << 23) + 5, 8), ((1 << 23) + 5, 7), (300_000, 8192)])
def test_many_rows_and_offsets_beyond_32_bits(rows, cols):
    """Rows do not depend on each other: the last and the first ones equal a call with these alone, bit for bit.  (The forward
    pass launches 2^23 rows of up to 512 elements at a time.)"""
    t, norms, d = inputs(1, rows, cols, torch.bfloat16, torch.bfloat16, "rms", "layer", "channel")
    got = run(t, norms, d, 1.0)
    for a, b in ((0, 70), (rows - 70, rows)):
        alone = run(*(lambda p: (p[0], norms, p[1]))(_rows(t, d, a, b)), 1.0)
        for k in ("stream", "normed", "d_x", "d_residual"):
            assert torch.equal(got[k][:, a:b], alone[k]), (k, a)


def test_many_samples():
    """more sums of samples than workgroups of the kernel that rounds them"""
    t, norms, d = inputs(70_000, 2, 24, torch.bfloat16, torch.float32, "layer", "rms", "sample")
    check(run(t, norms, d, 1.0), reference(t, norms, d, 1.0), "samples")


def test_one_tensor_in_two_places():
    """x as its own residual: the gradients of both places add up"""
    from butd_detr_amd.residual_norm import residual_norm
    t, norms, d = inputs(2, 9, 100, torch.float32, torch.float32, "rms", "layer", None)
    t["residual"] = t["x"]
    want = reference(t, norms, d, 0.5)
    x = t["x"].clone().requires_grad_(True)
    out = residual_norm(x, x, post_norm=norms["post"], residual_scale=0.5, pre_norm=norms["pre"])
    (g,) = torch.autograd.grad(out, [x], [d["stream"], d["normed"]])
    (vx, ex), (vr, er) = want["d_x"], want["d_residual"]
    check({"d_x": g}, {"d_x": (vx + vr, ex + er + 2.0 ** -24 * (vx.abs() + vr.abs()))}, "both")


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fw
    t, norms, d = inputs(1, 3, 8, torch.float32, torch.float32, "rms", None, None)
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        from butd_detr_amd.residual_norm import residual_norm
        residual_norm(fw.make_dual(t["x"], t["x"].clone()), post_norm=norms["post"])


def test_capture_beside_a_living_eager_graph_is_refused():
    from butd_detr_amd.residual_norm import residual_norm
    t, norms, d = inputs(2, 9, 100, torch.float32, torch.float32, "rms", "layer", None)
    x = t["x"].requires_grad_(True)
    alive = residual_norm(x, post_norm=norms["post"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="eager graph"):
            residual_norm(x, post_norm=norms["post"])
    del alive


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("deviation", [1.0, 0.03, 2.0 ** -11])
def test_default_epsilon_against_the_module(dtype, deviation):
    """nn.RMSNorm(eps=None): the module itself on the same tensor, before and after the block.  Both are off by their own
    rounding and 32-bit statistics; a row of zeros is zero."""
    from butd_detr_amd.residual_norm import residual_norm
    g = torch.Generator(device="cuda").manual_seed(11)
    m = nn.RMSNorm(288, device="cuda", dtype=dtype)
    with torch.no_grad():
        m.weight.copy_(1 + 0.2 * torch.randn(288, device="cuda", generator=g))
    x = (deviation * torch.randn(9, 288, device="cuda", generator=g)).to(dtype)
    x[4] = 0
    u = torch.finfo(dtype).eps / 2 + E
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    with torch.no_grad():
        want = m(x).double()
        # the module may round twice: the normalised value, then its product with the weight
        bound = want.abs() * (3 * u + u * u) + 3 * tiny
        for got in (residual_norm(x, pre_norm=m)[1], residual_norm(x, post_norm=m)[0]):
            assert float(((got.double() - want).abs() - bound).max()) <= 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_layer_norm_of_a_constant_row_is_zero(dtype):
    from butd_detr_amd.residual_norm import residual_norm
    x = torch.full((2, 40), 3.0, device="cuda", dtype=dtype)
    assert float(residual_norm(x, pre_norm=nn.LayerNorm(40, device="cuda", dtype=dtype))[1].abs().max()) == 0.0


class _Rounded(torch.autograd.Function):
    """rounds to ``dtype`` what goes forward and / or what comes back, values held in 64 bits; ``noise``: each value is moved by
    that much of the tensor's root mean square (normally distributed) before"""

    @staticmethod
    def _round(v, dtype, noise):
        if noise:
            v = v + noise * v.square().mean().sqrt() * torch.randn(v.shape, device=v.device, dtype=v.dtype)
        return v.to(dtype).double()

    @staticmethod
    def forward(ctx, v, dtype, forth, back, noise):
        ctx.dtype, ctx.back, ctx.noise = dtype, back, noise
        return _Rounded._round(v, dtype, noise) if forth else v.clone()

    @staticmethod
    def backward(ctx, g):
        return (_Rounded._round(g, ctx.dtype, ctx.noise) if ctx.back else g), None, None, None, None


def _unit(m, v):
    if m["bias"] is not None:
        v = v - v.mean(-1, keepdim=True)
    v = v * ((v * v).mean(-1, keepdim=True) + m["eps"]).rsqrt() * m["weight"]
    return v if m["bias"] is None else v + m["bias"]


def _emulated_stack(leaves, norms, dtype, d_out, noise=0.0):
    """Two sandwich blocks in 64 bits, rounded where the kernels round: normed, h and y forward; the gradients of h's two factors,
    of the FFN's input and output and of each use of the gate backward; every output.  -> outputs and gradients"""
    both, forth, back = (lambda v, f=f, b=b: _Rounded.apply(v, dtype, f, b, noise) for f, b in ((True, True), (True, False), (False, True)))
    leaves = [t.detach().double().requires_grad_(True) for t in leaves]
    x, gate, weights = leaves[0], leaves[1], leaves[2:]
    stream, normed = x, both(_unit(norms[0], x))
    for i, scale in enumerate((1.0, 0.7)):
        w_gate, w_up, w_down = weights[3 * i:3 * i + 3]
        a, b = back(normed @ w_gate.t()), back(normed @ w_up.t())
        v = a * torch.sigmoid(a) if i == 0 else 0.5 * a * torch.erfc(-a * 0.5 ** 0.5)
        y = both(forth(v * b) @ w_down.t())
        stream = scale * stream + back(gate)[:, None] * _unit(norms[2 * i + 1], y)
        normed = both(_unit(norms[2 * i + 2], stream))
    out = [stream, normed]
    out += torch.autograd.grad(out, leaves, [p.double() for p in d_out])
    wide = lambda i: i in (0, 2)                             # (the stream and x are 32 bits)       # noqa: E731
    return [t.detach() if wide(i) else _Rounded._round(t.detach(), dtype, noise) for i, t in enumerate(out)]


def stack_inputs(rows, dtype, device="cuda"):
    from butd_detr_amd.gated_ffn import GatedFeedForward
    torch.manual_seed(6)
    cols, hidden = 288, 512
    ffns = [GatedFeedForward(cols, hidden, a).to(device, dtype) for a in ("silu", "gelu")]
    norms = [norm_of(k, cols, torch.float32).to(device) for k in ("rms", "layer", "rms", "rms", "layer")]
    gate = torch.rand(rows[0], cols).to(device, dtype)
    x, p_stream, p_normed = (torch.randn(*rows, cols).to(device) for _ in range(3))
    leaves = [x.requires_grad_(True), gate.requires_grad_(True)] + [q for f in ffns for q in f.parameters()]
    n64 = [dict(weight=m.weight.detach().double(), bias=None if getattr(m, "bias", None) is None else m.bias.detach().double(), eps=m.eps)
           for m in norms]
    return ffns, norms, leaves, [p_stream, p_normed.to(dtype)], n64


def far(got, want):
    return [float((g.double() - w.double()).norm() / w.double().norm()) for g, w in zip(got, want)]


def stack_limits(leaves, n64, dtype, d_out):
    """How far an emulation goes whose every value is moved by a 32-bit computation's error before it is rounded.  A sum of n
    products in 32 bits rounds n times, each time a sum that has grown to sqrt(k) of its terms' size by 2^-24 of it at most, 0.4
    of that in the root mean square: 0.4 2^-24 sqrt(1 + 2 + ... + n) in all, 0.28 sqrt(n) 2^-24 of the result -- 2^-21.2 for the
    up to 600 products here, taken as 2^-21.  Moved values round the other way here and there, and that goes on through the
    later blocks: the distance of the two emulations, taken twice for the chance in it, is what the kernels may be off by; 2^-19
    for what is not rounded."""
    want = _emulated_stack(leaves, n64, dtype, d_out)
    return want, [2 * v + 2.0 ** -19 for v in far(_emulated_stack(leaves, n64, dtype, d_out, noise=2.0 ** -21), want)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [(1, 1), (2, 9), (2, 300)])
def test_a_stack_of_gated_blocks_rounds_where_the_kernels_do(rows, dtype):
    """The stack of test_a_stack_of_gated_blocks, begun by ``pre_norm``, against 64 bits with the same roundings."""
    from butd_detr_amd import attention_blocks as ab
    ffns, norms, leaves, d_out, n64 = stack_inputs(rows, dtype)
    prev = ab.get_backend()
    try:
        ab.set_backend("hip")
        stream, normed = ab.gated_ffn_block(ffns[0], leaves[0], pre_norm=norms[0], post_norm=norms[1], gate=leaves[1], next_norm=norms[2])
        assert normed.dtype == dtype
        out = ab.gated_ffn_block(ffns[1], stream, normed=normed, post_norm=norms[3], gate=leaves[1], residual_scale=0.7,
                                 next_norm=norms[4])
        got = [t.detach() for t in out + torch.autograd.grad(out, leaves, d_out)]
    finally:
        ab.set_backend(prev)
    want, limits = stack_limits(leaves, n64, dtype, d_out)
    for i, (g, off, limit) in enumerate(zip(got, far(got, want), limits)):
        assert g.dtype == (torch.float32 if i in (0, 2) else dtype) and off <= limit, (rows, dtype, i, off, limit)


def test_vmap_is_refused():
    from butd_detr_amd.residual_norm import residual_norm
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: residual_norm(v, pre_norm=nn.RMSNorm(8, device="cuda"))[1])(torch.randn(2, 3, 8, device="cuda"))
