"""-m gpu: the gated feed-forward block (include/butd_gated_ffn.h) against its formulas in 64 bits.

Tolerances are elementwise bounds carried through the formulas, not observed errors.  With u = half a step of the tensors'
type (``eps / 2``), every value that is rounded to that type (h, da, db, the outputs) contributes u of itself; a sum of n
products accumulated in 32 bits at most (n + 2) 2^-23 of the sum of their magnitudes; the activation and its slope, from
hardware exponentials and reciprocals (each within 2^-22 of the value) on arguments whose own rounding enters through the
exponential's slope, 2^-20 (1 + |a|).  Errors of a and b go through the slopes (|act''| <= 1.2 for all five)."""
import gc
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu", "gelu_tanh", "relu", "sigmoid"]
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
E32 = 2.0 ** -23


def inputs(rows, width, hidden, dtype, bias=True, seed=0):
    g = torch.Generator(device="cuda").manual_seed(1000 * seed + rows + 31 * width + 17 * hidden)
    n = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype)      # noqa: E731
    t = dict(x=n(rows, width), w_gate=n(hidden, width, scale=width ** -0.5), w_up=n(hidden, width, scale=width ** -0.5),
             w_down=n(width, hidden, scale=hidden ** -0.5))
    if bias:
        t.update(b_gate=n(hidden, scale=0.3), b_up=n(hidden, scale=0.3), b_down=n(width, scale=0.3))
    return t, n(rows, width, scale=0.3)


def act64(a, kind):
    if kind == "relu":
        return a.clamp_min(0), (a > 0).double()
    if kind in ("silu", "sigmoid"):
        s = torch.sigmoid(a)
        return (s, s * (1 - s)) if kind == "sigmoid" else (a * s, s * (1 + a * (1 - s)))
    if kind == "gelu":
        cdf = 0.5 * torch.erfc(-a * 0.5 ** 0.5)
        return a * cdf, cdf + a * torch.exp(-a * a / 2) * (2 * torch.pi) ** -0.5
    k = (2 / torch.pi) ** 0.5
    s = torch.sigmoid(2 * k * (a + 0.044715 * a ** 3))
    return a * s, s + a * s * (1 - s) * 2 * k * (1 + 3 * 0.044715 * a * a)


def reference(t, dy, kind):
    """{output: (value, bound)} in 64 bits"""
    u = torch.finfo(t["x"].dtype).eps / 2
    d = {k: v.detach().double() for k, v in t.items()}
    dy = dy.double()
    M, E = d["x"].shape
    F = d["w_gate"].shape[0]
    zero = torch.zeros((), device="cuda", dtype=torch.float64)
    bg, bu, bd = (d.get(k, zero) for k in ("b_gate", "b_up", "b_down"))
    mm = lambda p, q: p @ q                                                                        # noqa: E731
    a, b = mm(d["x"], d["w_gate"].t()) + bg, mm(d["x"], d["w_up"].t()) + bu
    ea = (E + 2) * E32 * (mm(d["x"].abs(), d["w_gate"].abs().t()) + bg.abs())
    eb = (E + 2) * E32 * (mm(d["x"].abs(), d["w_up"].abs().t()) + bu.abs())
    v, s = act64(a, kind)
    near = 2.0 ** -20 * (1 + a.abs())
    ev = s.abs() * ea + 0.6 * ea * ea + near * (1 + a.abs())
    es = 1.2 * ea + near
    if kind == "relu":                                       # (a slope that flips where a is within its own error of 0)
        ev, es = ea, (a.abs() <= ea).double()
    h = v * b
    eh = ev * b.abs() + v.abs() * eb + ev * eb + u * h.abs() + 1e-7 * u
    y = mm(h, d["w_down"].t()) + bd
    out = {"y": (y, mm(eh, d["w_down"].abs().t()) + (F + 2) * E32 * (mm(h.abs(), d["w_down"].abs().t()) + bd.abs()) + u * y.abs())}
    dh = mm(dy, d["w_down"])
    edh = (E + 2) * E32 * mm(dy.abs(), d["w_down"].abs())
    da, db = dh * b * s, dh * v
    # (16-bit: fp16's smallest steps are absolute -- 2^-25 each)
    tiny = 2.0 ** -25 if t["x"].dtype == torch.float16 else 0.0
    eda = edh * (b * s).abs() + dh.abs() * (s.abs() * eb + b.abs() * es + eb * es) + edh * (b.abs() * es + s.abs() * eb) + u * da.abs() + tiny
    edb = edh * v.abs() + dh.abs() * ev + edh * ev + u * db.abs() + tiny
    dx = mm(da, d["w_gate"]) + mm(db, d["w_up"])
    out["d_x"] = (dx, mm(eda, d["w_gate"].abs()) + mm(edb, d["w_up"].abs()) + u * dx.abs()
                  + (2 * F + 2) * E32 * (mm(da.abs(), d["w_gate"].abs()) + mm(db.abs(), d["w_up"].abs())))
    for k, p, ep in (("d_w_gate", da, eda), ("d_w_up", db, edb)):
        w = mm(p.t(), d["x"])
        out[k] = (w, mm(ep.t(), d["x"].abs()) + (M + 2) * E32 * mm(p.abs().t(), d["x"].abs()) + u * w.abs())
    w = mm(dy.t(), h)
    out["d_w_down"] = (w, mm(dy.abs().t(), eh) + (M + 2) * E32 * mm(dy.abs().t(), h.abs()) + u * w.abs())
    if "b_gate" in d:
        for k, p, ep in (("d_b_gate", da, eda), ("d_b_up", db, edb), ("d_b_down", dy, torch.zeros_like(dy))):
            out[k] = (p.sum(0), ep.sum(0) + (M + 2) * E32 * p.abs().sum(0) + u * p.sum(0).abs())
    return {k: (val, bnd + tiny) for k, (val, bnd) in out.items()}


def run(t, dy, kind, train=True):
    from butd_detr_amd.gated_ffn import gated_ffn
    leaves = {k: v.detach().requires_grad_(train) for k, v in t.items()}
    y = gated_ffn(leaves["x"], leaves["w_gate"], leaves["w_up"], leaves["w_down"], leaves.get("b_gate"), leaves.get("b_up"),
                  leaves.get("b_down"), activation=kind)
    if not train:
        return {"y": y}
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    return {"y": y.detach(), **{"d_" + k: g for k, g in zip(leaves, grads)}}


def check(got, want, what):
    for k, v in got.items():
        value, bound = want[k]
        assert v.shape == value.shape, (what, k)
        off = (v.double() - value).abs() - bound
        assert not torch.isnan(v).any() and float(off.max()) <= 0, (what, k, float(off.max()), float(bound.max()))


@pytest.fixture
def tile():
    """set(tile, split): every product on that tile"""
    from butd_detr_amd import _hiplib
    lib = _hiplib.load()
    yield lambda t, s: _hiplib.check(lib.butd_gated_ffn_set_tile(t, s), "butd_gated_ffn_set_tile")
    lib.butd_gated_ffn_set_tile(0, 0)


# rows: up to 16 / 32 / 64 take the streaming kernels, more the tiles; widths that are multiples of 16 bytes and not; the
# layers' own 288 x 256 and 288 x 2048
SIZES = [(1, 1, 1), (1, 8, 8), (2, 24, 40), (3, 5, 7), (16, 64, 96), (17, 40, 24), (33, 129, 65), (64, 288, 256), (65, 16, 8),
         (65, 1, 3), (80, 77, 130), (130, 72, 520), (257, 136, 264), (300, 64, 1027), (512, 288, 256), (515, 288, 2048)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
def test_against_the_formulas(size, dtype):
    kind = ACTS[sum(size) % 5]
    for bias in (False, True):
        t, dy = inputs(*size, dtype, bias)
        want = reference(t, dy, kind)
        check(run(t, dy, kind), want, (size, dtype, kind, bias))
        check(run(t, dy, kind, train=False), want, (size, dtype, kind, bias, "inference"))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ACTS)
def test_activations(kind, dtype):
    for rows in (9, 150):
        t, dy = inputs(rows, 48, 56, dtype)
        t["b_gate"] = (torch.linspace(-12, 12, 56, device="cuda")).to(dtype)      # the whole range of the activation
        check(run(t, dy, kind), reference(t, dy, kind), (rows, dtype, kind))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size, split", list(itertools.product((64, 128, 256), (1, 3))))
def test_every_tile_at_ragged_edges(tile, size, split, dtype):
    tile(size, split)
    for shape in [(200, 8, 16), (259, 264, 520), (300, 200, 77), (515, 100, 260)]:
        t, dy = inputs(*shape, dtype)
        check(run(t, dy, "silu"), reference(t, dy, "silu"), (shape, dtype, size, split))


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_sizes_by_the_rule(dtype):
    """several tiles in every direction, more tiles than CUs, a split contraction"""
    for shape in [(1500, 520, 3000), (4100, 288, 256), (100, 2056, 1000)]:
        t, dy = inputs(*shape, dtype)
        check(run(t, dy, "gelu"), reference(t, dy, "gelu"), (shape, dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 5, 70, 300])
def test_strided_and_misaligned_operands(rows, dtype):
    width, hidden = 72, 104
    t, dy = inputs(rows, width, hidden, dtype)
    want = reference(t, dy, "silu")

    def shifted(v, pad, offset):
        buf = torch.full((v.shape[0], v.shape[1] + pad), float("nan"), dtype=v.dtype, device="cuda")      # never read
        buf[:, offset:offset + v.shape[1]] = v
        return buf[:, offset:offset + v.shape[1]]
    for pad, offset in ((8, 0), (8, 8), (16, 3), (5, 1)):
        s = dict(t)
        s["x"], s["w_gate"] = shifted(t["x"], pad, offset), shifted(t["w_gate"], pad, offset)
        s["w_down"] = shifted(t["w_down"], pad, offset)
        check(run(s, shifted(dy, pad, offset), "silu"), want, (rows, dtype, pad, offset))
    s = dict(t)
    s["w_up"] = t["w_up"].t().contiguous().t()                # column-major: no contiguous last dimension
    s["x"] = t["x"].t().contiguous().t()
    check(run(s, dy.t().contiguous().t(), "silu"), want, (rows, dtype, "transposed"))
    x = t["x"].detach().requires_grad_(True)
    (g,) = torch.autograd.grad(_apply(dict(t, x=x), "silu").sum(), [x])      # an expanded gradient
    check({"d_x": g}, reference(t, torch.ones_like(dy), "silu"), (rows, dtype, "expanded"))


def _apply(t, kind):
    from butd_detr_amd.gated_ffn import gated_ffn
    return gated_ffn(t["x"], t["w_gate"], t["w_up"], t["w_down"], t.get("b_gate"), t.get("b_up"), t.get("b_down"), activation=kind)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_rows_and_more_dimensions(dtype):
    t, dy = inputs(0, 24, 40, dtype)
    got = run(t, dy, "silu")
    assert got["y"].shape == (0, 24) and got["d_x"].shape == (0, 24)
    for k in ("d_w_gate", "d_w_up", "d_w_down", "d_b_gate", "d_b_up", "d_b_down"):
        assert float(got[k].abs().sum()) == 0.0, k
    t, dy = inputs(6 * 15, 24, 40, dtype)
    want = reference(t, dy, "silu")
    t["x"], dy = t["x"].view(2, 3, 15, 24), dy.view(2, 3, 15, 24)
    got = run(t, dy, "silu")
    assert got["y"].shape == t["x"].shape == got["d_x"].shape
    check({k: v.reshape(want[k][0].shape) for k, v in got.items()}, want, "4-d")


def test_only_the_gradients_that_are_wanted():
    t, dy = inputs(100, 40, 56, torch.bfloat16)
    want = reference(t, dy, "silu")
    for names in (["x"], ["w_gate"], ["w_up"], ["w_down"], ["b_gate"], ["b_up"], ["b_down"], ["x", "b_down"], ["w_gate", "w_down"]):
        leaves = {k: v.detach().requires_grad_(k in names) for k, v in t.items()}
        grads = torch.autograd.grad(_apply(leaves, "silu"), [leaves[n] for n in names], dy)
        check({"d_" + n: g for n, g in zip(names, grads)}, want, names)


def test_infinities_and_nan_stay_in_their_rows():
    for rows in (7, 200):
        for dtype in DTYPES:
            t, dy = inputs(rows, 40, 56, dtype)
            clean = run(t, dy, "silu", train=False)["y"]
            t["x"] = t["x"].clone()
            t["x"][2, 3] = float("inf")
            t["x"][5] = float("nan")
            y = run(t, dy, "silu", train=False)["y"]
            rest = [r for r in range(rows) if r not in (2, 5)]
            assert torch.equal(y[rest], clean[rest]) and torch.isnan(y[5]).all() and not torch.isfinite(y[2]).any()


def test_large_preactivations_do_not_overflow():
    """|a| up to 400 in 32 bits: e^-a is infinite in places, nothing else is"""
    for kind in ACTS:
        t, dy = inputs(70, 16, 24, torch.float32)
        t["w_gate"] = t["w_gate"] * 100
        check(run(t, dy, kind), reference(t, dy, kind), kind)


@pytest.mark.parametrize("rows", [3, 90])
def test_gradient_against_differences(rows):
    """d/de L(p + e v) at e = 0 for random directions v, L = <y, dy>: the kernels' central difference and the gradient.
    The difference's truncation is taken from the formulas in 64 bits at the same step (twice what halving it changes);
    its rounding from the bound of y, over the step."""
    t, dy = inputs(rows, 24, 40, torch.float32)
    kind, eps = "gelu", 2.0 ** -6
    got = run(t, dy, kind)
    for name in t:
        v = torch.randn(t[name].shape, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
        v /= v.norm()

        def loss64(e, moved=name, direction=v):
            s = {k: p.double() for k, p in t.items()}
            s[moved] = s[moved] + e * direction.double()
            a, b = s["x"] @ s["w_gate"].t() + s["b_gate"], s["x"] @ s["w_up"].t() + s["b_up"]
            return float((((act64(a, kind)[0] * b) @ s["w_down"].t() + s["b_down"]) * dy.double()).sum())

        def loss(e, moved=name, direction=v):
            s = dict(t)
            s[moved] = s[moved] + e * direction
            y = run(s, dy, kind, train=False)["y"]
            return float((y.double() * dy.double()).sum()), float((reference(s, dy, kind)["y"][1] * dy.double().abs()).sum())
        full, half = ((loss64(e) - loss64(-e)) / (2 * e) for e in (eps, eps / 2))
        (up, e1), (down, e2) = loss(eps), loss(-eps)
        slope = float((got["d_" + name].double() * v.double()).sum())
        # (p + e v is rounded to 32 bits: |p| 2^-24 in each element, which the slope turns into a loss)
        moved = 2.0 ** -24 * float((got["d_" + name].double().abs() * (t[name].double().abs() + eps)).sum())
        assert abs(slope - (up - down) / (2 * eps)) <= 2 * abs(full - half) + (e1 + e2 + 2 * moved) / (2 * eps) + 1e-5 * abs(slope), name


def test_reproducible_streams_and_concurrent_calls():
    t, dy = inputs(700, 288, 256, torch.bfloat16)
    first = run(t, dy, "silu")
    sides = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for side in sides * 2:                                    # two streams, calls in flight on both
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            results.append(run(t, dy, "silu"))
    for side in sides:
        torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for got in results:
        for k in first:
            assert torch.equal(got[k], first[k]), k


@pytest.mark.parametrize("rows", [4, 700])
def test_captured_and_replayed(rows):
    """Two graphs (forward; forward + backward) of different inputs, replayed in turn with eager work between them."""
    sets = [inputs(rows, 288, 256, torch.bfloat16, seed=s) for s in range(3)]
    static = [{k: v.clone() for k, v in sets[0][0].items()} for _ in range(2)]
    dys = sets[0][1].clone()
    leaves = {k: v.requires_grad_(True) for k, v in static[1].items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        _apply(static[0], "silu")
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g0, g1 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g0), torch.no_grad():
        y0 = _apply(static[0], "silu")
    with torch.cuda.graph(g1):
        y1 = _apply(leaves, "silu")
        grads = torch.autograd.grad(y1, list(leaves.values()), dys)
    for turn in range(4):
        t, dy = sets[turn % 3]
        with torch.no_grad():
            for k in t:
                static[0][k].copy_(t[k])
                leaves[k].copy_(t[k])
            dys.copy_(dy)
        g0.replay()
        g1.replay()
        want = run(t, dy, "silu")
        infer = run(t, dy, "silu", train=False)["y"]
        torch.cuda.synchronize()
        assert torch.equal(y0, infer) and torch.equal(y1.detach(), want["y"])
        for k, g in zip(leaves, grads):
            assert torch.equal(g, want["d_" + k]), k


def test_module_and_torch_backend_agree():
    from butd_detr_amd import attention_blocks as ab
    from butd_detr_amd.gated_ffn import GatedFeedForward
    torch.manual_seed(0)
    ffn = GatedFeedForward(288, 256, "gelu_tanh", bias=True).cuda()
    x = torch.randn(2, 300, 288, device="cuda")
    prev, outs = ab.get_backend(), []
    try:
        for backend in ("torch", "hip"):
            ab.set_backend(backend)
            outs.append(ffn(x))
    finally:
        ab.set_backend(prev)
    want = reference({"x": x.reshape(-1, 288), "w_gate": ffn.gate.weight, "w_up": ffn.up.weight, "w_down": ffn.down.weight,
                      "b_gate": ffn.gate.bias, "b_up": ffn.up.bias, "b_down": ffn.down.bias}, torch.zeros(600, 288, device="cuda"),
                     "gelu_tanh")["y"]
    for out in outs:
        check({"y": out.detach().reshape(-1, 288)}, {"y": want}, "module")


def test_second_derivatives_are_refused():
    t, dy = inputs(5, 8, 8, torch.float32)
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    (g,) = torch.autograd.grad(_apply(leaves, "silu"), [leaves["x"]], dy.requires_grad_(True), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [leaves["x"]])


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fw
    t, dy = inputs(5, 8, 8, torch.float32)
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        _apply({**t, "x": fw.make_dual(t["x"], torch.ones_like(t["x"]))}, "silu")


def test_capture_beside_a_living_eager_graph_is_refused():
    t, dy = inputs(70, 48, 40, torch.bfloat16)
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    alive = _apply(leaves, "silu")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="eager graph"):
            _apply(leaves, "silu")
    (want,) = torch.autograd.grad(alive, [leaves["x"]], dy)
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (got,) = torch.autograd.grad(_apply(leaves, "silu"), [leaves["x"]], dy)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("rows", [9, 200])
def test_one_tensor_in_several_places_and_changed_in_place(rows):
    """W_gate is W_up and x feeds its own layer's weights: gradients of the places add up; a weight that changed between the
    passes is refused."""
    from butd_detr_amd.gated_ffn import gated_ffn
    t, dy = inputs(rows, 40, 40, torch.float32, bias=False)
    want = reference({**t, "w_up": t["w_gate"]}, dy, "silu")
    w = t["w_gate"].requires_grad_(True)
    x, down = t["x"].requires_grad_(True), t["w_down"].requires_grad_(True)
    y = gated_ffn(x, w, w, down)
    g = torch.autograd.grad(y, [x, w, down], dy, retain_graph=True)
    (vg, eg), (vu, eu) = want["d_w_gate"], want["d_w_up"]
    both = (vg + vu, eg + eu + E32 * (vg + vu).abs())
    check({"d_x": g[0], "d_w_gate": g[1], "d_w_down": g[2]}, {**want, "d_w_gate": both}, "shared")
    again = torch.autograd.grad(y, [x, w, down], dy, retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(g, again))
    with torch.no_grad():
        down.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, [x], dy)


def test_calls_from_several_threads():
    import threading
    jobs = [(inputs(rows, 96, 72, torch.bfloat16, seed=rows), kind) for rows, kind in ((3, "silu"), (130, "gelu"), (700, "relu"), (65, "sigmoid"))]
    want = [run(t, dy, kind) for (t, dy), kind in jobs]
    torch.cuda.synchronize()                                 # (their inputs come from this thread's stream)
    got = [[] for _ in jobs]

    def work(i):
        (t, dy), kind = jobs[i]
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                got[i].append(run(t, dy, kind))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    for w, runs in zip(want, got):
        assert len(runs) == 5
        for g in runs:
            for k in w:
                assert torch.equal(g[k], w[k]), k


def test_offsets_beyond_32_bits():
    """More than 2^31 elements between the first and the last row of h, a and b.  dy is zero but for the last 64 rows, so the
    gradients are those of these rows alone."""
    rows, width, hidden, last = 2_100_000, 16, 1040, 64
    t, dy = inputs(rows, width, hidden, torch.bfloat16)
    dy[:-last] = 0
    tail = {k: (v[-last:] if k == "x" else v) for k, v in t.items()}
    want = reference(tail, dy[-last:], "silu")
    got = run(t, dy, "silu")
    assert not got["d_x"][:-last].any()
    check({k: (v[-last:] if k in ("y", "d_x") else v) for k, v in got.items()}, want, "last rows")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, size", [(5, 64), (100, 64), (100, 128), (300, 256)])
def test_an_infinite_row_stays_infinite(tile, rows, size, dtype):
    """positive weights, one +inf in x, sigmoid: y of that row is +inf.  The hidden width fills no whole vector: what lies
    behind its last column must not turn the sum into NaN."""
    if rows > 16:
        tile(size, 1)
    t, _ = inputs(rows, 24, 37, dtype, bias=False)
    t = {k: v.abs() + 0.125 for k, v in t.items()}
    t["x"][1, 3] = float("inf")
    for train in (False, True):
        y = run(t, torch.zeros_like(t["x"]), "sigmoid", train=train)["y"]
        assert torch.isposinf(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2:]).all()


class _Rounded(torch.autograd.Function):
    """rounds to ``dtype`` what goes forward and / or what comes back, values held in 64 bits"""

    @staticmethod
    def forward(ctx, v, dtype, forth, back):
        ctx.dtype, ctx.back = dtype, back
        return v.to(dtype).double() if forth else v.clone()

    @staticmethod
    def backward(ctx, g):
        return (g.to(ctx.dtype).double() if ctx.back else g), None, None, None


def emulated(t, dy, kind):
    """The block in 64 bits with the roundings of include/butd_gated_ffn.h and no others: h forward, da and db backward --
    operands of the next product -- and every output.  The bias gradients are sums of the unrounded da and db."""
    dtype = t["x"].dtype
    p = {k: v.detach().double().requires_grad_(True) for k, v in t.items()}
    a, b = (_Rounded.apply(p["x"] @ p[w].t(), dtype, False, True) + p[v] for w, v in (("w_gate", "b_gate"), ("w_up", "b_up")))
    if kind == "sigmoid":
        v = torch.sigmoid(a)
    elif kind == "gelu":
        v = 0.5 * a * torch.erfc(-a * 0.5 ** 0.5)
    else:
        v = a * torch.sigmoid(a)
    h = _Rounded.apply(v * b, dtype, True, False)
    y = h @ p["w_down"].t() + p["b_down"]
    grads = torch.autograd.grad(y, list(p.values()), dy.double())
    return {k: v.detach().to(dtype) for k, v in {"y": y, **{"d_" + n: g for n, g in zip(p, grads)}}.items()}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [(5, 256, 512), (40, 136, 264), (700, 288, 256), (1100, 200, 300), (2048, 77, 130)])
def test_the_documented_roundings_and_no_others(size, dtype):
    """Against ``emulated``, relative to an output's norm.  What is left are the 32-bit errors in front of each rounding, 2^-20
    of the value: a value rounds the other way where it lies that close to a border between two of its neighbours 2 u apart,
    a share of 2^-20 / u of all values, and is then off by 2 u.  The root mean square of one such stage is 2 u sqrt(2^-20 / u),
    of the at most three stages on an output's way sqrt(3) times that: u / 18 for bf16, u / 6.5 for fp16 (u = 2^-8, 2^-11).
    One rounding too many or one too few is at least u / sqrt(6) (a mantissa anywhere in [1, 2), an error anywhere in
    [-u, u])."""
    for kind in ("silu", "gelu", "sigmoid"):               # (the smooth ones: no slope jumps within an error of a)
        t, dy = inputs(*size, dtype)
        got, want = run(t, dy, kind), emulated(t, dy, kind)
        u = torch.finfo(dtype).eps / 2
        limit = 2 * u * (3 * 2.0 ** -20 / u) ** 0.5
        for k in want:
            far = float((got[k].double() - want[k].double()).norm() / want[k].double().norm())
            assert far <= limit, (size, kind, k, far / u, limit / u)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [5, 130])
def test_autocast_casts_like_a_linear_layer(rows, kind):
    """float32 parameters, x of either type: the call on cast tensors, gradients in the types the leaves have."""
    from butd_detr_amd import attention_blocks as ab
    from butd_detr_amd.gated_ffn import GatedFeedForward
    t, dy = inputs(rows, 40, 56, torch.float32)
    dy = dy.to(kind)
    want = run({k: v.to(kind) for k, v in t.items()}, dy, "silu")
    for x_type in (torch.float32, kind):
        leaves = {k: v.to(x_type if k == "x" else torch.float32).requires_grad_(True) for k, v in t.items()}
        with torch.autocast("cuda", kind):
            y = _apply(leaves, "silu")
            with torch.no_grad():
                quiet = _apply(leaves, "silu")
        assert y.dtype == kind and torch.equal(y, want["y"]) and torch.equal(quiet, y)
        for (k, v), g in zip(leaves.items(), torch.autograd.grad(y, list(leaves.values()), dy)):
            assert g.dtype == v.dtype and torch.equal(g, want["d_" + k].to(v.dtype)), k
    torch.manual_seed(0)
    ffn, x = GatedFeedForward(40, 56, bias=True).cuda(), t["x"].to(kind)
    prev = ab.get_backend()
    try:
        for backend in ("torch", "hip"):
            ab.set_backend(backend)
            with torch.autocast("cuda", kind):
                assert ffn(x).dtype == kind and ffn(x.float()).dtype == kind
            with torch.autocast("cuda", kind, enabled=False):
                assert ffn(x.float()).dtype == torch.float32
    finally:
        ab.set_backend(prev)
    with torch.autocast("cuda", kind), pytest.raises(RuntimeError, match="not served"):
        _apply({k: v.double() for k, v in t.items()}, "silu")


def test_capture_beside_a_living_eager_graph_is_refused_under_autocast():
    """the leaves are looked at, not their casts"""
    t, _ = inputs(70, 48, 40, torch.float32)
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    with torch.autocast("cuda", torch.bfloat16):
        alive = _apply(leaves, "silu")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            with pytest.raises(RuntimeError, match="eager graph"):
                _apply(leaves, "silu")
    del alive


def test_vmap_is_refused():
    t, _ = inputs(6, 8, 8, torch.float32, bias=False)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda v: _apply({**t, "x": v}, "silu"))(t["x"].view(2, 3, 8))


def test_capture_beside_a_living_eager_graph_is_refused_for_casts_and_views():
    """Operands that the capture casts or views: their leaves' gradients belong to the living graph all the same.  So does what
    an eager graph hands over undetached.  (Only forward passes run here.)"""
    t, dy = inputs(70, 40, 40, torch.float32)
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    views = {"cast": lambda d: {k: v.bfloat16() for k, v in d.items()}, "view": lambda d: {**d, "w_up": d["w_up"].t().t()},
             "sum": lambda d: {**d, "x": (d["x"] + 1) * 2}}
    alive, between = _apply(leaves, "silu"), leaves["x"] * 2
    for view in views.values():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            fresh = {k: v.detach().requires_grad_(True) for k, v in leaves.items()}
            _apply(view(fresh), "silu")                      # (leaves of no other graph)
            with pytest.raises(RuntimeError, match="eager graph"):
                _apply(view({**fresh, "x": leaves["x"], "w_up": leaves["w_up"]}), "silu")
            with pytest.raises(RuntimeError, match="eager graph"):
                _apply({**fresh, "x": between}, "silu")
            _apply({**fresh, "x": between.detach()}, "silu")
    del alive, fresh, between
    gc.collect()                                             # (what the refused calls' tracebacks hold)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = _apply(views["cast"](leaves), "silu")
        (got,) = torch.autograd.grad(y, [leaves["w_up"]], dy.bfloat16())
    want = run({k: v.detach().bfloat16() for k, v in t.items()}, dy.bfloat16(), "silu")
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want["y"]) and torch.equal(got, want["d_w_up"].float())


def test_recomputed_and_offloaded_activations():
    """torch.utils.checkpoint and saved tensors kept on the host: the same gradients, bit for bit"""
    from torch.utils.checkpoint import checkpoint
    t, dy = inputs(130, 40, 56, torch.bfloat16)
    want = run(t, dy, "silu")
    leaves = {k: v.requires_grad_(True) for k, v in t.items()}
    ys = [checkpoint(lambda *a: _apply(dict(zip(leaves, a)), "silu"), *leaves.values(), use_reentrant=False)]
    with torch.autograd.graph.save_on_cpu():
        ys.append(_apply(leaves, "silu"))
    for y in ys:
        for k, g in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)):
            assert torch.equal(g, want["d_" + k]), k
