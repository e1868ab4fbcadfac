"""-m gpu: which products of the set-abstraction streaming kernels (butd_sa_thin_conv, butd_sa_colstats, butd_sa_mask_stats,
butd_sa_pool_bwd_stats, butd_sa_bn_finalize) are fused with their sums -- bit for bit, against 64-bit arithmetic on values
short enough that every product and sum is exact there, so that only the 32-bit roundings written in csrc/sa_ops.hip remain."""
import pytest
import torch

pytestmark = pytest.mark.gpu
CHUNK = 64                                                   # rows of a workgroup below 2^19 rows


def short(*shape, seed, bits=12, scale=2.0 ** -8):
    """multiples of ``scale`` below 2^bits of them: a product has up to 2 bits, a fused sum of a few fits 53"""
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-2 ** bits, 2 ** bits, shape, generator=g).double() * scale)


def f32(v):
    return v.float().double()


def call(name, *args):
    from butd_detr_amd import _hiplib
    raw = [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]
    _hiplib.check(getattr(_hiplib.load(), name)(*raw, torch.cuda.current_stream().cuda_stream), name)
    torch.cuda.synchronize()


def d(v, dtype=torch.float32):
    return v.to("cuda", dtype).contiguous()


def sums_by_phase(rows, threads, first):
    """what a workgroup's threads sum: row phase by phase in 32 bits (``first(sum, row)``), the phases in 64"""
    total = 0
    for sub in range(threads):
        s = torch.zeros(rows.shape[1], dtype=torch.float64)
        for r in rows[sub::threads]:
            s = first(s, r)
        total = total + s
    return total


@pytest.mark.parametrize("C", [64, 128])
def test_thin_conv(C):
    K, P = 6, 40
    x, w = short(P, 8, seed=1, bits=14), short(C, K, seed=2, bits=14, scale=2.0 ** -15)
    x[:, K:] = 0
    z = torch.zeros(P, C, dtype=torch.float64)
    fused = torch.arange(C) % 4 < 2
    for k in range(K):
        p = x[:, k:k + 1] * w[:, k]
        z = f32(torch.where(fused, z + p, z + f32(p)))
    assert not torch.equal(z, f32(f32(x[:, :K] @ w.t())))    # (roundings of the way, not one of the whole)
    out = torch.empty(P, C, device="cuda")
    s, q = torch.zeros(C, device="cuda", dtype=torch.float64), torch.zeros(C, device="cuda", dtype=torch.float64)
    call("butd_sa_thin_conv", P, C, K, d(x), 8, d(w), out, s, q)
    assert torch.equal(out.cpu().double(), z)
    assert torch.equal(s.cpu(), sums_by_phase(z, 1024 // C, lambda a, r: f32(a + r)))


@pytest.mark.parametrize("pool", [0, 16])
def test_column_statistics(pool):
    C, P = 64, 256
    z = short(P, C, seed=3, bits=14)
    fused = torch.arange(C) % 4 < 2
    once, twice = lambda a, r: f32(a + r * r), lambda a, r: f32(a + f32(r * r))              # noqa: E731
    s, q = 0, 0
    for block in z.split(CHUNK):                             # a workgroup's rows; its 16 phases take rows, or whole groups
        groups = block.view(-1, pool or 1, C)
        for sub in range(16):
            a, b, c = (torch.zeros(C, dtype=torch.float64) for _ in range(3))
            for r in groups[sub::16].reshape(-1, C):
                a, b, c = f32(a + r), once(b, r), twice(c, r)
            s, q = s + a, q + torch.where(fused, b, c)
    gs, gq = torch.zeros(C, device="cuda", dtype=torch.float64), torch.zeros(C, device="cuda", dtype=torch.float64)
    groups = P // pool if pool else 1
    mx, mn = torch.empty(groups, C, device="cuda"), torch.empty(groups, C, device="cuda")
    ax, an = (torch.empty(groups, C, device="cuda", dtype=torch.uint8) for _ in range(2))
    call("butd_sa_colstats", P, C, d(z), gs, gq, pool, mx, mn, ax, an)
    assert torch.equal(gs.cpu(), s) and torch.equal(gq.cpu(), q)
    assert not torch.equal(gq.cpu(), (z * z).sum(0))


def test_running_statistics_round_both_products():
    C, momentum = 64, 0.1
    mean0, var0 = short(C, seed=4, bits=20, scale=2.0 ** -18), short(C, seed=5, bits=20, scale=2.0 ** -18).abs() + 1
    count = 1 << 10
    total, squares = short(C, seed=6, bits=20, scale=2.0 ** -6), short(C, seed=7, bits=20, scale=2.0 ** -6).abs() + 2 ** 24
    m = total / count
    v = squares / count - m * m
    unbiased = v * count / (count - 1)
    a, b = f32(torch.tensor(momentum, dtype=torch.float64)), f32(1 - f32(torch.tensor(momentum, dtype=torch.float64)))
    want_mean, want_var = f32(f32(b * mean0) + f32(a * f32(m))), f32(f32(b * var0) + f32(a * f32(unbiased)))
    rm, rv = d(mean0), d(var0)
    one, outs = torch.ones(C, device="cuda"), [torch.empty(C, device="cuda") for _ in range(4)]
    batches = torch.zeros(1, device="cuda", dtype=torch.int64)
    call("butd_sa_bn_finalize", C, count, d(total, torch.float64), d(squares, torch.float64), 1, C, one, one, 1e-5, momentum, 1,
         rm, rv, batches, *outs)
    assert int(batches) == 1
    assert torch.equal(rm.cpu().double(), want_mean) and torch.equal(rv.cpu().double(), want_var)


def test_backward_statistics():
    """sum of dy (z - mean) rstd over the rows whose gate is open: the last product fused over dense rows, rounded over pooled
    ones"""
    C, P = 64, 8
    z, dy = short(P, C, seed=8, bits=12), short(P, C, seed=9, bits=11)
    scale, shift, mean, rstd = (short(C, seed=s, bits=10) for s in (10, 11, 12, 13))
    gate = (scale * z + shift > 0).double()
    p = f32(dy * f32(z - mean))
    want = {"butd_sa_mask_stats": torch.zeros(C, dtype=torch.float64), "butd_sa_pool_bwd_stats": torch.zeros(C, dtype=torch.float64)}
    threads = {"butd_sa_mask_stats": 16, "butd_sa_pool_bwd_stats": 4}
    for name in want:
        for sub in range(threads[name]):
            s = torch.zeros(C, dtype=torch.float64)
            for r in range(sub, P, threads[name]):
                if name == "butd_sa_mask_stats":
                    s = f32(s + gate[r] * p[r] * rstd)
                else:
                    s = torch.where(gate[r] > 0, f32(s + f32(p[r] * rstd)), s)
            want[name] = want[name] + s
    for name in want:
        s1, s2 = torch.zeros(C, device="cuda", dtype=torch.float64), torch.zeros(C, device="cuda", dtype=torch.float64)
        head = (P, C) if name == "butd_sa_mask_stats" else (1, P, C)
        call(name, *head, d(dy), d(z), d(scale), d(shift), d(mean), d(rstd), s1, s2)
        assert torch.equal(s1.cpu(), (dy * gate).sum(0)) and torch.equal(s2.cpu(), want[name]), name
