"""The embedding lookup and its gradient on the GPU against the plain form in 64 bits."""
import numpy as np
import pytest
import torch

import gpu_lib as G
import plain64 as P

pytestmark = pytest.mark.gpu
F16, F32, F64 = torch.float16, torch.float32, torch.float64
TYPES = [F16, F32, F64]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=gen(seed), dtype=F64) * scale).to(dtype)


def guarded(t, shift=0):
    g = G.Guarded(tuple(t.shape), t.dtype, shift)
    g.t.copy_(t)
    return g


def ids_of(kind, m, v, seed=3):
    g = gen(seed)
    if kind == "uniform":
        return torch.randint(0, v, (m,), generator=g)
    if kind == "skewed":  # as one over the rank
        return (torch.exp(torch.rand(m, generator=g, dtype=F64) * np.log(v + 1)) - 1).long().clamp(0, v - 1)
    if kind == "one":
        return torch.full((m,), v // 2)
    if kind == "all different":
        return torch.randperm(v, generator=g)[:m] if m <= v else torch.arange(m) % v
    if kind == "falling":
        return torch.arange(m).flip(0) * v // max(m, 1)
    if kind == "padded":
        t = torch.randint(0, v, (m,), generator=g)
        t[torch.rand(m, generator=g) < 0.4] = -1
        return t
    if kind == "outside":
        t = torch.randint(-2, v + 2, (m,), generator=g)
        t[::3] = v
        t[1::7] = 2 ** 31 - 1
        t[2::7] = -2 ** 31
        return t
    assert kind == "nothing"
    return torch.full((m,), -1)


KINDS = ["uniform", "skewed", "one", "all different", "falling", "padded", "outside", "nothing"]


def lookup(table, tokens, y, scale):
    G._call("embedding_i_ij", table.dtype, table.data_ptr(), tokens.data_ptr(), y.data_ptr(), scale, tokens.element_size(), table.shape[0],
            tokens.numel(), table.shape[1])


def scratch_for(dtype, v, m, n):
    return G.Guarded((int(G.lib()[0].mpEmbeddingReverseScratchBytes(G.KEY[dtype], v, m, n)),), torch.uint8)


def lookup_reverse(tokens, dy, dt, scratch, scale, alpha=0.0):
    G._call("embedding_i_ij_reverse", dy.dtype, tokens.data_ptr(), dy.data_ptr(), dt.data_ptr(), scratch.data_ptr(), scale, alpha,
            tokens.element_size(), dt.shape[0], tokens.numel(), dt.shape[1])


def check(dtype, kind, v, m, n, scale=1.0, alpha=0.0, wide=True, shifts=(0, 0, 0, 0)):
    what = f"{dtype} {kind} v={v} m={m} n={n} scale={scale} alpha={alpha} {'64' if wide else '32'}-bit ids shifts {shifts}"
    tokens = ids_of(kind, m, v).to(torch.int64 if wide else torch.int32)
    table, dy, old = normal((v, n), dtype, 1), normal((m, n), dtype, 2), normal((v, n), dtype, 5)
    dy[tokens < 0] = float("nan")  # the gradient of a padded place is in no sum
    t, k, y = guarded(table, shifts[0]), tokens.cuda(), G.Guarded((m, n), dtype, shifts[1], fill=float("nan"))
    G.say(f"lookup {what}")
    lookup(t.t, k, y.t, scale)
    torch.cuda.synchronize()
    t.check(what), y.check(what)
    P.close(y.t, *P.embedding(table, tokens, scale, dtype), f"lookup {what}")
    d, dt, sc = guarded(dy, shifts[2]), guarded(old if alpha else torch.full_like(old, float("nan")), shifts[3]), scratch_for(dtype, v, m, n)
    sc.t.fill_(255)
    G.say(f"lookup reverse {what}")
    lookup_reverse(k, d.t, dt.t, sc.t, scale, alpha)
    torch.cuda.synchronize()
    d.check(what), dt.check(what), sc.check(what)
    P.close(dt.t, *P.embedding_reverse(tokens, dy, v, scale, dtype, alpha, old), f"lookup reverse {what}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_kinds_of_tokens(dtype, kind):
    for v, m, n in ((1, 1, 1), (1, 9, 8), (50, 7, 33), (300, 64, 64), (511, 700, 40), (512, 1025, 16), (700, 3000, 24), (40000, 2500, 8)):
        check(dtype, kind, v, m, n, scale=0.75)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 3, 5, 8, 15, 16, 17, 60, 64, 127, 128, 129, 500, 512, 1000, 1024, 1030, 2048, 2304, 4096, 4100])
def test_widths_of_rows(dtype, n):
    check(dtype, "skewed", 90, 150, n, scale=2.5)
    check(dtype, "padded", 90, 41, n, alpha=1.0, wide=False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("alpha", [0.0, 1.0, -0.5])
@pytest.mark.parametrize("wide", [True, False])
def test_blends(dtype, alpha, wide):
    for kind in ("skewed", "outside", "nothing", "one"):
        check(dtype, kind, 130, 260, 72, scale=-1.5, alpha=alpha, wide=wide)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [24, 256, 1024])
@pytest.mark.parametrize("shifts", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 1, 1, 1)])
def test_operands_off_their_alignment(dtype, n, shifts):
    check(dtype, "skewed", 70, 90, n, scale=0.5, alpha=1.0, shifts=shifts)
    check(dtype, "skewed", 70, 90, n, scale=0.5, alpha=0.0, shifts=shifts)


@pytest.mark.parametrize("m", [1, 2, 63, 64, 65, 1023, 1024, 1025, 4095, 4096, 4097, 8191, 8192, 8193, 16385, 20000, 66000, 270000])
def test_numbers_of_tokens(m):
    """Around a wavefront, a tile of the sort, one workgroup's whole sort, and past 256 tiles."""
    check(F32, "skewed", 5000, m, 4, scale=1.0)
    check(F16, "uniform", 20, m, 4, scale=0.01)


@pytest.mark.parametrize("v", [1, 2, 510, 511, 512, 513, 1023, 262143, 262144, 300000])
def test_sizes_of_the_table(v):
    """Around what one, two and three passes of the sort hold."""
    check(F32, "uniform", v, 3000, 4)
    check(F32, "falling", v, 1500, 4, alpha=1.0)


def test_rows_beyond_32_bit_offsets():
    """A table, and a gradient, of more than 2^32 bytes and elements at its far end."""
    v, n = 150000, 32768  # 4.9e9 elements of two bytes
    table = torch.zeros(v, n, dtype=F16, device="cuda")
    tokens = torch.tensor([v - 1, 0, 140000, v - 1, -1, 140000, 5], device="cuda")
    table[tokens.clamp(min=0)] = normal((7, n), F16, 1).cuda()
    y = torch.empty(7, n, dtype=F16, device="cuda")
    G.say("lookup in a table past 2^32 elements")
    lookup(table, tokens, y, 2.0)
    torch.cuda.synchronize()
    want = 2.0 * table[tokens.clamp(min=0)]
    want[4] = 0
    assert torch.equal(y, want)
    dy = normal((7, n), F16, 2).cuda()
    sc = scratch_for(F16, v, 7, n)
    table.fill_(7.0)
    G.say("lookup reverse of a table past 2^32 elements")
    lookup_reverse(tokens, dy, table, sc.t, 1.0)
    torch.cuda.synchronize()
    sc.check("scratch")
    named = [0, 5, 140000, v - 1]
    ref = torch.stack([dy[1].float(), dy[6].float(), dy[2].float() + dy[5].float(), dy[0].float() + dy[3].float()]).to(F16)
    assert torch.equal(table[named], ref)  # one addition and one rounding: exact as the plain form
    table[named] = 0
    assert not bool(table.any())


@pytest.mark.parametrize("dtype", TYPES)
def test_no_tokens(dtype):
    v, n = 37, 50
    none, dy = torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, n, dtype=dtype, device="cuda")
    for alpha in (0.0, 1.0, 0.5):
        dt = normal((v, n), dtype, 5).cuda()
        want = (dt.double() * alpha).to(dtype)
        if alpha == 0.0:
            dt.fill_(float("nan"))
        G.say(f"lookup reverse {dtype} without tokens, alpha {alpha}")
        lookup(dt, none, dy, 1.0)
        lookup_reverse(none, dy, dt, torch.empty(16, dtype=torch.uint8, device="cuda"), 1.0, alpha)
        torch.cuda.synchronize()
        assert torch.equal(dt, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_stay_in_their_row(dtype):
    v, m, n = 40, 200, 24
    tokens = ids_of("uniform", m, v)
    dy = normal((m, n), dtype, 2)
    dy[tokens == 7] = float("inf")
    dy[tokens == 9] = float("nan")
    tokens[:3] = torch.tensor([7, 9, 11])
    dt, sc = torch.empty(v, n, dtype=dtype, device="cuda"), scratch_for(dtype, v, m, n)
    dy[0], dy[1] = float("inf"), float("nan")
    G.say(f"lookup reverse {dtype} infinities")
    lookup_reverse(tokens.cuda(), dy.cuda(), dt, sc.t, 1.0)
    torch.cuda.synchronize()
    P.close(dt, *P.embedding_reverse(tokens, dy, v, 1.0, dtype), f"infinities {dtype}")
    assert bool(torch.isinf(dt[7]).all()) and bool(torch.isnan(dt[9]).all())


@pytest.mark.parametrize("dtype", [F16, F32])
def test_results_do_not_change_from_run_to_run(dtype):
    v, m, n = 300, 9000, 96
    tokens, dy = ids_of("skewed", m, v).cuda(), normal((m, n), dtype, 2).cuda()
    sc, first = scratch_for(dtype, v, m, n), None
    for k in range(5):
        dt = torch.empty(v, n, dtype=dtype, device="cuda")
        lookup_reverse(tokens, dy, dt, sc.t, 1.0)
        torch.cuda.synchronize()
        first = dt if first is None else first
        assert torch.equal(dt, first)


def test_the_gradient_agrees_with_differences():
    """The lookup is linear: a step of 1 in a direction gives the slope up to rounding."""
    v, m, n = 30, 80, 12
    tokens, table, dy, way = ids_of("padded", m, v).cuda(), normal((v, n), F64, 1).cuda(), normal((m, n), F64, 2).cuda(), normal((v, n), F64, 3).cuda()
    dt, sc = torch.empty_like(table), scratch_for(F64, v, m, n)
    lookup_reverse(tokens, dy, dt, sc.t, 3.0)
    up, down = torch.empty_like(dy), torch.empty_like(dy)
    lookup(table + way, tokens, up, 3.0)
    lookup(table - way, tokens, down, 3.0)
    assert abs(float(((up - down) * dy).sum()) / 2 - float((dt * way).sum())) < 1e-9


@pytest.mark.parametrize("m", [1, 2, 31, 33, 64, 127, 128, 129, 200, 255, 256, 257])
@pytest.mark.parametrize("kind", KINDS)
def test_few_tokens(m, kind):
    """Around a wavefront's votes and what one launch without a workspace takes; rows of one pack to several strips."""
    for dtype, n in ((F16, 5), (F32, 36), (F64, 130), (F16, 1000), (F32, 1500)):
        for v, alpha in ((1, 0.0), (90, 0.5), (700, 0.0)):
            check(dtype, kind, v, m, n, scale=0.5, alpha=alpha, wide=m % 2 == 0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 24, 77, 2048])
def test_no_token_scales_the_gradient(dtype, n):
    v, old = 37, normal((37, n), dtype, 5)
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    for alpha in (0.0, 1.0, -0.25):
        dt = guarded(old if alpha else torch.full_like(old, float("nan")))
        G._call("embedding_i_ij_reverse", dtype, none.data_ptr(), None, dt.t.data_ptr(), None, 2.0, alpha, 8, v, 0, n)
        assert torch.equal(dt.t.cpu(), (old.double() * alpha).to(dtype)), f"{dtype} n={n} alpha={alpha}"
        dt.check(f"no token {dtype} n={n} alpha={alpha}")


@pytest.mark.parametrize("m", [300, 9000])
def test_many_tokens_and_rows_beyond_32_bit_offsets(m):
    """As above, by both ways of ordering the tokens; named rows sit at both ends of the table."""
    v, n = 140000, 32768
    g = torch.full((v, n), 7.0, dtype=F16, device="cuda")
    tokens = torch.cat([torch.arange(m // 2), torch.arange(v - m // 3, v), torch.full((m - m // 2 - m // 3,), -1)])
    tokens = tokens[torch.randperm(m, generator=gen(4))].cuda()
    dy = torch.randn(m, n, device="cuda", dtype=torch.float32).to(F16)
    sc = scratch_for(F16, v, m, n)
    G.say(f"lookup reverse of {m} tokens, a table past 2^32 elements")
    lookup_reverse(tokens, dy, g, sc.t, 0.5)
    torch.cuda.synchronize()
    sc.check("scratch")
    order = torch.argsort(tokens)
    live = order[tokens[order] >= 0]  # every id once: halving is exact (or rounds as the plain form does)
    assert torch.equal(g[tokens[live]], dy[live] * 0.5)
    g[tokens[live]] = 0
    assert not bool(g.any())


@pytest.mark.parametrize("m", [200, 256, 300, 9000])
def test_a_common_id_keeps_small_addends(m):
    """One id whose first row is 1 and the others a little under half a step of 1 (in the type it is added in): a sum that
    goes through all places in turn in that type loses every one of them, m - 1 times 2^-24. The sums' bound is that of at
    most 64 additions in the type."""
    v, n = 5, 20
    for dtype in (F32, F64):
        tokens = torch.full((m,), 3)
        dy = torch.full((m, n), 0.99 * P.U[dtype], dtype=dtype)
        dy[0] = 1.0
        dt, sc = torch.full((v, n), float("nan"), dtype=dtype, device="cuda"), scratch_for(dtype, v, m, n)
        G.say(f"lookup reverse {dtype} of a common id, {m} places")
        lookup_reverse(tokens.cuda(), dy.cuda(), dt, sc.t, 1.0)
        torch.cuda.synchronize()
        # 0.99 * (m - 1) / 2^53 beside 1 is more than fp64 sums hold exactly: long double
        ref = np.zeros((v, n), np.longdouble)
        ref[3] = np.longdouble(1.0) + (m - 1) * np.longdouble(float(dy[1, 0]))
        err = np.abs(P.host64(dt).astype(np.longdouble) - ref)
        bound = (64 + 4 + 1) * P.U[dtype] * np.abs(ref)
        print(f"[bound] {dtype} {m} places: worst err/bound={float((err[3] / bound[3]).max()):.3f}", flush=True)
        assert bool((err <= bound).all()), float((err[3] / bound[3]).max())


@pytest.mark.parametrize("m,n", [(2 ** 29 + 3, 1), (2 ** 23 + 10, 2056)])
def test_more_rows_than_a_launch_has_threads(m, n):
    """A launch takes fewer than 2^32 threads: 2^24 workgroups of 32 narrow rows, or of half a row."""
    v = 211
    table = normal((v, n), F16, 1).cuda()
    tokens = (torch.arange(m, dtype=torch.int32, device="cuda") * 7) % (v + 1) - 1  # -1: a padded place
    y = torch.full((m, n), float("nan"), dtype=F16, device="cuda")
    G.say(f"lookup of {m} rows of {n}")
    lookup(table, tokens, y, 1.0)
    torch.cuda.synchronize()
    rows = torch.cat([torch.zeros(1, n, dtype=F16, device="cuda"), table])
    step = max(1, 2 ** 28 // n)
    for lo in range(0, m, step):
        assert torch.equal(y[lo:lo + step], rows[(tokens[lo:lo + step] + 1).long()]), f"rows from {lo}"


@pytest.mark.parametrize("m", [1, 256, 300, 9000])
@pytest.mark.parametrize("alpha", [0.0, 0.5])
def test_more_rows_to_clear_than_a_launch_has_threads(m, alpha):
    """A table of 2^30 + 64 narrow rows, which takes 2^24 + 1 workgroups to clear or to scale; by every way of
    ordering the places, named rows at both ends."""
    v = 2 ** 30 + 64
    g = torch.full((v, 1), 4.0, dtype=F16, device="cuda")
    tokens = torch.cat([torch.arange(m // 2), torch.arange(v - (m - m // 2), v)])[torch.randperm(m, generator=gen(4))]
    dy = normal((m, 1), F16, 2).cuda()
    sc = scratch_for(F16, v, m, 1)
    G.say(f"lookup reverse of {m} tokens, a table of {v} rows, alpha {alpha}")
    lookup_reverse(tokens.cuda(), dy, g, sc.t, 0.5, alpha)
    torch.cuda.synchronize()
    sc.check("scratch")
    named, rest = tokens.cuda(), 4.0 * alpha
    want = (dy.float() * 0.5 + rest).to(F16)  # every id once: exact in fp32, then rounded once
    assert torch.equal(g[named], want)
    g[named] = rest
    assert bool((g == rest).all())
