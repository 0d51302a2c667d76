"""Layer normalisation on the GPU against the plain form in 64 bits: every type, rows of one element to
rows beyond one workgroup's registers, operands at any alignment, blends, and the values where a
variance goes wrong."""
import numpy as np
import pytest
import torch

import gpu_lib as G
import plain64 as P

pytestmark = pytest.mark.gpu
F16, F32, F64 = torch.float16, torch.float32, torch.float64
TYPES = [F16, F32, F64]
EPS = 1e-5


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(shape, dtype, seed, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=gen(seed), dtype=F64) * scale + shift).to(dtype)


def guarded(t, shift=0):
    g = G.Guarded(tuple(t.shape), t.dtype, shift)
    g.t.copy_(t)
    return g


def forward(x, gain, bias, y, eps=EPS):
    m, n = x.shape
    G._call("layernorm_ij_j", x.dtype, x.data_ptr(), gain.data_ptr() if gain is not None else None,
            bias.data_ptr() if bias is not None else None, y.data_ptr(), eps, m, n)


def scratch_for(dtype, m, n):
    return G.Guarded((int(G.lib()[0].mpLayernormReverseScratchBytes(G.KEY[dtype], m, n)),), torch.uint8)


def reverse(x, gain, dy, dx, dg, db, scratch, eps=EPS, alpha=0.0):
    m, n = x.shape
    G._call("layernorm_ij_j_reverse", x.dtype, x.data_ptr(), gain.data_ptr() if gain is not None else None, dy.data_ptr(), dx.data_ptr(),
            dg.data_ptr() if dg is not None else None, db.data_ptr() if db is not None else None, scratch.data_ptr(), eps, alpha, m, n)


def check_forward(x, gain, bias, what, shifts=(0, 0, 0, 0), eps=EPS, in_place=False):
    dt = x.dtype
    X = guarded(x, shifts[0])
    g = guarded(gain, shifts[1]) if gain is not None else None
    b = guarded(bias, shifts[2]) if bias is not None else None
    Y = X if in_place else G.Guarded(tuple(x.shape), dt, shifts[3], fill=float("nan"))
    G.say(f"layernorm forward {what}")
    forward(X.t, g.t if g else None, b.t if b else None, Y.t, eps)
    torch.cuda.synchronize()
    for k in (X, Y, g, b):
        if k is not None:
            k.check(what)
    ref, bound = P.layernorm(x, gain, bias, eps, dt)
    P.close(Y.t, ref, bound, f"layernorm {what}")


def check_reverse(x, gain, dy, what, shifts=(0, 0, 0, 0, 0), eps=EPS, alpha=0.0, want=(True, True), in_place=False):
    dt = x.dtype
    m, n = x.shape
    old = [normal(s, dt, 90 + k) for k, s in enumerate(((m, n), (n,), (n,)))]
    if in_place:
        old[0] = dy
    start = old if alpha else [torch.full_like(o, float("nan")) for o in old]
    X, D = guarded(x, shifts[0]), guarded(dy, shifts[1])
    g = guarded(gain, shifts[2]) if gain is not None else None
    dx = D if in_place else guarded(start[0], shifts[3])
    dg, db = (guarded(s, shifts[4]) if w else None for s, w in zip(start[1:], want))
    sc = scratch_for(dt, m, n)
    sc.t.fill_(255)
    G.say(f"layernorm reverse {what}")
    reverse(X.t, g.t if g else None, D.t, dx.t, dg.t if dg else None, db.t if db else None, sc.t, eps, alpha)
    torch.cuda.synchronize()
    for k in (X, D, g, dx, dg, db, sc):
        if k is not None:
            k.check(what)
    refs, bounds = P.layernorm_reverse(x, gain, dy, eps, dt, alpha, old)
    for name, got, ref, bound in zip(("dx", "dg", "db"), (dx, dg, db), refs, bounds):
        if got is not None:
            P.close(got.t, ref, bound, f"layernorm {name} {what}")


# one element; packs and their neighbours; a wavefront's worth of packs and its neighbours; ragged and
# whole rows around 4, 8 and 16 KiB; rows that a power-of-two group would leave partly idle
LENGTHS = [1, 2, 3, 7, 8, 9, 31, 64, 65, 100, 127, 128, 200, 257, 511, 512, 513, 768, 1000, 1024, 1027, 1280, 2047, 2048, 2560, 4096, 4100,
           5121, 6144]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", LENGTHS)
def test_rows_of_every_length(dtype, n):
    for m in (1, 5, 67):
        x, gain, bias, dy = normal((m, n), dtype, n, 2.0, 0.5), normal((n,), dtype, 2, 0.2, 1.0), normal((n,), dtype, 3, 0.3), normal((m, n), dtype, 4)
        check_forward(x, gain, bias, f"{dtype} [{m},{n}]")
        check_reverse(x, gain, dy, f"{dtype} [{m},{n}]")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [8192, 12288, 16384, 16388, 20000, 40961])
def test_long_rows(dtype, n):
    for m in (1, 6):
        x, gain, bias, dy = normal((m, n), dtype, n, 2.0, 0.5), normal((n,), dtype, 2, 0.2, 1.0), normal((n,), dtype, 3, 0.3), normal((m, n), dtype, 4)
        check_forward(x, gain, bias, f"{dtype} [{m},{n}]")
        check_reverse(x, gain, dy, f"{dtype} [{m},{n}]", alpha=1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(2500, 64), (3001, 200), (2100, 1024), (1031, 2560), (700, 5120)])
def test_many_rows(dtype, m, n):
    """More rows than the workgroups of a launch hold at once."""
    x, gain, bias, dy = normal((m, n), dtype, n, 2.0, 0.5), normal((n,), dtype, 2, 0.2, 1.0), normal((n,), dtype, 3, 0.3), normal((m, n), dtype, 4)
    check_forward(x, gain, bias, f"{dtype} [{m},{n}]")
    check_reverse(x, gain, dy, f"{dtype} [{m},{n}]", alpha=0.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [24, 256, 1024, 4096])
@pytest.mark.parametrize("shifts", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 1, 1, 1)])
def test_operands_off_their_alignment(dtype, n, shifts):
    m = 9
    x, gain, bias, dy = normal((m, n), dtype, n), normal((n,), dtype, 2, 0.2, 1.0), normal((n,), dtype, 3, 0.3), normal((m, n), dtype, 4)
    check_forward(x, gain, bias, f"{dtype} [{m},{n}] shifts {shifts}", shifts)
    check_reverse(x, gain, dy, f"{dtype} [{m},{n}] shifts {shifts}", (*shifts, shifts[0]), alpha=1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 96, 1024, 4096, 40960])
@pytest.mark.parametrize("alpha", [0.0, 1.0, -0.25])
def test_blends_and_results_that_are_not_wanted(dtype, n, alpha):
    m = 11
    x, gain, dy = normal((m, n), dtype, 1), normal((n,), dtype, 2, 0.2, 1.0), normal((m, n), dtype, 4)
    for want in ((True, True), (False, True), (True, False), (False, False)):
        check_reverse(x, gain, dy, f"{dtype} [{m},{n}] alpha {alpha} want {want}", alpha=alpha, want=want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [6, 256, 1024, 4096, 40960])
def test_no_gain_and_no_bias(dtype, n):
    m = 7
    x, gain, bias, dy = normal((m, n), dtype, 1), normal((n,), dtype, 2, 0.2, 1.0), normal((n,), dtype, 3), normal((m, n), dtype, 4)
    check_forward(x, None, None, f"{dtype} [{m},{n}] plain")
    check_forward(x, gain, None, f"{dtype} [{m},{n}] no bias")
    check_forward(x, None, bias, f"{dtype} [{m},{n}] no gain")
    check_reverse(x, None, dy, f"{dtype} [{m},{n}] no gain")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [9, 128, 1024, 4096, 5121, 40960])
def test_in_place(dtype, n):
    m = 7
    x, gain, bias, dy = normal((m, n), dtype, 1), normal((n,), dtype, 2, 0.2, 1.0), normal((n,), dtype, 3), normal((m, n), dtype, 4)
    check_forward(x, gain, bias, f"{dtype} [{m},{n}] in place", in_place=True)
    check_reverse(x, gain, dy, f"{dtype} [{m},{n}] dx over dy", in_place=True)
    check_reverse(x, gain, dy, f"{dtype} [{m},{n}] dx over dy, blended", in_place=True, alpha=0.5)


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("n", [8, 100, 1024, 4096, 5121, 40960])
def test_rows_far_from_zero(dtype, n):
    """A mean a thousand times the spread: the variance must not come from a difference of squares,
    and the mean's own rounding must not show."""
    x, gain, bias, dy = normal((5, n), dtype, 1, 1.0, 1000.0), normal((n,), dtype, 2, 0.2, 1.0), normal((n,), dtype, 3), normal((5, n), dtype, 4)
    check_forward(x, gain, bias, f"{dtype} n={n} mean 1000")
    check_reverse(x, gain, dy, f"{dtype} n={n} mean 1000")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 16, 1000, 4096, 40960])
def test_constant_rows(dtype, n):
    """No variance at all: (x - mean) is zero and r = 1/sqrt(eps)."""
    x = torch.tensor([[0.0], [3.0], [-1.5]], dtype=F64).expand(3, n).to(dtype).contiguous()
    gain, bias, dy = normal((n,), dtype, 2, 0.2, 1.0), normal((n,), dtype, 3), normal((3, n), dtype, 4, 0.01)
    check_forward(x, gain, bias, f"{dtype} constant rows n={n}")
    check_reverse(x, gain, dy, f"{dtype} constant rows n={n}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [64, 1024, 4096])
def test_one_large_value_in_a_row(dtype, n):
    x = normal((4, n), dtype, 1, 0.5)
    for i, j in enumerate((0, 1, n // 2, n - 1)):
        x[i, j] = 900.0
    gain, bias, dy = normal((n,), dtype, 2, 0.2, 1.0), normal((n,), dtype, 3), normal((4, n), dtype, 4)
    check_forward(x, gain, bias, f"{dtype} outliers n={n}")
    check_reverse(x, gain, dy, f"{dtype} outliers n={n}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [16, 1024, 4096, 40960])
def test_a_row_with_an_infinity_or_a_nan_spoils_itself_alone(dtype, n):
    x = normal((6, n), dtype, 1)
    x[1, n // 3], x[3, 0], x[4, n - 1] = float("inf"), float("nan"), float("-inf")
    gain, bias = normal((n,), dtype, 2, 0.2, 1.0), normal((n,), dtype, 3)
    X, g, b, Y = guarded(x), guarded(gain), guarded(bias), G.Guarded((6, n), dtype)
    G.say(f"layernorm forward {dtype} n={n} infinities")
    forward(X.t, g.t, b.t, Y.t)
    torch.cuda.synchronize()
    fine = [0, 2, 5]
    ref, bound = P.layernorm(x[fine], gain, bias, EPS, dtype)
    P.close(Y.t[fine], ref, bound, f"rows beside a spoilt one {dtype} n={n}")
    assert bool(torch.isnan(Y.t[[1, 3, 4]]).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_no_rows(dtype):
    n = 40
    empty = torch.empty((0, n), dtype=dtype, device="cuda")
    gain = normal((n,), dtype, 2).cuda()
    for alpha in (0.0, 1.0, 0.5):
        dg, db = normal((n,), dtype, 5).cuda(), normal((n,), dtype, 6).cuda()
        want = [alpha * t.double() if alpha else torch.zeros_like(t, dtype=F64) for t in (dg, db)]
        G.say(f"layernorm reverse {dtype} without rows, alpha {alpha}")
        forward(empty, gain, gain, empty)
        reverse(empty, gain, empty, empty, dg, db, torch.empty(16, dtype=torch.uint8, device="cuda"), EPS, alpha)
        torch.cuda.synchronize()
        assert all(torch.equal(t, w.to(dtype)) for t, w in zip((dg, db), want))


@pytest.mark.parametrize("dtype", [F16, F32])
def test_results_do_not_change_from_run_to_run(dtype):
    m, n = 1500, 1024
    x, gain, dy = normal((m, n), dtype, 1).cuda(), normal((n,), dtype, 2).cuda(), normal((m, n), dtype, 4).cuda()
    sc, first = scratch_for(dtype, m, n), None
    for k in range(4):
        dx, dg, db = torch.empty_like(x), torch.empty_like(gain), torch.empty_like(gain)
        reverse(x, gain, dy, dx, dg, db, sc.t)
        torch.cuda.synchronize()
        first = first or (dx, dg, db)
        assert all(torch.equal(a, b) for a, b in zip(first, (dx, dg, db)))


def test_the_gradient_agrees_with_differences():
    """Central differences of sum(dy * y) in double precision, one direction at a time: with a step of
    1e-5 they are off by the third derivative's 1e-10 and by 2^-53 / 1e-5 = 1e-11 of the sum."""
    m, n, step = 3, 37, 1e-5
    x, gain, bias, dy = (normal(s, F64, k).cuda() for k, s in enumerate(((m, n), (n,), (n,), (m, n))))
    dx, dg, db = torch.empty_like(x), torch.empty_like(gain), torch.empty_like(gain)
    reverse(x, gain, dy, dx, dg, db, scratch_for(F64, m, n).t)

    def value(x, gain, bias):
        y = torch.empty_like(x)
        forward(x, gain, bias, y)
        return float((y * dy).sum())

    for k, (t, grad) in enumerate(((x, dx), (gain, dg), (bias, db))):
        args = [x, gain, bias]
        for trial in range(4):
            way = normal(t.shape, F64, 50 + trial).cuda()
            up, down = list(args), list(args)
            up[k], down[k] = t + step * way, t - step * way
            slope = (value(*up) - value(*down)) / (2 * step)
            assert abs(slope - float((grad * way).sum())) < 1e-7 * max(1.0, abs(slope))


def test_rows_beyond_32_bit_offsets():
    """Operands of more than 2^32 elements, with values in their first and last rows."""
    m, n, k = 140000, 32768, 3
    part = torch.cat([torch.arange(k), torch.arange(m - k, m)])
    xs, ds, gain, bias = normal((2 * k, n), F16, 1), normal((2 * k, n), F16, 2), normal((n,), F16, 3), normal((n,), F16, 4)
    x, other = torch.zeros(m, n, dtype=F16, device="cuda"), torch.full((m, n), 9.0, dtype=F16, device="cuda")
    x[part] = xs.cuda()
    G.say("layernorm forward past 2^32 elements")
    forward(x, gain.cuda(), bias.cuda(), other)
    torch.cuda.synchronize()
    P.close(other[part], *P.layernorm(xs, gain, bias, EPS, F16), "layernorm past 2^32 elements")
    assert torch.equal(other[k:m - k:997].cpu(), bias.expand(len(range(k, m - k, 997)), n))  # rows of zeros
    other.zero_()
    other[part] = ds.cuda()
    dg, db, sc = torch.empty(n, dtype=F16, device="cuda"), torch.empty(n, dtype=F16, device="cuda"), scratch_for(F16, m, n)
    G.say("layernorm reverse past 2^32 elements")
    reverse(x, gain.cuda(), other, other, dg, db, sc.t)
    torch.cuda.synchronize()
    sc.check("scratch")
    refs, bounds = P.layernorm_reverse(xs, gain, ds, EPS, F16)  # rows without a gradient add nothing
    for name, got, ref, bound in zip(("dx", "dg", "db"), (other[part], dg, db), refs, bounds):
        P.close(got, ref, bound, f"{name} past 2^32 elements")
    assert not bool(other[k:m - k].any())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(1, 4096), (2, 4096), (4, 4096), (5, 4096), (16, 512), (32, 512), (33, 512), (64, 256), (65, 256), (130, 128), (257, 64), (4, 20000)])
def test_few_rows(dtype, m, n):
    """Around what one workgroup takes, which writes the vectors' gradients by itself."""
    x, dy, gain = normal((m, n), dtype, 1), normal((m, n), dtype, 2), normal((n,), dtype, 3)
    for alpha in (0.0, 0.5):
        check_reverse(x, gain, dy, f"{dtype} few rows {m}x{n} alpha {alpha}", alpha=alpha)
        check_reverse(x, gain, dy, f"{dtype} few rows {m}x{n} alpha {alpha}, off alignment", shifts=(1, 0, 0, 1, 1), alpha=alpha)
    check_reverse(x, gain, dy, f"{dtype} few rows {m}x{n}, no bias", want=(True, False))
    check_reverse(x, None, dy, f"{dtype} few rows {m}x{n}, no gain", want=(False, True), in_place=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n", [(7, 9), (5000, 24), (3000, 200), (3001, 1027), (2500, 2048), (1500, 5121), (600, 12288), (5, 40961)])
@pytest.mark.parametrize("alpha", [0.0, 0.5])
def test_many_rows_in_place(dtype, m, n, alpha):
    """Workgroups that walk several rows, with the next ones on their way while these are written: over dy, and over x."""
    x, gain, bias, dy = normal((m, n), dtype, 1), normal((n,), dtype, 2, 0.2, 1.0), normal((n,), dtype, 3), normal((m, n), dtype, 4)
    if alpha == 0.0:
        check_forward(x, gain, bias, f"{dtype} [{m},{n}] in place", in_place=True)
    check_reverse(x, gain, dy, f"{dtype} [{m},{n}] dx over dy alpha {alpha}", in_place=True, alpha=alpha)
    what = f"{dtype} [{m},{n}] dx over x alpha {alpha}"
    X, D, old = guarded(x), guarded(dy), [x, normal((n,), dtype, 5), normal((n,), dtype, 6)]
    dg, db, sc = guarded(old[1]), guarded(old[2]), scratch_for(dtype, m, n)
    G.say(f"layernorm reverse {what}")
    reverse(X.t, gain.cuda(), D.t, X.t, dg.t, db.t, sc.t, alpha=alpha)
    torch.cuda.synchronize()
    for k in (X, D, dg, db, sc):
        k.check(what)
    refs, bounds = P.layernorm_reverse(x, gain, dy, EPS, dtype, alpha, old)
    for name, got, ref, bound in zip(("dx", "dg", "db"), (X, dg, db), refs, bounds):
        P.close(got.t, ref, bound, f"layernorm {name} {what}")


@pytest.mark.parametrize("n", [8, 100, 1024, 4096, 5121, 8192, 12288, 16384, 40960])
def test_half_precision_rows_far_from_zero(n):
    """A mean a thousand times the spread, in the type whose pivot is the mean of all elements: sums about it come from
    sum - held * pivot. At 1000 an r16 step is 0.5, which the rows hold as their spread."""
    for mean in (1000.0, -30.0):
        x, gain, bias, dy = normal((5, n), F16, 1, 1.0, mean), normal((n,), F16, 2, 0.2, 1.0), normal((n,), F16, 3), normal((5, n), F16, 4)
        check_forward(x, gain, bias, f"r16 n={n} mean {mean}")
        check_reverse(x, gain, dy, f"r16 n={n} mean {mean}")


@pytest.mark.parametrize("n", [8, 100, 1024, 4096, 5121, 16384, 40960])
def test_subnormal_half_precision_values(n):
    """dy and x below the normal range of r16, of one sign, so that their sums and their means count: rows of little
    spread scale them up by up to 1 / sqrt(eps)."""
    for m in (1, 5, 300):
        dy = (normal((m, n), F16, 4).abs().double() * 1e-6).to(F16)
        assert bool((dy > 0).any()) and float(dy.max()) < 2.0 ** -14
        gain = normal((n,), F16, 2, 0.2, 1.0)
        check_reverse(normal((m, n), F16, 1, 2.0, 0.5), gain, dy, f"r16 [{m},{n}] subnormal dy")
        x = (normal((m, n), F16, 1).abs().double() * 1e-6).to(F16)
        check_forward(x, gain, None, f"r16 [{m},{n}] subnormal x", eps=1e-14)
        check_reverse(x, gain, dy, f"r16 [{m},{n}] subnormal x and dy", eps=1e-9)


@pytest.mark.parametrize("dtype,n", [(F32, 2 ** 28), (F64, 2 ** 27)])
def test_vectors_of_more_columns_than_a_launch_has_threads(dtype, n):
    """The last sums of dg and db by more workgroups than fewer than 2^32 threads make. Values whose sums are exact: x
    +1, -1, ... and dy +1, +1, -1, -1, ..., so every mean is zero, h is x * r and dx is dy * r."""
    x = torch.ones(2, n, dtype=dtype, device="cuda")
    x[:, 1::2] = -1.0
    dy = torch.ones(2, n, dtype=dtype, device="cuda")
    dy[:, 2::4] = -1.0
    dy[:, 3::4] = -1.0
    dy[1] *= 2.0
    dx, dg, db = torch.full_like(x, float("nan")), torch.full_like(x[0], float("nan")), torch.full_like(x[0], float("nan"))
    sc = scratch_for(dtype, 2, n)
    G.say(f"layernorm reverse {dtype} of rows of {n}")
    reverse(x, None, dy, dx, dg, db, sc.t, eps=1.0)
    torch.cuda.synchronize()
    sc.check("scratch")
    r = 2.0 ** -0.5
    # a reciprocal square root good to one ulp and four roundings
    near = lambda got, ref: float((got - ref).abs().max()) <= 8 * P.U[dtype] * 3.0  # noqa: E731
    assert torch.equal(db, dy[0] + dy[1])
    assert near(dg, (dy[0] + dy[1]) * x[0] * r)
    assert near(dx, dy * r)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,kib", [(1, 0), (2, 64), (3, 48), (4, 48)])
def test_what_one_workgroup_takes(dtype, m, kib):
    """Two rows of 64 KiB together, three or four of 48, are left to one workgroup, which writes dg and db itself and
    leaves the workspace alone; more go to a workgroup each, which leave their sums there. Rows long enough for a
    workgroup to hold one at a time, a little below and a little above."""
    each = kib * 1024 // dtype.itemsize // m // 16 * 16 - 16
    for n, alone in (((16384 // dtype.itemsize, True),) if m == 1 else ((each, True), (each + 32, False), (32768 // dtype.itemsize, m * 32 <= kib))):
        x, dy, gain = normal((m, n), dtype, 1), normal((m, n), dtype, 2), normal((n,), dtype, 3)
        dx, dg, db, sc = guarded(x), guarded(gain), guarded(gain), scratch_for(dtype, m, n)
        sc.t.fill_(255)
        what = f"{dtype} [{m},{n}] by {'one workgroup' if alone else 'several'}"
        G.say(f"layernorm reverse {what}")
        reverse(x.cuda(), gain.cuda(), dy.cuda(), dx.t, dg.t, db.t, sc.t)
        torch.cuda.synchronize()
        for k in (dx, dg, db, sc):
            k.check(what)
        assert bool((sc.t == 255).all()) == alone, what
        refs, bounds = P.layernorm_reverse(x, gain, dy, EPS, dtype)
        for name, got, ref, bound in zip(("dx", "dg", "db"), (dx, dg, db), refs, bounds):
            P.close(got.t, ref, bound, f"layernorm {name} {what}")


@pytest.mark.parametrize("n", [12280, 12288, 12289, 12296, 14001, 16376, 16384, 16385])
@pytest.mark.parametrize("alpha", [0.0, 1.0])
def test_half_precision_rows_around_the_plans_of_long_rows(n, alpha):
    """Where two packs a lane become four, which differs with a blend; more rows than workgroups, whole and ragged."""
    x, gain, dy = normal((600, n), F16, n, 2.0, 0.5), normal((n,), F16, 2, 0.2, 1.0), normal((600, n), F16, 4)
    check_reverse(x, gain, dy, f"r16 [600,{n}] alpha {alpha}", alpha=alpha)
    check_reverse(x[:7], gain, dy[:7], f"r16 [7,{n}] alpha {alpha} off alignment", shifts=(1, 1, 0, 1, 1), alpha=alpha)
