"""The norm of many tensors and clipping by it, on the GPU, against the plain form in 64 bits."""
import ctypes

import numpy as np
import pytest
import torch

import gpu_lib as G
import plain64 as P
from metaphor_amd import ffi

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


def addresses(tensors):
    return (ctypes.c_void_p * max(1, len(tensors)))(*[t.data_ptr() for t in tensors])


def lengths(tensors):
    return (ctypes.c_ulong * max(1, len(tensors)))(*[t.numel() for t in tensors])


def scratch_for(dtype, count):
    return G.Guarded((int(G.lib()[0].mpGradientNormScratchBytes(G.KEY[dtype], count)),), torch.uint8)


def norm_of(tensors, dtype, norm, alpha=0.0):
    sc = scratch_for(dtype, len(tensors))
    sc.t.fill_(255)
    G._call("gradient_norm", dtype, addresses(tensors), lengths(tensors), norm.data_ptr(), sc.t.data_ptr() if len(tensors) else None, alpha, len(tensors))
    torch.cuda.synchronize()
    sc.check("scratch")


def scale(tensors, outs, dtype, norm, max_norm):
    G._call("gradient_scale", dtype, addresses(tensors), addresses(outs), lengths(tensors), norm.data_ptr(), max_norm, len(tensors))


def clip(tensors, outs, dtype, norm, max_norm):
    sc = scratch_for(dtype, len(tensors))
    sc.t.fill_(255)
    G._call("gradient_clip", dtype, addresses(tensors), addresses(outs), lengths(tensors), norm.data_ptr(), sc.t.data_ptr(), max_norm, len(tensors))
    torch.cuda.synchronize()
    sc.check("scratch")


def a_norm(value=float("nan")):
    return torch.full((1,), value, dtype=F64, device="cuda")


def check(dtype, sizes, max_norm, what, in_place=False, shift=0, spread=1.0):
    plain = [normal((k,), dtype, 7 + i, spread) for i, k in enumerate(sizes)]
    src = [guarded(t, (i * shift) % 7) for i, t in enumerate(plain)]
    out = src if in_place else [G.Guarded((k,), dtype, (i * 3 * shift) % 5, fill=float("nan")) for i, k in enumerate(sizes)]
    norm = a_norm()
    G.say(f"clip {what}")
    clip([s.t for s in src], [o.t for o in out], dtype, norm, max_norm)
    ref, bound = P.gradient_norm(plain)
    P.close(norm, np.array([ref]), np.array([bound]), f"norm {what}")
    for k, (p, s, o) in enumerate(zip(plain, src, out)):
        s.check(what), o.check(what)
        P.close(o.t, *P.clipped(p, ref, max_norm, dtype), f"clipped {k} {what}")
        if not in_place:
            assert torch.equal(s.t.cpu(), p)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[1], [2], [7], [8], [9], [255, 1], [1024], [4097, 3, 0, 12], [0, 0, 5], [65536], [100003, 17, 8192, 31],
                                   [300007, 2, 2, 2, 2, 70001]])
@pytest.mark.parametrize("in_place", [False, True])
def test_tensors_of_every_size(dtype, sizes, in_place):
    check(dtype, sizes, 0.5, f"{dtype} {sizes} in place {in_place}", in_place)
    check(dtype, sizes, 0.5, f"{dtype} {sizes} in place {in_place} off alignment", in_place, shift=1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count", [2, 95, 96, 97, 192, 193, 500])
def test_numbers_of_tensors(dtype, count):
    """Around what the arguments of one launch hold."""
    check(dtype, [(37 * k) % 1000 for k in range(count)], 2.0, f"{dtype} {count} tensors")


@pytest.mark.parametrize("dtype", TYPES)
def test_a_norm_within_the_limit_leaves_the_values_as_they_are(dtype):
    for in_place in (False, True):
        for max_norm in (1e6, float("inf")):
            plain = [normal((k,), dtype, k) for k in (5, 40000, 129)]
            src = [t.cuda() for t in plain]
            out = src if in_place else [torch.full_like(t, float("nan")) for t in src]
            clip(src, out, dtype, a_norm(), max_norm)
            assert all(torch.equal(o.cpu(), p) for o, p in zip(out, plain))


@pytest.mark.parametrize("dtype,values", [(F16, (6e4, 6e-8)), (F32, (1e30, 1e-30)), (F64, (1e150, 1e-150))])
def test_values_whose_squares_leave_the_type(dtype, values):
    for value in values:
        t = torch.full((5000,), value, dtype=dtype, device="cuda")
        out, norm = torch.empty_like(t), a_norm()
        G.say(f"clip {dtype} values {value}")
        limit = float(t[0]) * 10
        clip([t], [out], dtype, norm, limit)
        ref, bound = P.gradient_norm([t.cpu()])
        P.close(norm, np.array([ref]), np.array([bound]), f"norm of {value}")
        P.close(out, *P.clipped(t.cpu(), ref, limit, dtype), f"clipped {value}")


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_to_add(dtype):
    norm = a_norm(3.0)
    G.say("norm of no tensors")
    norm_of([], dtype, norm, 1.0)
    assert float(norm) == 3.0
    norm_of([], dtype, norm, 0.0)
    assert float(norm) == 0.0
    zeros, out = torch.zeros(1000, dtype=dtype, device="cuda"), torch.ones(1000, dtype=dtype, device="cuda")
    clip([zeros], [out], dtype, norm, 0.0)
    assert float(norm) == 0.0 and not bool(out.any())


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nans_show_in_the_norm(dtype):
    t = normal((3000,), dtype, 1)
    for bad in (float("inf"), float("-inf"), float("nan")):
        t[1234] = bad
        src, out, norm = t.cuda(), torch.empty(3000, dtype=dtype, device="cuda"), a_norm()
        G.say(f"clip with {bad}")
        clip([src], [out], dtype, norm, 1.0)
        if np.isnan(bad):
            assert bool(torch.isnan(norm)) and bool(torch.isnan(out).all())
        else:
            assert float(norm) == float("inf")
            assert bool(torch.isnan(out[1234])) and int((out != 0).sum()) == 1  # 0 * inf alone is not zero


def test_tensors_of_three_types_under_one_norm():
    plain = {dt: [normal((k,), dt, k + 1) for k in sizes] for dt, sizes in ((F16, (500, 7)), (F32, (70000, 3)), (F64, (41,)))}
    dev = {dt: [t.cuda() for t in ts] for dt, ts in plain.items()}
    norm = a_norm()
    G.say("one norm over three types")
    for k, (dt, ts) in enumerate(dev.items()):
        norm_of(ts, dt, norm, 1.0 if k else 0.0)
    ref, bound = P.gradient_norm([t for ts in plain.values() for t in ts])
    P.close(norm, np.array([ref]), np.array([bound]), "norm over three types")
    for dt, ts in dev.items():
        scale(ts, ts, dt, norm, 1.0)
    torch.cuda.synchronize()
    for dt, ts in dev.items():
        for t, p in zip(ts, plain[dt]):
            P.close(t, *P.clipped(p, ref, 1.0, dt), f"scaled {dt}")


def test_the_same_tensor_twice():
    """Counted twice in the norm, written twice with the same values where the results are apart."""
    t = normal((3000,), F32, 1)
    src, a, b, norm = t.cuda(), torch.empty(3000, device="cuda"), torch.empty(3000, device="cuda"), a_norm()
    clip([src, src], [a, b], F32, norm, 1.0)
    ref, bound = P.gradient_norm([t, t])
    P.close(norm, np.array([ref]), np.array([bound]), "twice")
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_results_do_not_change_from_run_to_run(dtype):
    ts = [normal((k,), dtype, k).cuda() for k in (100000, 3, 70001)]
    first = None
    for _ in range(5):
        norm, outs = a_norm(), [torch.empty_like(t) for t in ts]
        clip(ts, outs, dtype, norm, 1.0)
        got = [norm, *outs]
        first = first or got
        assert all(torch.equal(x, y) for x, y in zip(got, first))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("count", [119, 120, 121, 122, 240, 241, 242])
@pytest.mark.parametrize("in_place", [False, True])
def test_numbers_of_runs(dtype, count, in_place):
    """Tensors apart from each other, around one and two launches' arguments."""
    check(dtype, [(37 * k) % 1000 + 1 for k in range(count)], 2.0, f"{dtype} {count} runs in place {in_place}", in_place, shift=1)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("count", [139, 140, 141, 195, 196, 197, 280, 281, 392, 393])
@pytest.mark.parametrize("in_place", [False, True])
def test_more_numbers_of_runs(dtype, count, in_place):
    """The same where results of their own take room among the arguments, and where none do."""
    check(dtype, [(37 * k) % 300 + 1 for k in range(count)], 2.0, f"{dtype} {count} runs in place {in_place}", in_place, shift=1)


def test_some_results_in_place_and_some_apart():
    plain = [normal((300 + k,), F32, k) for k in range(9)]
    src, norm = [guarded(t) for t in plain], a_norm()
    out = [s if k % 3 else G.Guarded((300 + k,), F32, 1, fill=float("nan")) for k, s in enumerate(src)]
    clip([s.t for s in src], [o.t for o in out], F32, norm, 1.0)
    ref, _ = P.gradient_norm(plain)
    for k, (p, s, o) in enumerate(zip(plain, src, out)):
        s.check(f"gradient {k}"), o.check(f"result {k}")
        P.close(o.t, *P.clipped(p, ref, 1.0, F32), f"clipped {k}")
        assert k % 3 or torch.equal(s.t.cpu(), p)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_pieces_that_the_last_launch_adds_up_or_not(dtype):
    """Around 2048 pieces of 16 KiB, and a last piece that ends in a pack, behind one and in the middle of one."""
    each = 16384 // dtype.itemsize
    for pieces in (2047, 2048, 2049):
        for less in (0, 1, each - 1, each // 2):
            check(dtype, [pieces * each - less], 3.0, f"{dtype} {pieces} pieces less {less} elements", in_place=True)


def test_a_tensor_of_more_than_2_32_elements():
    k = 2 ** 32 + 12345
    t, small = torch.zeros(k, dtype=F16, device="cuda"), torch.full((5,), 2.0, dtype=F16, device="cuda")
    where = torch.tensor([0, 2 ** 31 + 1, 2 ** 32 - 1, 2 ** 32, k - 1], device="cuda")
    t[where] = 4.0
    norm = a_norm()
    G.say("clip a tensor of more than 2^32 elements")
    clip([t, small], [t, small], F16, norm, 5.0)
    assert float(norm) == 10.0  # 5 * 16 + 5 * 4 under the root
    assert torch.equal(t[where], torch.full((5,), 2.0, dtype=F16, device="cuda")) and bool((small == 1.0).all())
    t[where] = 0
    assert not bool(t.any())


@pytest.mark.parametrize("dtype,value,limits", [(F32, 1e38, (1.0, 1e-2, 1e-6, 1e-30)), (F32, 3e38, (1e-8,)), (F64, 1e150, (1e-150, 1e-200)),
                                                (F16, 6e4, (1e-30, 1e-40))])
@pytest.mark.parametrize("count", [1, 9, 5003, 9000001])
@pytest.mark.parametrize("in_place", [False, True])
def test_factors_below_the_range_of_the_type(dtype, value, limits, count, in_place):
    """max_norm / norm is subnormal or zero in the computing type (for r64 in fp64 too), g * max_norm / norm is not:
    g / norm is at most one, so it is computed from that here. Both ways of scaling, up to 2048 pieces and more."""
    for limit in limits:
        g = normal((count,), dtype, 3, 0.25 * value)
        g = torch.where(g.abs() > value, torch.full_like(g, value), g)
        src, norm = g.cuda(), a_norm()
        out = src if in_place else torch.full_like(src, float("nan"))
        G.say(f"clip {dtype} {count} values of {value} to {limit}")
        clip([src], [out], dtype, norm, limit)
        ref, bound = P.gradient_norm([g])
        P.close(norm, np.array([ref]), np.array([bound]), f"norm of {value}")
        want = P.host64(g) / ref * limit
        # the norm is off by 1e-12 of itself, the product is rounded a few times in fp64, the result once
        P.close(out, want, (4 * P.U[F64] + P.HALF[dtype] + 1e-12) * np.abs(want) + P.TINY[dtype], f"clipped {value} to {limit}")


def test_a_largest_norm_of_zero_and_an_infinite_norm():
    """A factor of zero: zeros with their sign kept out of the comparison, NaN where the gradient is infinite."""
    for dtype in TYPES:
        t = normal((3000,), dtype, 1)
        out, norm = torch.full_like(t, float("nan")).cuda(), a_norm()
        clip([t.cuda()], [out], dtype, norm, 0.0)
        assert not bool(out.any()) and float(norm) > 0
        t[17] = float("inf")
        src = t.cuda()
        clip([src], [src], dtype, norm, 0.5)
        assert float(norm) == float("inf") and bool(torch.isnan(src[17])) and int((src != 0).sum()) == 1
