"""The ends of a token model's training step as they are used together: embedding, layer norm, softmax
and their reverses, the table's gradient and the clipping of all gradients; through the launchers in
every type, on two streams at once, replayed from captured graphs, and through the C++ graph."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

import gpu_lib as G
import oracle_lib as O
import plain64 as P
from metaphor_amd import ffi

pytestmark = pytest.mark.gpu
F16, F32, F64 = torch.float16, torch.float32, torch.float64
EPS, SCALE, MAX_NORM = 1e-5, 1.5, 0.5


class Step:
    """Operands, workspaces and results of one step; `enqueue(call)` runs it, call(stem, dtype, *args)
    enqueueing a launcher on the stream the step belongs to."""

    def __init__(self, dtype, v, m, n, seed):
        kernels, _ = G.lib()
        key = G.KEY[dtype]
        g = torch.Generator()
        g.manual_seed(seed)
        mk = lambda *s, scale=1.0, shift=0.0: (torch.randn(s, generator=g, dtype=F64) * scale + shift).to(dtype).cuda()  # noqa: E731
        self.dtype, self.v, self.m, self.n = dtype, v, m, n
        self.table, self.gain, self.bias, self.dp = mk(v, n), mk(n, scale=0.1, shift=1.0), mk(n, scale=0.1), mk(m, n)
        tokens = torch.randint(0, v, (m,), generator=g) * torch.randint(0, 2, (m,), generator=g)
        tokens[::11] = -1
        self.tokens = tokens.cuda()
        like = lambda t: torch.full_like(t, float("nan"))  # noqa: E731
        self.x, self.h, self.p, self.dh, self.dx = (like(self.dp) for _ in range(5))
        self.dgain, self.dbias, self.dtable = like(self.gain), like(self.bias), like(self.table)
        self.norm = torch.full((1,), float("nan"), dtype=F64, device="cuda")
        self.clipped = [like(t) for t in (self.dtable, self.dgain, self.dbias)]
        size = lambda b: torch.empty(max(16, int(b)), dtype=torch.uint8, device="cuda")  # noqa: E731
        self.s_norm, self.s_emb = size(kernels.mpLayernormReverseScratchBytes(key, m, n)), size(kernels.mpEmbeddingReverseScratchBytes(key, v, m, n))
        self.s_clip = size(kernels.mpGradientNormScratchBytes(key, 3))
        self.grads = (ctypes.c_void_p * 3)(*[t.data_ptr() for t in (self.dtable, self.dgain, self.dbias)])
        self.outs = (ctypes.c_void_p * 3)(*[t.data_ptr() for t in self.clipped])
        self.sizes = (ctypes.c_ulong * 3)(v * n, n, n)

    def enqueue(self, call):
        d, m, n = self.dtype, self.m, self.n
        p = lambda t: t.data_ptr()  # noqa: E731
        call("embedding_i_ij", d, p(self.table), p(self.tokens), p(self.x), SCALE, 8, self.v, m, n)
        call("layernorm_ij_j", d, p(self.x), p(self.gain), p(self.bias), p(self.h), EPS, m, n)
        call("softmax_ij_j", d, p(self.h), p(self.p), None, m, n)
        call("softmax_ij_j_reverse", d, p(self.p), p(self.dp), p(self.dh), None, 0.0, m, n)
        call("layernorm_ij_j_reverse", d, p(self.x), p(self.gain), p(self.dh), p(self.dx), p(self.dgain), p(self.dbias), p(self.s_norm), EPS, 0.0, m, n)
        call("embedding_i_ij_reverse", d, p(self.tokens), p(self.dx), p(self.dtable), p(self.s_emb), SCALE, 0.0, 8, self.v, m, n)
        call("gradient_clip", d, self.grads, self.outs, self.sizes, p(self.norm), p(self.s_clip), MAX_NORM, 3)

    def results(self):
        return [self.x, self.h, self.p, self.dh, self.dx, self.dgain, self.dbias, self.dtable, self.norm, *self.clipped]

    def check(self, what):
        """Every stage against the plain form of what the stage before it left."""
        d = self.dtype
        c = lambda t: t.cpu()  # noqa: E731
        P.close(self.x, *P.embedding(c(self.table), c(self.tokens), SCALE, d), f"{what} x")
        P.close(self.h, *P.layernorm(c(self.x), c(self.gain), c(self.bias), EPS, d), f"{what} h")
        G.compare(self.p, O.softmax_ij_j(G.host(self.h)), d, f"{what} p", **G.softmax_tol(d))
        ph, dph = G.host(self.p), G.host(self.dp)
        G.compare(self.dh, O.softmax_ij_j_reverse(ph, dph), d, f"{what} dh", scale=G.softmax_reverse_scale(ph, dph))
        refs, bounds = P.layernorm_reverse(c(self.x), c(self.gain), c(self.dh), EPS, d)
        for name, got, ref, bound in zip(("dx", "dgain", "dbias"), (self.dx, self.dgain, self.dbias), refs, bounds):
            P.close(got, ref, bound, f"{what} {name}")
        P.close(self.dtable, *P.embedding_reverse(c(self.tokens), c(self.dx), self.v, SCALE, d), f"{what} dtable")
        grads = [c(t) for t in (self.dtable, self.dgain, self.dbias)]
        norm, bound = P.gradient_norm(grads)
        P.close(self.norm, np.array([norm]), np.array([bound]), f"{what} norm")
        for t, g in zip(self.clipped, grads):
            P.close(t, *P.clipped(g, norm, MAX_NORM, d), f"{what} clipped")


@pytest.mark.parametrize("dtype", [F16, F32, F64])
@pytest.mark.parametrize("v,m,n", [(60, 1, 8), (500, 300, 96), (40, 33, 257), (3000, 9000, 64), (700, 513, 1024)])
def test_a_step(dtype, v, m, n):
    s = Step(dtype, v, m, n, seed=v + m)
    G.say(f"step {dtype} v={v} m={m} n={n}")
    s.enqueue(G._call)
    torch.cuda.synchronize()
    s.check(f"{dtype} [{v},{m},{n}]")


def test_two_streams_at_once():
    """Each with operands and workspaces of its own and nothing but its own order."""
    a, b = Step(F32, 900, 700, 512, 1), Step(F16, 5000, 9000, 128, 2)
    with G.BlasStream() as s0, G.BlasStream() as s1:
        torch.cuda.synchronize()
        G.say("two steps on two streams")
        for _ in range(3):
            a.enqueue(s0.enqueue)
            b.enqueue(s1.enqueue)
        s0.sync()
        s1.sync()
    a.check("first stream")
    b.check("second stream")


def test_replays_of_captured_steps_match_eager():
    """Two graphs, one of each way the places are ordered, which share the workspace of the embedding's
    gradient: their replays are ordered, with eager work between them, and new operands each time."""
    a, b = Step(F32, 900, 700, 512, 3), Step(F32, 400, 9000, 72, 4)
    shared = a.s_emb if a.s_emb.numel() > b.s_emb.numel() else b.s_emb
    a.s_emb = b.s_emb = shared
    for s in (a, b):
        s.enqueue(G._call)
    torch.cuda.synchronize()
    graphs = []
    for s in (a, b):
        graph = torch.cuda.CUDAGraph()
        G.say("capture")
        with torch.cuda.graph(graph):
            s.enqueue(G._call)
        graphs.append(graph)
    for replay in range(4):
        for s in (a, b):
            s.tokens.copy_(s.tokens.roll(replay + 1))
            s.dp.mul_(-0.5)
            for t in s.results():
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        G.say(f"replay {replay}")
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in s.results()] for s in (a, b)]
        for s, r in zip((a, b), got):
            s.enqueue(G._call)  # eager work of the program between replays
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(r, s.results())), f"replay {replay}"
    a.check("after the replays")
    b.check("after the replays")


def test_on_a_side_stream_of_torch():
    s = Step(F32, 300, 257, 640, 5)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        s.enqueue(G._call)  # the context of torch's current stream
    side.synchronize()
    s.check("side stream")


@pytest.mark.parametrize("m,n", [(1, 4096), (30, 200), (256, 96), (3, 20000)])
def test_replays_of_a_captured_short_batch(m, n):
    s = Step(F16, 700, m, n, 6)
    s.enqueue(G._call)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    G.say(f"capture of a short batch {m}x{n}")
    with torch.cuda.graph(graph):
        s.enqueue(G._call)
    for replay in range(4):
        s.tokens.copy_((s.tokens + replay * 37) % 700)
        s.dp.mul_(-0.5)
        for t in s.results():
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in s.results()]
        s.enqueue(G._call)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, s.results())), f"replay {replay}"
    s.check("after the replays")


def _load(d, name, shape, dtype=np.float32):
    return torch.from_numpy(np.fromfile(os.path.join(d, name + ".bin"), dtype=dtype).reshape(shape))


def test_through_the_host_graph(tmp_path):
    exe = os.path.join(ffi.LIB_DIR, "host_check")
    G.say("host_check (token model)")
    res = subprocess.run([exe, str(tmp_path)], capture_output=True, text=True, timeout=120)
    print(res.stdout, res.stderr)
    assert res.returncode == 0, res.stderr
    assert "embedding / layer norm / clipping through the graph ok" in res.stdout
    d, v, m, n, k = str(tmp_path), 50, 37, 24, 11
    ids = _load(d, "tok_ids", (m,), np.int32)
    table, gain, bias, w = _load(d, "tok_table", (v, n)), _load(d, "tok_gain", (n,)), _load(d, "tok_bias", (n,)), _load(d, "tok_w", (n, k))
    x, h, p, dp = _load(d, "tok_x", (m, n)), _load(d, "tok_h", (m, n)), _load(d, "tok_p", (m, k)), _load(d, "tok_dp", (m, k))
    P.close(x, *P.embedding(table, ids, 2.0, F32), "host x")
    P.close(h, *P.layernorm(x, gain, bias, 1e-5, F32), "host h")
    logits, scale = O.inner_product(h.numpy(), w.numpy(), 1.0, with_scale=True)
    G.compare(p, O.softmax_ij_j(logits.astype(np.float32)), F32, "host p", atol=4e-6)  # softmax of logits off by 1e-6 of their terms

    # the gradients in 64 bits from the definition, by autograd; r32 intermediates are each off by at most a few 1e-6
    # of their terms, which is what the tolerance of 2e-5 of the largest term covers
    T, g, b, W = (t.double().requires_grad_() for t in (table, gain, bias, w))
    inside = (ids >= 0)[:, None]
    X = torch.where(inside, T[ids.clamp(min=0).long()] * 2.0, torch.zeros(()))
    C = X - X.mean(-1, keepdim=True)
    H = C / torch.sqrt((C * C).mean(-1, keepdim=True) + 1e-5)
    Y = H * g + b
    first = torch.autograd.grad((torch.softmax(Y @ W, -1) * dp.double()).sum(), (T, g, b, W), retain_graph=True)
    near = lambda got, ref: float((got.double() - ref).abs().max()) <= 2e-5 * float(ref.abs().max())  # noqa: E731
    for name, ref in zip(("dtable", "dgain", "dbias", "dw"), first):
        assert near(_load(d, "tok_" + name, ref.shape), ref), name
    second = torch.autograd.grad((H * g * h.double()).sum(), (T, g))
    assert near(_load(d, "tok_dtable2", (v, n)), first[0] + second[0]) and near(_load(d, "tok_dgain2", (n,)), first[1] + second[1])

    # the norm over two dtypes, from the gradients as they stand
    grads = [_load(d, "tok_dtable2", (v, n)), _load(d, "tok_dgain2", (n,)), _load(d, "tok_dbias", (n,)), _load(d, "tok_dw", (n, k)),
             torch.tensor([3.0, -4.0, 0.5, 0.0, 1.0], dtype=F64)]
    norm, bound = P.gradient_norm(grads)
    got = float(_load(d, "tok_norm", (1,), np.float64))
    assert abs(got - norm) <= bound, (got, norm)
    P.close(_load(d, "tok_clipped_table", (v, n)), *P.clipped(grads[0], norm, 0.75, F32), "clipped table")
    P.close(_load(d, "tok_clipped_bias", (n,)), *P.clipped(grads[2], norm, 0.75, F32), "clipped bias")
    P.close(_load(d, "tok_clipped_d", (5,), np.float64), *P.clipped(grads[4], norm, 0.75, F64), "clipped d")
