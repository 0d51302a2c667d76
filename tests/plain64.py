"""Plain implementations in 64 bits of layer normalisation, the embedding lookup and the clipping of
gradients, each with the bound that follows from its arithmetic.

Units: `u` is half a step of the type a kernel computes in (fp32 for r16 / r32, fp64 for r64), `half`
half a step of the storage type, which every stored result is rounded by once (r32 and r64 results are
in the type they are computed in: half = u). A sum of k terms in some order, every partial sum rounded,
is off by at most depth * u * sum |terms|, depth being the longest chain of additions a term goes
through. Bounds keep the first order in u."""
import numpy as np
import torch

U = {torch.float16: 2.0 ** -24, torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}
HALF = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}
# half of the smallest subnormal: what rounding is off by below the normal range
TINY = {torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150, torch.float64: 2.0 ** -1075}

# A row of up to 65536 elements is held by at least 64 lanes once it is longer than 512 elements, in no
# more than 1024 of their registers: a lane adds at most 64 elements in sequence for the lengths of these
# tests, lanes and wavefronts are folded in at most 16 further steps, the rest of a formula (a
# reciprocal square root good to one ulp, products, differences) is counted as 8.
ROW_DEPTH = 64 + 16 + 8


def host64(t):
    return None if t is None else t.detach().double().cpu().numpy()


def close(got, ref, bound, what):
    """|got - ref| <= bound everywhere; infinities and NaNs where the reference has them."""
    g, ref, bound = host64(got), np.asarray(ref, np.float64), np.asarray(bound, np.float64)
    assert g.shape == ref.shape, f"{what}: shape {g.shape} vs {ref.shape}"
    if g.size == 0:
        return
    same = (g == ref) | (np.isnan(g) & np.isnan(ref))
    with np.errstate(invalid="ignore"):
        err = np.where(same, 0.0, np.abs(g - ref))
        bad = ~same & ~(err <= bound)
        ratio = np.where(same, 0.0, np.where(np.isfinite(err), err / np.maximum(bound, 1e-320), np.inf))
    at = np.unravel_index(int(np.argmax(ratio)), ref.shape)
    print(f"[bound] {what}: n={g.size} worst err/bound={ratio[at]:.3f}", flush=True)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {g.size} outside; worst at {at}: got {g[at]!r} ref {ref[at]!r} "
                           f"err {err[at]:.3e} bound {np.broadcast_to(bound, ref.shape)[at]:.3e}")


# ---------------------------------------------------------------- layer normalisation

def _stats(x, eps):
    with np.errstate(invalid="ignore"):
        # the mean of a row near 1000 is itself off by 1000 * 2^-53, more than a kernel in fp64 is: the
        # differences' own mean, zero but for that, is taken off again
        d = x - x.mean(axis=-1, keepdims=True)
        d = d - d.mean(axis=-1, keepdims=True)
        r = 1.0 / np.sqrt((d * d).mean(axis=-1, keepdims=True) + eps)
        return d, r


def layernorm(x, gain, bias, eps, dtype):
    """(y, bound). x - c is exact or off by u of itself for a pivot c near the mean, the mean of those
    differences by depth * u of their mean size (at most the row's deviation), and r by half the
    variance's relative error: h = (x - mean) * r is off by at most K * u * (1 + |h|), K = ROW_DEPTH."""
    x, u = host64(x), U[dtype]
    g = 1.0 if gain is None else host64(gain)
    b = 0.0 if bias is None else host64(bias)
    d, r = _stats(x, eps)
    with np.errstate(invalid="ignore"):
        h = d * r
        y = h * g + b
        bound = u * ROW_DEPTH * np.abs(g) * (1 + np.abs(h)) + 2 * u * (np.abs(h * g) + np.abs(b)) + HALF[dtype] * np.abs(y) + TINY[dtype]
    return y, bound


def layernorm_reverse(x, gain, dy, eps, dtype, alpha=0.0, old=(None, None, None)):
    """((dx, dg, db), bounds). With e = dy * g, A = mean|e|, B = mean|e * h| and h off by K * u * (1 + |h|):
    mean(e) is off by K*u*A, mean(e * h) by K*u*(A + 2B), so dx = r * (e - mean(e) - h * mean(e*h)) by at
    most K*u*r * (2|e| + 2A + |h| * (A + 3B) + (1 + |h|) * B). dg and db add m terms; a chain of them is no
    longer than one workgroup's share of the rows (at least 128 workgroups, or a row each) and its
    groups, 16 rows, so D = m / 128 + 48 additions; the partial rows are added in fp64."""
    x, dy, u = host64(x), host64(dy), U[dtype]
    m, n = x.shape
    g = 1.0 if gain is None else host64(gain)
    d, r = _stats(x, eps)
    with np.errstate(invalid="ignore"):
        h, e = d * r, dy * g
        mean_e, mean_eh = (e.mean(-1, keepdims=True), (e * h).mean(-1, keepdims=True)) if n else (0.0, 0.0)
        A, B = (np.abs(e).mean(-1, keepdims=True), np.abs(e * h).mean(-1, keepdims=True)) if n else (0.0, 0.0)
        dx = r * (e - mean_e - h * mean_eh)
        bx = ROW_DEPTH * u * r * (2 * np.abs(e) + 2 * A + np.abs(h) * (A + 3 * B) + (1 + np.abs(h)) * B)
        dg, db = (dy * h).sum(0), dy.sum(0)
        depth = m / 128 + 48
        bg = ROW_DEPTH * u * (np.abs(dy) * (1 + np.abs(h))).sum(0) + depth * u * np.abs(dy * h).sum(0)
        bb = depth * u * np.abs(dy).sum(0)
        out, bounds = [], []
        for val, b, o in ((dx, bx, old[0]), (dg, bg, old[1]), (db, bb, old[2])):
            if alpha != 0.0:
                b = b + 2 * u * np.abs(alpha * host64(o))
                val = val + alpha * host64(o)
            out.append(val)
            bounds.append(b + HALF[dtype] * np.abs(val) + TINY[dtype])
    return out, bounds


# ---------------------------------------------------------------- embedding

def embedding(table, tokens, scale, dtype):
    """(y, bound): the factor is rounded to the computing type, the product once, the result once."""
    t, ids = host64(table), tokens.cpu().numpy().astype(np.int64)
    y = np.zeros((ids.size, t.shape[1]))
    inside = (ids >= 0) & (ids < t.shape[0])
    y[inside] = t[ids[inside]] * scale
    return y, (2 * U[dtype] + HALF[dtype]) * np.abs(y) + TINY[dtype]


def embedding_reverse(tokens, dy, v, scale, dtype, alpha=0.0, old=None):
    """(dT, bound): at most 64 terms are added in the computing type, the rest in fp64, the factor is
    rounded and multiplied once."""
    d, ids = host64(dy), tokens.cpu().numpy().astype(np.int64)
    out, size = np.zeros((v, d.shape[1])), np.zeros((v, d.shape[1]))
    for i, k in enumerate(ids):
        if 0 <= k < v:
            out[k] += d[i]
            size[k] += np.abs(d[i])
    out *= scale
    bound = (64 + 4) * U[dtype] * abs(scale) * size
    if alpha != 0.0:
        bound = bound + 2 * U[dtype] * np.abs(alpha * host64(old))
        out = out + alpha * host64(old)
    return out, bound + HALF[dtype] * np.abs(out) + TINY[dtype]


# ---------------------------------------------------------------- the norm of many tensors

def gradient_norm(tensors, alpha=0.0, old=0.0):
    """Squares and sums are fp64 throughout: 1e-12 allows chains of thousands of additions."""
    s = sum(float((host64(t) ** 2).sum()) for t in tensors)
    norm = float(np.sqrt(s + (alpha * old * old if alpha else 0.0)))
    return norm, 1e-12 * norm


def clipped(t, norm, max_norm, dtype):
    """(out, bound): the factor is rounded once, the product once, the result once."""
    g = host64(t)
    with np.errstate(invalid="ignore", divide="ignore"):
        out = g * (1.0 if norm <= max_norm else max_norm / norm)
        return out, (2 * U[dtype] + HALF[dtype] + 1e-12) * np.abs(out) + TINY[dtype]
