"""The 4-bit cache's operators in 64 bits on the CPU (numpy), from the definitions in include/trmoe.h, and the error
bounds that their 32-bit forms keep."""
import numpy as np

BLOCK = 64


def held(x):
    """the values that rows x (.., head_dim; any float type) stand for once the cache holds them, as float32"""
    with np.errstate(all="ignore"):
        g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
        lo, hi = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
        m = lo.astype(np.float16).astype(np.float64)
        d = (np.maximum(hi - m, 0) / 15).astype(np.float16).astype(np.float64)
        bad = ~np.isfinite(m) | ~np.isfinite(d) | ~np.isfinite(g).all(-1, keepdims=True)
        c = np.clip(np.rint(np.divide(g - m, d, out=np.zeros_like(g), where=d > 0)), 0, 15)
        return np.where(bad, np.nan, m + d * c).astype(np.float32).reshape(x.shape)


def unit_of(most):
    return np.ldexp(1.0, np.frexp(np.float64(most))[1] - 7)


def bounds(k):
    """(lo, hi, unit) of each whole block of one sequence's held keys (positions, KV heads, head_dim)"""
    n = k.shape[0] // BLOCK
    b = k[:n * BLOCK].astype(np.float64).reshape(n, BLOCK, *k.shape[1:])
    lo, hi = b.min(1), b.max(1)
    bad = np.isnan(lo).any(-1)
    unit = np.where(bad, np.inf, unit_of(np.maximum(abs(lo), abs(hi)).max(-1)))
    with np.errstate(invalid="ignore"):
        return (np.where(bad[..., None], 0, np.clip(np.floor(lo / unit[..., None]), -127, 127)),
                np.where(bad[..., None], 0, np.clip(np.ceil(hi / unit[..., None]), -127, 127)), unit)


def selected(k, q, pos, n_sel):
    """the blocks (KV heads, n_sel; -1 behind the last) that a query q (heads, head_dim) at pos attends to"""
    kv, home = k.shape[1], pos // BLOCK
    lo, hi, unit = bounds(k)
    q = np.asarray(q, np.float64).reshape(kv, -1, q.shape[-1])
    out = np.full((kv, n_sel), -1, np.int32)
    for h in range(kv):
        if np.isfinite(q[h]).all():
            z = np.clip(np.rint(q[h] / unit_of(abs(q[h]).max())), -127, 127)
        else:
            z = np.zeros_like(q[h])
        whole = (np.maximum(z, 0).sum(0) * hi[:home, h] + np.minimum(z, 0).sum(0) * lo[:home, h]).sum(-1)
        with np.errstate(invalid="ignore"):
            score = np.where(np.isinf(unit[:home, h]), np.inf, whole.astype(np.float32) * unit[:home, h])
        best = np.argsort(-score, kind="stable")[:n_sel - 1]
        ids = np.sort(np.append(best, home))
        out[h, :len(ids)] = ids
    return out


def attention(q, k, v, scale, seen=None):
    """(out, scores' magnitude): q (heads, head_dim) over held keys and values (positions, KV heads, head_dim);
    seen: (KV heads, positions) truth values"""
    kv = k.shape[1]
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    g = q.reshape(kv, -1, q.shape[-1])
    s = np.einsum("hgd,thd->hgt", g, k) * scale
    size = np.einsum("hgd,thd->hgt", abs(g), abs(k)) * abs(scale)
    if seen is not None:
        s = np.where(seen[:, None, :], s, -np.inf)
        size = np.where(seen[:, None, :], size, 0)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return np.einsum("hgt,thd->hgd", p, v).reshape(q.shape), float(np.nanmax(size))


def tolerance(size, v, out, kind):
    """How far an output may be from the 64-bit one.
    Scores: a product's terms are summed in 32 bits, at most head_dim + 32 roundings one after another over terms of
    magnitude `size` in sum, and q enters as two 16-bit floats (22 bits: 2^-23 at most): (160 / 2^24 + 2^-23) x size, and
    the multiplication by log2(e) and the subtraction of the maximum add 4 / 2^24 x size. A probability is off by that
    relative amount and by 2^-21 of the exponential, above and below the fraction bar, so the output by twice it times
    the values' largest magnitude. The sums over positions add 2^-24 a position at most, at most 2^12 of them here one
    after another: 2^-12 in the worst case, and their roundings' mean is 0: 2^-17 bounds 64 standard deviations.
    The 16-bit types: a probability times a scale is rounded twice to 16 bits (2 x 2^-11), the minimum's term once, and
    the result once by half a step of the type. Prompts round the keys and the values themselves to 16 bits: 2^-11 x size
    in a score, and once more on the values."""
    big = float(np.nanmax(abs(v)))
    tol = 2 * big * (size * (164 / 2 ** 24 + 2 ** -23) + 2 ** -21) + big * 2 ** -17
    if kind != "f32":
        tol += 2 * big * size * 2 ** -11 + big * 4 * 2 ** -11 + abs(out) * (2 ** -8 if kind == "bf16" else 2 ** -11)
    return tol + 1e-30
