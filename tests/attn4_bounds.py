"""Outputs of the 4-bit cache's attention in 64 bits with how far each of them may be off, counted for each value from the
weights and the magnitudes in its own group of 32 values, so that one large value loosens no other output."""
import numpy as np

from tests import attn4_oracle as orc

HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def takes_prompt_kernel(torch, entries, max_rows, heads, kv):
    """whether an attend call of 16-bit rows is one of the prompt kernel's (the rule of tr_gpu_attn4_attend_dev)"""
    sm = torch.cuda.get_device_properties(0).multi_processor_count
    rows = max_rows * (heads // kv)
    tiles, ctas = -(-rows // 16) * kv * entries, -(-rows // 256) * kv * entries
    return rows > 8 and 2 * tiles >= 7 * sm * -(-ctas // sm)


def attention(q, k, v, scale, kind, prompt=False, seen=None):
    """(out, tolerance), both of q's shape (heads, head_dim); k, v: held rows (positions, KV heads, head_dim), finite;
    seen: (KV heads, positions) truth values.

    With M_t the largest |v_t| of the output's group (so |m| + 15 d <= 3 M_t) and p_t the weights:
    - a score is off by at most size_t (160 / 2^24 + 2^-23 + 4 / 2^24) (its terms' sum, q in two parts, the factor), the
      exponential by 2^-21; prompts round each key to f16: 2^-11 size_t, and 2^-25 a query value where a key is smaller
      than f16's normal numbers. A weight's relative error e_t counts above and below the fraction bar: 2 sum p_t e_t M_t.
    - 16-bit rows: p is rounded to f16 (above and below: 2 x 2^-11 M_t), p d once more (2^-11 x 15 d <= 2^-11 x 2 M_t), and
      the tensor core's sums of subnormal codes drop at most 2^-13 of 15 d; prompts round the values instead (2^-11 M_t
      and 2^-25). Together 5 x 2^-11 sum p_t M_t.
    - f32 rows: p and p d in two parts each 2^-21, the minimum's term 2^-21, additions: 2^-17 sum p_t M_t holds them.
    - what f16 drops below its smallest number: 2^-25 of p, whose largest is at least 2^7 (f32 rows 2^14) over 2^ed, ed the
      binary logarithm of the KV head's largest value scale where that is above 1: 2^(ed - 32) x 3 M_t a position (f32: 2^(ed -
      39)); and as much of each code's share 15 p d, where scales below 2^-8 are multiplied up to 1: 15 x 2^(ed - 32) x min(1,
      2^8 x the KV head's largest d) a position (d <= 2 M / 15).
    - the output's rounding: half a step, or 2^-25 below f16's normal numbers."""
    kv = k.shape[1]
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    n, hd = k.shape[0], q.shape[-1]
    g = q.reshape(kv, -1, hd)
    s = np.einsum("hgd,thd->hgt", g, k) * scale
    size = np.einsum("hgd,thd->hgt", abs(g), abs(k)) * abs(scale)
    off = size * (164 / 2 ** 24 + 2.0 ** -23) + 2.0 ** -21
    if prompt:
        off = off + size * 2.0 ** -11 + abs(g).sum(-1, keepdims=True) * abs(scale) * 2.0 ** -25
    if seen is not None:
        s = np.where(seen[:, None, :], s, -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    out = np.einsum("hgt,thd->hgd", p, v)
    m = abs(v).reshape(n, kv, -1, 32).max(-1)
    weight = p * (2 * np.where(p > 0, off, 0) + (2.0 ** -17 if kind == "f32" else 5 * 2.0 ** -11))
    tol = np.einsum("hgt,thx->hgx", weight, m)
    if not prompt:
        x = v.reshape(n, kv, -1, 32)
        d = (x.max(-1) - x.min(-1)).max((0, 2)) / 15  # (KV heads)
        low = 2.0 ** (np.maximum(0, np.frexp(d)[1]) - (39.0 if kind == "f32" else 32.0))
        tol += low[:, None, None] * (3 * m.sum(0) + n * 15 * np.minimum(1, 256 * d)[:, None])[:, None]
    else:
        tol += 2.0 ** -32 * 3 * m.sum(0)[:, None]
    tol = np.repeat(tol, 32, -1) + abs(out) * HALF_STEP[kind] + (2.0 ** -25 if kind == "f16" else 0) + 1e-37
    return out.reshape(q.shape), tol.reshape(q.shape)


def far(got, want, tol):
    """the largest error over its tolerance (NaN where an output is one and should not be)"""
    return float((abs(got - want) / tol).max())


def far_in_norm(got, want, kind, spread=0.0):
    """The largest error of a (row, head) in norm over what outputs of values of mean 0 may be off by, whose sums leave
    little of the values: errors of the positions are independent there, as the values are. With p's rounding (2^-11 of each
    term) and p d's (2^-11 of c d, which is about twice the value in norm) the error is below 2^-11 sqrt(1 + 4) < 2^-10 x 1.2
    of the output, and below half a step more by its own rounding. spread (prompts): the largest norm of q k's terms in a
    score, whose keys are rounded by 2^-11 independently."""
    size = {"f32": 2.0 ** -17, "bf16": 1.2 * 2.0 ** -10 + 2.0 ** -8, "f16": 1.2 * 2.0 ** -10 + 2.0 ** -11}[kind] + spread * 2.0 ** -11
    return float((np.linalg.norm(got - want, axis=-1) / (size * np.linalg.norm(want, axis=-1))).max())


def held_in(torch, kind, a):
    """a rounded to the kind's type, as float32"""
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[kind]
    return torch.from_numpy(np.ascontiguousarray(a)).to(t).float().numpy()


def seen_of(blocks, pos):
    """(KV heads, pos + 1) truth values of selected blocks (KV heads, n_sel)"""
    seen = np.zeros((blocks.shape[0], (pos // orc.BLOCK + 1) * orc.BLOCK), bool)
    for h, row in enumerate(blocks):
        for b in row[row >= 0]:
            seen[h, b * orc.BLOCK:(b + 1) * orc.BLOCK] = True
    return seen[:, :pos + 1]
