"""The prompt kernel of the 4-bit KV cache (many 16-bit query rows) on shapes that reach it, which each test checks first:
against definitions in 64 bits with bounds for each value and for each row's norm (tests/attn4_bounds.py)."""
import numpy as np
import pytest

from tests import attn4_bounds as bnd
from tests.test_gpu_attention4 import Session, _rows

pytestmark = pytest.mark.gpu

KINDS = ("bf16", "f16")


def _check(s, entries, q, kind, scale=None, norms=True):
    """attend against the definition for every row that has an entry; rows of padding stay as they were"""
    assert bnd.takes_prompt_kernel(s.torch, len(entries), max(e[2] for e in entries), s.heads, s.kv)
    q = bnd.held_in(s.torch, kind, q)
    scale = s.hd ** -0.5 if scale is None else scale
    got, row = s.attend(entries, q, kind, scale), 0
    for slot, pos0, rows in entries:
        for pos in range(pos0, pos0 + rows):
            if slot < 0:
                assert (got[row] == 99.0).all()
            else:
                k, v = s.k[slot, :pos + 1], s.v[slot, :pos + 1]
                want, tol = bnd.attention(q[row], k, v, scale, kind, prompt=True)
                far = bnd.far(got[row], want, tol)
                assert far <= 1, (slot, pos, far)
                if norms:
                    spread = np.sqrt(np.einsum("hgd,thd->hgt", (q[row] * scale).reshape(s.kv, -1, s.hd) ** 2.0, k ** 2.0).max())
                    far = bnd.far_in_norm(got[row], want, kind, spread)
                    assert far <= 1, (slot, pos, far)
            row += 1
    s.s.check()
    return got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd", ((32, 8, 128), (20, 4, 64), (14, 2, 128), (9, 9, 64), (24, 3, 64), (40, 8, 128)))
def test_ragged_prompts(cuda, kind, heads, kv, hd):
    """tiles that end inside a token's heads, inside a record and inside a block; entries of one row, of none and of padding
    beside long ones; starts far into a sequence"""
    rng = np.random.default_rng(41)
    ctx = 520
    s = Session(cuda, 5, heads, kv, hd, ctx)
    s.write([(i, 0, ctx) for i in range(5)], *_rows(rng, 5 * ctx, kv, hd), kind)
    longest = next(n for n in range(100, 500) if bnd.takes_prompt_kernel(cuda, 7, n, heads, kv))
    entries = [(2, 0, longest), (0, ctx - 97, 97), (-1, 0, 3), (1, 131, 1), (4, 7, 0), (3, 200, 65), (4, 0, 1)]
    n = sum(e[2] for e in entries)
    _check(s, entries, 1.5 * rng.normal(size=(n, heads, hd)), kind)
    _check(s, entries, 1.5 * rng.normal(size=(n, heads, hd)), kind, scale=-0.05)
    s.close()


def _session(cuda, rng, kind, change, kv=4, ctx=300):
    s = Session(cuda, 2, 8 * kv, kv, 128, ctx)
    k, v = _rows(rng, 2 * ctx, kv, 128)
    change(k.reshape(2, ctx, kv, 128), v.reshape(2, ctx, kv, 128))
    s.write([(0, 0, ctx), (1, 0, ctx)], k, v, kind)
    return s, rng.normal(size=(2 * ctx, 8 * kv, 128)).astype(np.float32)


def test_values_past_16_bits(cuda):
    """keys and values that a cache of bf16 rows holds but f16 does not: the tiles are made again in other units. What one
    position of one head holds loosens no other head, no other group and no row before it"""
    def change(k, v):
        v[0, 90, 1, 7], v[0, 200, 0, 100], v[1, 131, 3, 64:96] = 8e5, 1e5, np.linspace(-65000, 9e5, 32)
        k[1, 40, 2, 5] = 3e5  # (of another head than the large values)
    rng = np.random.default_rng(42)
    s, q = _session(cuda, rng, "bf16", change)
    assert np.isfinite(s.k).all() and np.isfinite(s.v).all() and s.k.max() > 65504 and s.v.max() > 65504
    _check(s, [(0, 0, 300), (1, 0, 300)], q, "bf16", norms=False)
    _check(s, [(0, 0, 300), (1, 0, 300)], 1e-6 * q, "bf16", norms=False)
    s.close()


@pytest.mark.parametrize("kind", KINDS)
def test_nan_in_seen_and_unseen_places(cuda, kind):
    """a NaN among the keys reaches the heads of its KV head from its position on, one among the values its group; a row
    before it, another head and another sequence are as if it were not there"""
    def change(k, v):
        k[0, 100, 0, 3], v[0, 150, 1, 70], k[0, 299, 3, 5], v[0, 33, 2, 1] = np.nan, np.inf, -np.inf, np.nan
    rng = np.random.default_rng(43)
    s, q = _session(cuda, rng, kind, change)
    got = s.attend([(0, 0, 300), (1, 0, 300)], q, kind)
    nan = np.zeros((600, 32, 128), bool)
    nan[100:300, :8], nan[150:300, 8:16, 64:96], nan[299, 24:], nan[33:300, 16:24, :32] = True, True, True, True
    assert np.array_equal(np.isnan(got), nan)
    s.k[0, 100:, 0], s.k[0, 299, 3], s.v[0, 150:, 1, 64:96], s.v[0, 33:, 2, :32] = 0, 0, 0, 0  # (the finite rest, as held)
    held = bnd.held_in(cuda, kind, q)
    for row in (0, 32, 33, 99, 100, 149, 150, 220, 298, 299, 300, 410, 599):
        slot, pos = divmod(row, 300)
        want, tol = bnd.attention(held[row], s.k[slot, :pos + 1], s.v[slot, :pos + 1], 128 ** -0.5, kind, prompt=True)
        ok = nan[row] | (abs(got[row] - want) <= tol)
        if slot == 0 and pos >= 100:
            ok[:8] = True  # (all NaN)
        assert ok.all(), row
    s.close()


@pytest.mark.parametrize("kind", KINDS)
def test_both_kernels_agree_on_a_mixed_batch(cuda, kind):
    """one prompt and many decode rows in one call (the prompt kernel's) and in two: within the bounds of both, whatever
    max_rows says"""
    rng = np.random.default_rng(44)
    s, q = _session(cuda, rng, kind, lambda k, v: None)
    entries = [(0, 0, 300)] + [(1, 13 * i, 1) for i in range(20)]
    assert bnd.takes_prompt_kernel(cuda, 21, 300, 32, 4) and not bnd.takes_prompt_kernel(cuda, 20, 1, 32, 4)
    one = _check(s, entries, q[:320], kind)
    two = s.attend(entries[1:], q[300:320], kind)
    held = bnd.held_in(cuda, kind, q)
    for i in range(20):
        want, tol = bnd.attention(held[300 + i], s.k[1, :13 * i + 1], s.v[1, :13 * i + 1], 128 ** -0.5, kind)
        assert bnd.far(two[i], want, tol) <= 1 and bnd.far_in_norm(two[i], want, kind) <= 1, i
    assert np.isfinite(one).all()
    s.close()
