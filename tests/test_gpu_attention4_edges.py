"""The 4-bit KV cache at the edges of what its calls allow: values, queries and scales that 16- and 32-bit numbers hold
barely, against definitions in 64 bits with bounds for each value (tests/attn4_bounds.py)."""
import numpy as np
import pytest

from tests import attn4_bounds as bnd
from tests import attn4_oracle as orc
from tests.test_gpu_attention4 import KINDS, Session, _rows

pytestmark = pytest.mark.gpu


def _check(s, entries, q, kind, scale=None, n_sel=None, prompt=False):
    """attend (or select) against the definition, value by value; got"""
    q = bnd.held_in(s.torch, kind, q)
    scale = s.hd ** -0.5 if scale is None else scale
    got, row = s.attend(entries, q, kind, scale, n_sel), 0
    got, blocks = got if n_sel else (got, None)
    for slot, pos0, rows in entries:
        for pos in range(pos0, pos0 + rows):
            seen = None
            if n_sel:
                assert np.array_equal(blocks[row], orc.selected(s.k[slot], q[row], pos, n_sel)), (slot, pos)
                seen = bnd.seen_of(blocks[row], pos)
            want, tol = bnd.attention(q[row], s.k[slot, :pos + 1], s.v[slot, :pos + 1], scale, kind, prompt, seen)
            far = bnd.far(got[row], want, tol)
            assert far <= 1, (slot, pos, far)
            row += 1
    return got


def _prompt(s, rows, kind, entries=2):
    """entries of `rows` rows from position 0 on, enough for the prompt kernel"""
    assert kind != "f32" and bnd.takes_prompt_kernel(s.torch, entries, rows, s.heads, s.kv)
    return [(i, 0, rows) for i in range(entries)]


def _single(s, entries, q, kind, scale, n_sel=None):
    """rows of which one position has all the weight: its value, to the output's rounding (prompts': and f16's)"""
    got, row = s.attend(entries, q, kind, scale, n_sel), 0
    got = got[0] if n_sel else got
    for slot, pos0, rows in entries:
        for pos in range(pos0, pos0 + rows):
            want = np.repeat(s.v[slot, pos], s.heads // s.kv, 0)
            size = np.repeat(abs(want).reshape(s.heads, -1, 32).max(-1), 32, -1).reshape(want.shape)
            tol = size * ((2.0 ** -17 if kind == "f32" else 5 * 2.0 ** -11) + bnd.HALF_STEP[kind])
            far = bnd.far(got[row], want, tol)
            assert far <= 1, (slot, pos, scale, far)
            row += 1


def test_near_constant_groups(cuda):
    """groups whose values differ by less than their minimum's last place: scales among f16's smallest numbers, rounded by
    up to a third, so that quotients pass 15"""
    rng = np.random.default_rng(31)
    rows = []
    for base in (1.0, -1.0, 0.125, -0.125, 0.25, 0.5, -0.5, 2.0, 1000.0, 0.0999755859375):
        ulp = float(np.spacing(np.float32(abs(base))))
        for reach in (1, 2, 5, 8, 11, 16, 21, 22, 23, 24, 40, 63, 90, 150, 217, 230):  # in 2^-24, the least d
            n = max(1, int(reach * 2.0 ** -24 / ulp))
            for up in (1, -1):
                j = rng.integers(0, n + 1, size=32)
                j[:2] = 0, n
                rows.append(np.float32(base) + np.float32(ulp) * (up * j).astype(np.float32))
        rows.append(np.full(32, np.nextafter(np.float32(base), np.float32(2e3)), np.float32))
    rows.append((1 + np.minimum(np.arange(32), 11) * 2.0 ** -23).astype(np.float32))
    while len(rows) % 2:
        rows.append(np.zeros(32, np.float32))
    x = np.stack(rows).reshape(-1, 1, 64)
    s = Session(cuda, 1, 1, 1, 64, x.shape[0])
    s.write([(0, 0, x.shape[0])], x, x[::-1])
    gk, gv = s.read([(0, 0, x.shape[0])])
    assert np.array_equal(gk, s.k[0]) and np.array_equal(gv, s.v[0])
    s.close()


def test_f32_rows_over_wide_values(cuda):
    """value groups up to f16's limits (m + 15 d up to 16 x 65504) among ordinary ones, at positions that rows see and at
    positions of the same record that they do not"""
    rng = np.random.default_rng(32)
    s = Session(cuda, 1, 4, 2, 128, 300)
    k, v = _rows(rng, 300, 2, 128)
    v[70, 0, 5], v[70, 1, 40], v[200, 0, 64:96] = 2e5, -6e4, np.linspace(65504, 65504 * 16, 32)
    v[130, 1, 96:] = np.linspace(-65504, 65504 * 14, 32)
    s.write([(0, 0, 300)], k, v)
    assert np.isfinite(s.v).all() and s.v.max() > 1e6
    q = rng.normal(size=(8, 4, 128)).astype(np.float32)
    for entries in ([(0, 69, 1), (0, 70, 1), (0, 71, 1), (0, 128, 2), (0, 199, 2), (0, 299, 1)], [(0, 64, 8)], [(0, 196, 8)]):
        n = sum(e[2] for e in entries)
        _check(s, entries, q[:n], "f32")
        _check(s, entries, q[:n], "f32", n_sel=2)
    got = s.s.decode(0, 0, 299, q[0], k[299], v[299], 0.1)
    want, tol = bnd.attention(q[0], s.k[0], s.v[0], 0.1, "f32")
    assert bnd.far(got, want, tol) <= 1
    s.s.check()
    s.close()


def test_f32_rows_over_small_values(cuda):
    """values of every size down to f16's smallest scales: what the minimum's two parts drop is relative to them"""
    rng = np.random.default_rng(33)
    s = Session(cuda, 1, 2, 2, 128, 500)
    for size in (1e-2, 1e-4, 3e-6):
        k, v = _rows(rng, 500, 2, 128)
        v[:, :, 32:] *= size
        s.write([(0, 0, 500)], k, v)
        _check(s, [(0, 499, 1), (0, 33, 1)], rng.normal(size=(2, 2, 128)), "f32")
    s.close()


@pytest.mark.parametrize("kind", ("bf16", "f16"))
def test_prompt_rows_that_are_not_finite(cuda, kind):
    """a query row with a NaN or an infinity among a prompt's is NaN in its head, and in no other row or head"""
    rng = np.random.default_rng(34)
    s = Session(cuda, 2, 32, 4, 128, 260)
    s.write([(0, 0, 260), (1, 0, 260)], *_rows(rng, 520, 4, 128), kind)
    q = rng.normal(size=(520, 32, 128)).astype(np.float32)
    entries = _prompt(s, 260, kind)
    clean = s.attend(entries, q, kind)
    bad = ((0, 3, 5), (17, 0, 0), (100, 31, 127), (259, 9, 64), (260, 8, 1), (400, 16, 33))
    for i, (r, h, x) in enumerate(bad):
        q[r, h, x] = (np.nan, np.inf, -np.inf)[i % 3]
    got = s.attend(entries, q, kind)
    for r, h, _ in bad:
        assert np.isnan(got[r, h]).all(), (r, h)
        got[r, h] = clean[r, h]
    assert np.array_equal(got, clean)
    s.close()


@pytest.mark.parametrize("kind", KINDS)
def test_scales_that_are_not_finite(cuda, kind):
    """a NaN or an infinity as scale gives NaN, whichever kernel a call takes"""
    rng = np.random.default_rng(35)
    s = Session(cuda, 2, 32, 4, 128, 260)
    s.write([(0, 0, 260), (1, 0, 260)], *_rows(rng, 520, 4, 128), kind)
    q = rng.normal(size=(520, 32, 128)).astype(np.float32)
    for scale in (np.nan, np.inf, -np.inf):
        assert np.isnan(s.attend([(0, 259, 1), (1, 0, 1)], q[:2], kind, scale)).all()
        out, blocks = s.attend([(0, 259, 1), (1, 0, 1)], q[:2], kind, scale, n_sel=2)
        assert np.isnan(out).all() and np.array_equal(blocks, s.attend([(0, 259, 1), (1, 0, 1)], q[:2], kind, 1.0, n_sel=2)[1])
        if kind != "f32":
            assert np.isnan(s.attend(_prompt(s, 260, kind), q, kind, scale)).all()
    if kind == "f32":
        assert np.isnan(s.s.decode(0, 0, 259, q[0], s.k[0, 259], s.v[0, 259], np.nan)).all()
    s.close()


@pytest.mark.parametrize("kind", ("f32", "bf16"))
def test_queries_near_the_largest_number(cuda, kind):
    """queries of 2^112 to 2^127 whose scale brings the scores back"""
    rng = np.random.default_rng(36)
    s = Session(cuda, 2, 32, 4, 128, 260)
    s.write([(0, 0, 260), (1, 0, 260)], *_rows(rng, 520, 4, 128), kind)
    q = rng.normal(size=(520, 32, 128)).astype(np.float32)
    for size in (112, 114, 120, 124):
        _check(s, [(0, 259, 1), (1, 100, 1)], np.ldexp(q[:2], size), kind, 0.1 * 2.0 ** -size)
    if kind != "f32":
        _prompt(s, 260, kind)
        _check(s, [(0, 0, 260), (1, 0, 260)], np.ldexp(q, 122), kind, 0.1 * 2.0 ** -122, prompt=True)
    s.close()


@pytest.mark.parametrize("kind", KINDS)
def test_scores_past_a_million(cuda, kind):
    """scores whose neighbours in 32 bits lie further apart than a softmax can tell: the best position has all the weight"""
    rng = np.random.default_rng(37)
    s = Session(cuda, 2, 32, 4, 128, 260)
    k, v = _rows(rng, 520, 4, 128)
    k[:] = np.sign(rng.normal(size=k.shape)) * (1 + np.arange(520) % 260)[:, None, None] / 260  # the later, the larger
    s.write([(0, 0, 260), (1, 0, 260)], k, v, kind)
    q = np.sign(rng.normal(size=(520, 32, 128))).astype(np.float32)
    for i in range(2):
        for r in range(260):
            q[260 * i + r] = np.repeat(np.sign(s.k[i, r]), 8, 0) + 0.0  # (its own key: no other is as large)
    for size in (1e5, 1e6, 3e6, 1e7, 3e7, 1e8, 1e9):
        scale = size / 128
        _single(s, [(0, 259, 1), (1, 0, 1), (1, 33, 1), (0, 100, 3)], q[[259, 260, 293, 100, 101, 102]], kind, scale)
        _single(s, [(0, 259, 1), (1, 200, 1)], q[[259, 460]], kind, scale, n_sel=2)
        if kind != "f32" and size <= 1e8:
            _single(s, _prompt(s, 260, kind), q, kind, scale)
    # scores that are all far below zero: the least far has the weight, and a row's first position sees itself alone
    for size in (1e8, 1e34, 1e36) if kind != "f16" else (1e8,):
        _single(s, [(0, 0, 1), (1, 0, 1)], -q[[0, 260]], kind, size / 128)
    s.close()


@pytest.mark.parametrize("size,sink,kind", [(1e-5, 20, "f32"), *[(size, 16, kind) for size in (1e-3, 1e-4, 3e-5) for kind in KINDS]])
def test_small_values_behind_a_sink(cuda, size, sink, kind):
    """values whose scales are f16's smallest, and one position whose weight is 2^sink times the others': what the others
    add is not lost"""
    rng = np.random.default_rng(38)
    n = 8192
    s = Session(cuda, 1, 2, 2, 128, n)
    k = (0.05 * rng.normal(size=(n, 2, 128))).astype(np.float32)
    v = (size * (1 + rng.normal(size=(n, 2, 128)))).astype(np.float32)
    q = np.sign(rng.normal(size=(1, 2, 128))).astype(np.float32)
    k[5] = q[0] * (sink * np.log(2) * 128 ** -0.5)
    v[5] *= 0.01
    s.write([(0, 0, n)], k, v, kind)
    got = _check(s, [(0, n - 1, 1)], q, kind)[0]
    want, _ = bnd.attention(bnd.held_in(cuda, kind, q)[0], s.k[0], s.v[0], 128 ** -0.5, kind)
    # f16 outputs of this size lie 2^-24 apart
    tol = np.linalg.norm(want) * {"f32": 2.0 ** -14, "bf16": 2.0 ** -8, "f16": 2.0 ** -10}[kind]
    assert np.linalg.norm(got - want) <= tol + (2.0 ** -25 * 16 if kind == "f16" else 0)
    s.close()


@pytest.mark.parametrize("kind", KINDS)
def test_values_that_grow(cuda, kind):
    """value scales that grow through 2^-24 .. 2^4 along a sequence, whose sums change their units on the way"""
    rng = np.random.default_rng(39)
    n = 4096
    s = Session(cuda, 1, 16, 2, 64, n)
    k, v = _rows(rng, n, 2, 64)
    v *= np.ldexp(1.0, -22 + np.arange(n) // 150)[:, None, None].astype(np.float32)
    s.write([(0, 0, n)], k, v, kind)
    q = 0.5 * rng.normal(size=(3, 16, 64))
    for at in (100, 700, 1700, 2400, 3300, n - 3):
        _check(s, [(0, at, 1), (0, at, 2)], q, kind)
        _check(s, [(0, at, 1), (0, at, 2)], q, kind, n_sel=5)
    s.close()


def test_more_selecting_rows_than_a_launch_holds(cuda):
    """max_rows x heads past a launch's size: refused (in 32 bits the size would wrap to a launch of one row)"""
    ctx = (1 << 23) + 1
    s = Session.__new__(Session)
    from trochilus_b200 import moe
    s.torch, s.moe, s.layer, s.heads, s.kv, s.hd, s.ctx, s.keep = cuda, moe, 0, 256, 1, 64, ctx, []
    s.s = moe.GpuAttn4(1, 1, 256, 1, 64, ctx)
    q, out = cuda.ones((2, 256 * 64), device="cuda"), cuda.zeros((2, 256 * 64), device="cuda")
    for n_tok, max_rows, want in ((ctx, ctx, -1), (ctx, 1 << 22, -1), (2, ctx, 0), (2, 2, 0)):
        b = s.batch([(0, 0, 2)], n_tok=n_tok, max_rows=max_rows)
        rc = moe.lib().tr_gpu_attn4_select_dev(s.s.a, 0, b, moe.F32, q.data_ptr(), 256 * 64, 0.1, 2, out.data_ptr(), 256 * 64, None,
                                               None)
        assert rc == want and (rc == 0 or "too many" in moe.last_error())
    s.s.check()
    s.s.close()
