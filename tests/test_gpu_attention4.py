"""The 4-bit KV cache on the GPU (tr_gpu_attn4_*) against its definitions in 64 bits (tests/attn4_oracle.py): rows
quantised and read back bit for bit, attention within bounds derived there, the selected blocks equal."""
import ctypes as C

import numpy as np
import pytest

from tests import attn4_oracle as orc

pytestmark = pytest.mark.gpu

KINDS = ("f32", "bf16", "f16")


def _kind(torch, moe, kind):
    return {"f32": (torch.float32, moe.F32), "bf16": (torch.bfloat16, moe.BF16), "f16": (torch.float16, moe.F16)}[kind]


class Session:
    """A session with a mirror of what its cache holds (numpy, float32) for one layer."""

    def __init__(self, torch, n_seq, heads, kv, hd, ctx, n_layers=1, layer=0):
        from trochilus_b200 import moe
        self.torch, self.moe, self.layer = torch, moe, layer
        self.heads, self.kv, self.hd, self.ctx = heads, kv, hd, ctx
        self.s = moe.GpuAttn4(n_layers, n_seq, heads, kv, hd, ctx)
        self.k = np.zeros((n_seq, ctx, kv, hd), np.float32)
        self.v = np.zeros((n_seq, ctx, kv, hd), np.float32)
        self.keep = []

    def batch(self, entries, n_tok=None, max_rows=None, starts=None):
        """entries: (slot, pos0, rows); rows one after another from row 0"""
        t = self.torch
        if starts is None:
            starts = np.cumsum([0] + [e[2] for e in entries])
        arr = [t.tensor(list(a), dtype=t.int32, device="cuda") for a in
               ([e[0] for e in entries], [e[1] for e in entries], starts)]
        self.keep.append(arr)
        return self.moe.Attn4Batch(len(entries), int(starts[-1]) if n_tok is None else n_tok,
                                   max_rows or max([1] + [e[2] for e in entries]), *[a.data_ptr() for a in arr])

    def write(self, entries, k, v, kind="f32", stream=0):
        """k, v: numpy (rows, kv, hd); returns nothing; the mirror follows"""
        t = self.torch
        dt, typ = _kind(t, self.moe, kind)
        dk, dv = (t.from_numpy(np.ascontiguousarray(a)).to("cuda").to(dt) for a in (k, v))
        row = self.kv * self.hd
        self.s.write_dev(self.layer, self.batch(entries), typ, dk.data_ptr(), row, dv.data_ptr(), row, stream=stream)
        t.cuda.synchronize()
        hk, hv = (orc.held(a.float().cpu().numpy()) for a in (dk, dv))
        at = 0
        for slot, pos0, rows in entries:
            if slot >= 0:
                self.k[slot, pos0:pos0 + rows], self.v[slot, pos0:pos0 + rows] = hk[at:at + rows], hv[at:at + rows]
            at += rows

    def read(self, entries, kind="f32", fill=7.0):
        t = self.torch
        dt, typ = _kind(t, self.moe, kind)
        b = self.batch(entries)
        k, v = (t.full((b.n_tok, self.kv, self.hd), fill, dtype=dt, device="cuda") for _ in "kv")
        row = self.kv * self.hd
        self.s.read_dev(self.layer, b, typ, k.data_ptr(), row, v.data_ptr(), row)
        t.cuda.synchronize()
        return k.float().cpu().numpy(), v.float().cpu().numpy()

    def attend(self, entries, q, kind="f32", scale=None, n_sel=None, stream=0):
        """numpy out (rows, heads, hd) (and blocks), with every input rounded to the kind first"""
        t = self.torch
        dt, typ = _kind(t, self.moe, kind)
        dq = t.from_numpy(np.ascontiguousarray(q)).to("cuda").to(dt)
        out = t.full_like(dq, 99.0)
        row, b = self.heads * self.hd, self.batch(entries)
        scale = self.hd ** -0.5 if scale is None else scale
        if n_sel is None:
            self.s.attend_dev(self.layer, b, typ, dq.data_ptr(), row, scale, out.data_ptr(), row, stream=stream)
            t.cuda.synchronize()
            return out.float().cpu().numpy()
        blocks = t.full((b.n_tok, self.kv, n_sel), -7, dtype=t.int32, device="cuda")
        self.s.select_dev(self.layer, b, typ, dq.data_ptr(), row, scale, n_sel, out.data_ptr(), row,
                          blocks_ptr=blocks.data_ptr(), stream=stream)
        t.cuda.synchronize()
        return out.float().cpu().numpy(), blocks.cpu().numpy()

    def check_attend(self, entries, q, kind="f32", scale=None, n_sel=None):
        t = self.torch
        q = t.from_numpy(np.ascontiguousarray(q)).to(_kind(t, self.moe, kind)[0]).float().numpy()
        scale = self.hd ** -0.5 if scale is None else scale
        got = self.attend(entries, q, kind, scale, n_sel)
        got, blocks = got if n_sel else (got, None)
        row = 0
        for slot, pos0, rows in entries:
            for j in range(rows):
                pos = pos0 + j
                if slot < 0:
                    assert (got[row] == 99.0).all() and (blocks is None or (blocks[row] == -7).all())
                    row += 1
                    continue
                k, v = self.k[slot, :pos + 1], self.v[slot, :pos + 1]
                seen = None
                if n_sel:
                    want = orc.selected(self.k[slot], q[row], pos, n_sel)
                    assert np.array_equal(blocks[row], want), (slot, pos, blocks[row], want)
                    seen = np.zeros((self.kv, (pos // 64 + 1) * 64), bool)
                    for h in range(self.kv):
                        for b in want[h][want[h] >= 0]:
                            seen[h, b * 64:b * 64 + 64] = True
                    seen = seen[:, :pos + 1]
                want, size = orc.attention(q[row], k, v, scale, seen)
                tol = orc.tolerance(size, v, want, kind)
                off, nan = abs(got[row] - want), np.isnan(want) & np.isnan(got[row])
                assert ((off <= tol) | nan).all(), (slot, pos, float(np.nanmax(off / tol)))
                row += 1

    def close(self):
        self.s.close()


def _rows(rng, n, kv, hd):
    k = rng.normal(size=(n, kv, hd)) * np.exp(0.5 * rng.normal(size=(kv, hd))) + 3 * rng.normal(size=(kv, hd))
    return k.astype(np.float32), rng.normal(size=(n, kv, hd)).astype(np.float32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", (64, 128))
def test_write_and_read_back_bit_for_bit(cuda, kind, hd):
    """ragged entries at odd starts, several heads, a padding entry; positions around them as they were"""
    rng = np.random.default_rng(1)
    s = Session(cuda, n_seq=4, heads=6, kv=3, hd=hd, ctx=517, n_layers=3, layer=1)
    entries = [(2, 5, 1), (0, 61, 130), (-1, 3, 4), (3, 516, 1), (1, 0, 517)]
    k, v = _rows(rng, sum(e[2] for e in entries), 3, hd)
    s.write(entries, k, v, kind)
    s.write([(0, 64, 3), (2, 127, 2)], *_rows(rng, 5, 3, hd), kind)  # over written rows, and behind the sequence
    gk, gv = s.read([(i, 0, 517) for i in range(4)])
    assert np.array_equal(gk, s.k.reshape(gk.shape)) and np.array_equal(gv, s.v.reshape(gv.shape))
    gk, gv = s.read([(1, 3, 2), (-1, 0, 2), (0, 63, 2)], kind)
    for got, held in ((gk, s.k), (gv, s.v)):
        t = cuda.from_numpy(np.concatenate([held[1, 3:5], np.full((2, 3, hd), 7.0, np.float32), held[0, 63:65]]))
        assert np.array_equal(got, t.to(_kind(cuda, s.moe, kind)[0]).float().numpy())
    s.s.check()
    s.s.write_dev(0, s.batch([(0, 0, 0)]), s.moe.F32, 256, 3 * hd, 256, 3 * hd)  # no rows: nothing is read
    for layer in (0, 2):  # the layers beside it hold nothing
        s.layer = layer
        assert not any(a.any() for a in s.read([(i, 0, 517) for i in range(4)]))
    s.close()


def test_quantiser_borders(cuda):
    """groups whose quotients are ties, constants, subnormals, f16's limits, infinities and NaN"""
    rng = np.random.default_rng(2)
    rows = []
    for i in range(400):  # exact ties and near ties: m + (c + 1/2) d, and one unit of the last place beside it
        d, m = np.float32(np.float16(rng.uniform(0.01, 3))), np.float32(np.float16(rng.normal()))
        c = rng.integers(0, 15, size=32)
        x = (m + (c + 0.5) * d).astype(np.float32)
        x[0], x[1] = m, m + 15 * d
        x[2:12] = np.nextafter(x[2:12], np.float32(np.inf) if i % 2 else np.float32(-np.inf))
        rows.append(x)
    for i in range(100):
        rows.append((rng.normal(size=32) * 10.0 ** rng.uniform(-9, 4)).astype(np.float32))
        rows.append(np.full(32, rng.normal() * 10.0 ** rng.uniform(-9, 4), np.float32))
        rows.append((rng.normal() * 100 + rng.normal(size=32) * 1e-4).astype(np.float32))  # m rounds by more than d
    special = [np.zeros(32), np.full(32, -0.0), np.full(32, 65519.0), np.full(32, 65520.0), np.full(32, -65520.0),
               np.full(32, 1e30), np.linspace(-65504, 65504, 32), np.linspace(0, 65504 * 15, 32),
               np.linspace(0, 65520 * 15, 32), np.linspace(0, 15 * 2.0 ** -25, 32), np.linspace(0, 15 * 2.1 ** -25, 32),
               np.linspace(0, 2.0 ** -20, 32), np.full(32, 1e-40), np.full(32, 3.0e-8), np.full(32, 2.9e-8)]
    for bad in (np.inf, -np.inf, np.nan):
        x = rng.normal(size=32)
        x[rng.integers(0, 32)] = bad
        special.append(x)
    rows += [np.asarray(x, np.float32) for x in special]
    while len(rows) % 4:
        rows.append(np.zeros(32, np.float32))
    x = np.stack(rows).reshape(-1, 1, 128)
    s = Session(cuda, 1, 1, 1, 128, x.shape[0])
    s.write([(0, 0, x.shape[0])], x, x[::-1])
    gk, gv = s.read([(0, 0, x.shape[0])])
    assert np.array_equal(gk, orc.held(x), equal_nan=True)
    assert np.array_equal(gv, orc.held(x[::-1]), equal_nan=True)
    s.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd", ((16, 16, 128), (8, 2, 128), (14, 2, 64), (16, 1, 64), (40, 2, 128), (3, 1, 128), (256, 1, 64)))
def test_decode_attention(cuda, kind, heads, kv, hd):
    """one row a sequence, lengths from one position on, in one call"""
    rng = np.random.default_rng(3)
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 127, 129, 300, 1000, 1025]
    n = len(lengths)
    s = Session(cuda, n, heads, kv, hd, 1030)
    k, v = _rows(rng, n * 1030, kv, hd)
    s.write([(i, 0, 1030) for i in range(n)], k, v, kind)  # later positions hold other rows: masked
    entries = [(n - 1 - i, lengths[i] - 1, 1) for i in range(n)] + [(-1, 0, 1), (4, 700, 1)]  # a sequence twice
    s.check_attend(entries, 2 * rng.normal(size=(len(entries), heads, hd)).astype(np.float32), kind)
    s.check_attend(entries[:1], rng.normal(size=(1, heads, hd)).astype(np.float32), kind, scale=0.7)
    s.s.check()
    s.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd", ((2, 2, 128), (8, 2, 64), (7, 1, 128)))
def test_attention_of_several_rows(cuda, kind, heads, kv, hd):
    """prompts and drafted tokens: each row up to its own position; entries without rows and padding between"""
    rng = np.random.default_rng(4)
    s = Session(cuda, 5, heads, kv, hd, 400)
    s.write([(i, 0, 400) for i in range(5)], *_rows(rng, 2000, kv, hd), kind)
    entries = [(0, 0, 130), (1, 61, 7), (2, 5, 0), (-1, 0, 3), (3, 399, 1), (4, 190, 129), (2, 0, 1)]
    s.check_attend(entries, 2 * rng.normal(size=(sum(e[2] for e in entries), heads, hd)).astype(np.float32), kind)
    s.close()


@pytest.mark.parametrize("kind", ("bf16", "f16"))
@pytest.mark.parametrize("heads,kv,hd", ((4, 2, 128), (5, 1, 64), (14, 2, 128), (3, 3, 64)))
def test_attention_of_prompts(cuda, kind, heads, kv, hd):
    """more query rows than a CTA holds; tiles that end inside a token's heads, inside a record and inside a block; one
    entry whose rows fit one tile; a prompt that starts far into its sequence"""
    rng = np.random.default_rng(14)
    s = Session(cuda, 4, heads, kv, hd, 900)
    s.write([(i, 0, 900) for i in range(4)], *_rows(rng, 3600, kv, hd), kind)
    entries = [(2, 0, 331), (0, 517, 383), (1, 200, 9), (3, 131, 128), (-1, 0, 5)]
    s.check_attend(entries, 2 * rng.normal(size=(sum(e[2] for e in entries), heads, hd)).astype(np.float32), kind)
    s.check_attend([(1, 0, 200)], rng.normal(size=(200, heads, hd)).astype(np.float32), kind, scale=-0.3)
    s.s.check()
    s.close()


def test_prompt_of_values_past_16_bits(cuda):
    """keys and values that a cache of bf16 rows holds but f16 does not, in one head and in some rows' future"""
    rng = np.random.default_rng(15)
    s = Session(cuda, 2, 4, 2, 128, 400)
    k, v = _rows(rng, 800, 2, 128)
    k[130, 0, :40] *= 2e5  # (the lowest pass f16: this one is held as NaN)
    v[90, 1, 7] = 8e5
    k[700, 1, 5], v[420, 0, 100] = 3e5, 1e5
    s.write([(0, 0, 400), (1, 0, 400)], k, v, "bf16")
    q = rng.normal(size=(800, 4, 128)).astype(np.float32)
    s.check_attend([(0, 0, 400), (1, 0, 400)], q, "bf16")
    s.check_attend([(0, 0, 400)], 1e-6 * q[:400], "bf16")
    s.close()


@pytest.mark.parametrize("kind", KINDS)
def test_nan_and_infinity(cuda, kind):
    """a NaN in a position that a row does not see does not reach it; in one that it sees it does; neither does one
    cross heads, and a score of minus infinity's size leaves the others"""
    rng = np.random.default_rng(5)
    s = Session(cuda, 2, 4, 2, 128, 300)
    k, v = _rows(rng, 600, 2, 128)
    k[100, 0, 3], v[150, 1, 70], k[299, 1, 5], v[20 + 300, 0, 1] = np.nan, np.inf, -np.inf, np.nan
    s.write([(0, 0, 300), (1, 0, 300)], k, v, kind)
    q = rng.normal(size=(300, 4, 128)).astype(np.float32)
    got = s.attend([(0, 0, 300)], q, kind)
    assert np.isfinite(got[:100]).all() and np.isfinite(got[:150, 2:]).all() and np.isfinite(got[150:299, 2:, :64]).all()
    assert np.isnan(got[100:, :2]).all() and np.isnan(got[150:, 2:, 64:96]).all() and np.isnan(got[299, 2:]).all()
    s.k[0, 100:], s.v[0, 100:] = 0, 0
    s.check_attend([(0, 0, 100)], q[:100], kind)
    got = s.attend([(1, 19, 1), (1, 20, 1)], q[:2], kind)
    assert np.isfinite(got[0]).all() and np.isnan(got[1, :2, :32]).all() and np.isfinite(got[1, :2, 32:]).all()
    q[3, 2, 7], q[4, 0, 0] = np.nan, np.inf
    got = s.attend([(1, 0, 1)] * 5, q[:5], kind)
    assert np.isnan(got[3, 2]).all() and np.isfinite(got[3, [0, 1, 3]]).all() and np.isfinite(got[:3]).all()
    s.close()


@pytest.mark.parametrize("kind", KINDS)
def test_scales_and_query_sizes(cuda, kind):
    """a scale of 0, negative ones, queries that are zero, tiny and large"""
    rng = np.random.default_rng(18)
    s = Session(cuda, 1, 4, 2, 64, 500)
    s.write([(0, 0, 500)], *_rows(rng, 500, 2, 64), kind)
    q = rng.normal(size=(5, 4, 64)).astype(np.float32)
    q[1] = 0
    q[2] *= 1e-7 if kind == "f16" else 1e-30
    q[3] *= 50
    for scale in (0.0, -0.2, 0.05, 1e-6, 3.0):
        s.check_attend([(0, 499, 1), (0, 100, 1), (0, 3, 1), (0, 64, 1), (0, 0, 1)], q, kind, scale=scale)
        s.check_attend([(0, 430, 5)], q, kind, scale=scale, n_sel=3)
    s.close()


def test_large_scores_and_a_far_sink(cuda):
    """scores hundreds apart; one position with nearly all the weight and tiny values beside a thousand others"""
    rng = np.random.default_rng(6)
    s = Session(cuda, 1, 2, 2, 128, 2000)
    k, v = _rows(rng, 2000, 2, 128)
    k[0] = 0.4 * np.sign(k[1])
    v[0] *= 1e-3
    s.write([(0, 0, 2000)], k, v)
    q = np.stack([40 * k[7], 9 * np.sign(k[1]), 1e-4 * k[3], -30 * k[1999], 0 * k[0]]).astype(np.float32)
    s.check_attend([(0, 1999, 1)] * 5, q)
    s.check_attend([(0, 1234, 1)] * 5, q)
    s.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd", ((4, 4, 128), (8, 2, 64), (7, 1, 128), (40, 2, 64)))
def test_selection(cuda, kind, heads, kv, hd):
    """the blocks equal the definition's, the output attention over them; fewer blocks than asked for; ties"""
    rng = np.random.default_rng(7)
    s = Session(cuda, 3, heads, kv, hd, 2300)
    for i in range(3):
        k, v = _rows(rng, 2300, kv, hd)
        if i == 1:
            k[640:960] = np.tile(k[640:704], (5, 1, 1))  # five equal blocks: the lowest are taken
        if i == 2:
            k[:] = k[0]  # all equal
        s.write([(i, 0, 2300)], k, v, kind)
    entries = [(0, 2299, 1), (1, 2200, 1), (2, 1999, 1), (0, 63, 1), (1, 64, 1), (2, 700, 1), (-1, 5, 1), (0, 0, 1),
               (1, 1024, 1), (0, 1400, 3)]
    q = rng.normal(size=(12, heads, hd)).astype(np.float32)
    q[5] = 0
    for n_sel in (1, 2, 6, 12, 40):
        s.check_attend(entries, q, kind, n_sel=n_sel)
    s.s.check()
    s.close()


def test_selection_follows_what_is_written(cuda):
    """a sequence that is cut back and written on, a row overwritten inside a whole block, a NaN among the keys"""
    rng = np.random.default_rng(8)
    s = Session(cuda, 1, 4, 2, 128, 1200)
    s.write([(0, 0, 1200)], *_rows(rng, 1200, 2, 128))
    q = rng.normal(size=(2, 4, 128)).astype(np.float32)
    at = [(0, 1190, 1), (0, 1199, 1)]
    s.check_attend(at, q, n_sel=4)
    k, v = _rows(rng, 700, 2, 128)
    s.write([(0, 333, 1)], 9 * k[:1], v[:1])
    s.check_attend(at, q, n_sel=4)
    s.write([(0, 500, 400)], 2 * k[:400], v[:400])
    s.check_attend(at, q, n_sel=4)
    for p in range(900, 1000):  # a token at a time
        s.write([(0, p, 1)], 0.1 * k[p - 400:p - 399], v[p - 400:p - 399])
    s.check_attend([(0, 999, 1)] * 2, q, n_sel=5)
    k[0, 1, 9] = np.nan
    s.write([(0, 70, 1)], k[:1], v[:1])
    got, blocks = s.attend(at, q, n_sel=2)
    assert (blocks[:, 1, 0] == 1).all() and np.isnan(got[:, 2:]).all() and np.isfinite(got[:, :2]).all()
    q[0, 0, 3] = np.inf  # a query that cannot be scored selects by index; its head is NaN
    got, blocks = s.attend(at, q, n_sel=3)
    assert blocks[0, 0].tolist() == [0, 1, 18] and np.isnan(got[0, 0]).all() and np.isfinite(got[0, 1]).all()
    s.close()


def test_rows_that_belong_to_no_entry_stay(cuda):
    """rows before the first start and behind the last, and strides wider than a row"""
    torch = cuda
    rng = np.random.default_rng(9)
    s = Session(torch, 2, 4, 2, 64, 100)
    s.write([(0, 0, 100), (1, 0, 100)], *_rows(rng, 200, 2, 64))
    qkv = torch.from_numpy(rng.normal(size=(9, 4 * 64 + 2 * 2 * 64)).astype(np.float32)).to("cuda")
    before = qkv.clone()
    b = s.batch([(1, 40, 3), (0, 50, 2)], n_tok=9, max_rows=3, starts=[2, 5, 7])
    row = qkv.shape[1]
    s.s.write_dev(0, b, s.moe.F32, qkv.data_ptr() + 4 * 256, row, qkv.data_ptr() + 4 * 384, row)
    for slot, p, r in ((1, 40, slice(2, 5)), (0, 50, slice(5, 7))):
        for t, c in ((s.k, 256), (s.v, 384)):
            t[slot, p:p + r.stop - r.start] = orc.held(before[r, c:c + 128].reshape(-1, 2, 64).cpu().numpy())
    gk, gv = s.read([(0, 0, 100), (1, 0, 100)])
    assert np.array_equal(gk, s.k.reshape(gk.shape)) and np.array_equal(gv, s.v.reshape(gv.shape))
    out = torch.full((9, 300), 5.0, device="cuda")
    s.s.attend_dev(0, b, s.moe.F32, qkv.data_ptr(), row, 0.125, out.data_ptr(), 300)
    blocks = torch.full((9, 2, 3), -9, dtype=torch.int32, device="cuda")
    out2 = torch.full((9, 300), 5.0, device="cuda")
    s.s.select_dev(0, b, s.moe.F32, qkv.data_ptr(), row, 0.125, 3, out2.data_ptr(), 300, blocks_ptr=blocks.data_ptr())
    torch.cuda.synchronize()
    for o in (out, out2):
        o = o.cpu().numpy()
        assert (o[:2] == 5).all() and (o[7:] == 5).all() and (o[:, 256:] == 5).all()
        for r, (slot, p) in zip(range(2, 7), ((1, 40), (1, 41), (1, 42), (0, 50), (0, 51))):
            q = before[r, :256].reshape(4, 64).cpu().numpy()
            want, size = orc.attention(q, s.k[slot, :p + 1], s.v[slot, :p + 1], 0.125)
            assert (abs(o[r, :256].reshape(4, 64) - want) <= orc.tolerance(size, s.v[slot, :p + 1], want, "f32")).all()
    blocks = blocks.cpu().numpy()
    assert (blocks[:2] == -9).all() and (blocks[7:] == -9).all() and (blocks[2:7] == [0, -1, -1]).all()
    assert torch.equal(qkv, before)
    s.close()


def test_refused_calls_and_entries(cuda):
    torch = cuda
    rng = np.random.default_rng(10)
    s = Session(torch, 2, 4, 2, 64, 100, n_layers=2)
    s.write([(0, 0, 100), (1, 0, 100)], *_rows(rng, 200, 2, 64))
    buf = torch.zeros(4096, device="cuda")
    p, moe, L = buf.data_ptr(), s.moe, s.moe.lib()
    good = s.batch([(0, 0, 1), (1, 0, 1)])
    calls = (lambda layer, b, t, x, sx, y, sy: L.tr_gpu_attn4_write_dev(s.s.a, layer, b, t, x, sx, y, sy, None),
             lambda layer, b, t, x, sx, y, sy: L.tr_gpu_attn4_read_dev(s.s.a, layer, b, t, x, sx, y, sy, None),
             lambda layer, b, t, x, sx, y, sy: L.tr_gpu_attn4_attend_dev(s.s.a, layer, b, t, x, sx, 1.0, y, sy, None),
             lambda layer, b, t, x, sx, y, sy: L.tr_gpu_attn4_select_dev(s.s.a, layer, b, t, x, sx, 1.0, 2, y, sy, None,
                                                                         None))
    B = moe.Attn4Batch
    n, sl, po, st = good.n_entries, good.slot, good.pos0, good.start
    for f in calls:
        for args in ((2, good, moe.F32, p, 256, p, 256), (-1, good, moe.F32, p, 256, p, 256),
                     (0, good, moe.Q8_0, p, 256, p, 256), (0, good, moe.F32, None, 256, p, 256),
                     (0, good, moe.F32, p, 256, None, 256), (0, good, moe.F32, p + 4, 256, p, 256),
                     (0, good, moe.F32, p, 256, p + 8, 256), (0, good, moe.F32, p, 127, p, 256),
                     (0, good, moe.F32, p, 256, p, 64), (0, good, moe.F32, p, 258, p, 256),
                     (0, good, moe.BF16, p, 260, p, 256), (0, good, moe.F32, p, -256, p, 256),
                     (0, B(-1, 2, 1, sl, po, st), moe.F32, p, 256, p, 256),
                     (0, B(65536, 2, 1, sl, po, st), moe.F32, p, 256, p, 256),
                     (0, B(n, 1 << 31, 1, sl, po, st), moe.F32, p, 256, p, 256),
                     (0, B(n, 3, 1, sl, po, None), moe.F32, p, 256, p, 256),
                     (0, B(n, 2, 0, sl, po, st), moe.F32, p, 256, p, 256),
                     (0, B(n, 2, 101, sl, po, st), moe.F32, p, 256, p, 256),
                     (0, B(n, 2, 1, None, po, st), moe.F32, p, 256, p, 256),
                     (0, B(n, 2, 1, sl + 2, po, st), moe.F32, p, 256, p, 256)):
            assert f(*args) == -1 and moe.last_error(), args
        assert f(0, B(0, 0, 1, None, None, None), moe.F32, p, 256, p, 256) == 0
    for bad in (0, 4097):
        assert L.tr_gpu_attn4_select_dev(s.s.a, 0, good, moe.F32, p, 256, 1.0, bad, p, 256, None, None) == -1
    s.s.check()  # none of these reached the device
    # entries that the kernels leave out: outside the sequences, the positions, the rows, or of more than max_rows
    q = rng.normal(size=(8, 4, 64)).astype(np.float32)
    for entries, kw in (([(2, 0, 1), (1, 9, 2)], {}), ([(1, 99, 2), (0, 1, 1)], {}), ([(1, -1, 1), (0, 1, 1)], {}),
                        ([(1, 5, 3), (0, 1, 1)], {"max_rows": 2}), ([(1, 5, 2), (0, 1, 7)], {"n_tok": 8}),
                        ([(1, 5, 3), (0, 1, 0)], {"starts": [1, 4, 2]})):
        b = s.batch(entries, **({"n_tok": 8} | kw))
        dq = torch.from_numpy(q).to("cuda")
        out = torch.full_like(dq, 99.0)
        s.s.attend_dev(0, b, moe.F32, dq.data_ptr(), 256, 0.1, out.data_ptr(), 256)
        with pytest.raises(RuntimeError, match="left out"):
            s.s.check()
        s.s.select_dev(0, b, moe.F32, dq.data_ptr(), 256, 0.1, 2, out.data_ptr(), 256)
        with pytest.raises(RuntimeError, match="left out"):
            s.s.check()
        s.s.read_dev(0, b, moe.F32, out.data_ptr(), 256, out.data_ptr() + 512, 256)
        with pytest.raises(RuntimeError, match="left out"):
            s.s.check()
    ones = torch.ones((3, 2, 64), device="cuda")
    s.s.write_dev(0, s.batch([(1, 3, 1), (0, 7, 1), (1, 60, 1)]), moe.F32, ones.data_ptr(), 128, ones.data_ptr(), 128)
    with pytest.raises(RuntimeError, match="one sequence"):
        s.s.check()
    s.k[1, 3], s.v[1, 3], s.k[0, 7], s.v[0, 7] = 1, 1, 1, 1  # the first of the two was written
    gk, gv = s.read([(0, 0, 100), (1, 0, 100)])
    assert np.array_equal(gk, s.k.reshape(gk.shape)) and np.array_equal(gv, s.v.reshape(gv.shape))
    s.s.check()
    with pytest.raises(RuntimeError, match="outside the cache"):
        s.s.write(0, 0, 99, np.zeros((2, 128)), np.zeros((2, 128)))
    with pytest.raises(RuntimeError, match="outside the cache"):
        s.s.decode(0, 0, 100, np.zeros(256), np.zeros(128), np.zeros(128), 1.0)
    with pytest.raises(RuntimeError, match="outside the cache"):
        s.s.decode(0, 2, 0, np.zeros(256), np.zeros(128), np.zeros(128), 1.0)
    s.close()


def test_captured_and_replayed(cuda):
    """a decode step (write, attend, select) in a CUDA graph, replayed as the positions move on; another session's calls
    on another stream meanwhile"""
    torch = cuda
    rng = np.random.default_rng(11)
    s, o = (Session(torch, 3, 8, 2, 128, 700) for _ in range(2))
    for x in (s, o):
        x.write([(i, 0, 640) for i in range(3)], *_rows(rng, 3 * 640, 2, 128), "bf16")
    slot = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    pos = torch.tensor([600, 0, 63], dtype=torch.int32, device="cuda")
    k, v = (torch.zeros((3, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in "kv")
    q = torch.zeros((3, 8, 128), dtype=torch.bfloat16, device="cuda")
    out, out2 = torch.zeros_like(q), torch.zeros_like(q)
    blocks = torch.zeros((3, 2, 4), dtype=torch.int32, device="cuda")
    b = s.moe.Attn4Batch(3, 3, 1, slot.data_ptr(), pos.data_ptr(), None)

    def step(stream):
        s.s.write_dev(0, b, s.moe.BF16, k.data_ptr(), 256, v.data_ptr(), 256, stream=stream)
        s.s.attend_dev(0, b, s.moe.BF16, q.data_ptr(), 1024, 0.1, out.data_ptr(), 1024, stream=stream)
        s.s.select_dev(0, b, s.moe.BF16, q.data_ptr(), 1024, 0.1, 4, out2.data_ptr(), 1024,
                       blocks_ptr=blocks.data_ptr(), stream=stream)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    side = torch.cuda.Stream()
    oq = torch.from_numpy(rng.normal(size=(3, 8, 128)).astype(np.float32)).to("cuda")
    oout = torch.zeros_like(oq)
    ob = o.batch([(0, 639, 1), (1, 600, 1), (2, 30, 1)])
    want, first = None, None
    for it in range(30):
        hk, hv = _rows(rng, 3, 2, 128)
        k.copy_(torch.from_numpy(hk))
        v.copy_(torch.from_numpy(hv))
        q.copy_(torch.from_numpy(rng.normal(size=(3, 8, 128)).astype(np.float32)))
        at = [600 + it, it, 63 + it]
        pos.copy_(torch.tensor(at, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            o.s.attend_dev(0, ob, o.moe.F32, oq.data_ptr(), 1024, 0.1, oout.data_ptr(), 1024, stream=side.cuda_stream)
            o.s.select_dev(0, ob, o.moe.F32, oq.data_ptr(), 1024, 0.1, 3, oout.data_ptr(), 1024, stream=side.cuda_stream)
        torch.cuda.synchronize()
        first = oout.clone() if first is None else first
        assert torch.equal(oout, first)
        for i, sl in enumerate((2, 0, 1)):
            s.k[sl, at[i]], s.v[sl, at[i]] = orc.held(k[i].float().cpu().numpy()), orc.held(v[i].float().cpu().numpy())
        if it % 7 == 0:
            for i, sl in enumerate((2, 0, 1)):
                hq, K, V = q[i].float().cpu().numpy(), s.k[sl, :at[i] + 1], s.v[sl, :at[i] + 1]
                want, size = orc.attention(hq, K, V, 0.1)
                assert (abs(out[i].float().cpu().numpy() - want) <= orc.tolerance(size, V, want, "bf16")).all()
                assert np.array_equal(blocks[i].cpu().numpy(), orc.selected(s.k[sl], hq, at[i], 4))
    s.s.check()
    s.close(), o.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd", ((4, 4, 128), (8, 2, 128), (16, 1, 64), (20, 1, 128)))
def test_long_contexts(cuda, kind, heads, kv, hd):
    """many CTAs and warps on one tile of query rows, of which some, most or all but one have a position; drafted tokens;
    the selection's threshold over several CTAs"""
    rng = np.random.default_rng(16)
    ctx = 20001
    s = Session(cuda, 2, heads, kv, hd, ctx)
    s.write([(1, 0, ctx)], *_rows(rng, ctx, kv, hd), kind)
    s.write([(0, 0, 600)], *_rows(rng, 600, kv, hd), kind)
    q = rng.normal(size=(8, heads, hd)).astype(np.float32)
    for entries in ([(1, 20000, 1)], [(1, 16383, 1)], [(1, 300, 1)], [(0, 31, 1)], [(0, 599, 1), (1, 9000, 1)], [(1, 19993, 8)]):
        n = sum(e[2] for e in entries)
        s.check_attend(entries, q[:n], kind)
        s.check_attend(entries, q[:n], kind, n_sel=7)
    s.check_attend([(1, 20000, 1)], q[:1], kind, n_sel=200)
    s.s.check()
    s.close()


def test_f32_sums_over_long_contexts(cuda):
    """f32 rows: the error must not grow with the number of positions. Counted against the outputs' norm, for values of mean 0
    whose sum is as large as their roundings' sums let it be: a probability in two f16 parts and its product with a scale
    2^-21, the exponential 2^-22, a score near 0 of query values in two parts 2^-20, a value's minimum 2^-21, 60 rounded
    additions a warp 2^-24 x 8, its sums' and the joins' 2^-23: below 2^-18.5 together were all at their worst, and they
    are independent, so that a norm over 1024 outputs stays below 2^-19."""
    rng = np.random.default_rng(23)
    ctx = 100_000
    s = Session(cuda, 1, 8, 8, 128, ctx)
    s.write([(0, 0, ctx)], *[rng.normal(size=(ctx, 8, 128)).astype(np.float32) for _ in "kv"])
    q = rng.normal(size=(1, 8, 128)).astype(np.float32)
    got = s.attend([(0, ctx - 1, 1)], q)[0]
    want, _ = orc.attention(q[0], s.k[0], s.v[0], 128 ** -0.5, None)
    assert np.linalg.norm(got - want) < 2 ** -19 * np.linalg.norm(want)
    s.s.check()
    s.close()


def test_overlapping_calls(cuda):
    """one session's calls on two streams at once, eager and as two captured graphs: each gives what it gives alone"""
    torch = cuda
    rng = np.random.default_rng(17)
    s = Session(torch, 4, 8, 2, 128, 3000)
    s.write([(i, 0, 3000) for i in range(4)], *_rows(rng, 12000, 2, 128), "f16")
    jobs = []
    for entries in ([(0, 2999, 1), (1, 700, 1)], [(2, 2000, 1), (3, 64, 1), (0, 2998, 1)]):
        b = s.batch(entries)
        q = torch.from_numpy(rng.normal(size=(len(entries), 8, 128)).astype(np.float32)).to("cuda").half()
        jobs.append((b, q, torch.zeros_like(q), torch.zeros_like(q), torch.cuda.Stream()))

    def run(job, stream):
        b, q, out, picked, _ = job
        for _ in range(4):
            s.s.attend_dev(0, b, s.moe.F16, q.data_ptr(), 1024, 0.1, out.data_ptr(), 1024, stream=stream)
            s.s.select_dev(0, b, s.moe.F16, q.data_ptr(), 1024, 0.1, 5, picked.data_ptr(), 1024, stream=stream)

    alone = []
    for job in jobs:
        run(job, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        alone.append((job[2].clone(), job[3].clone()))
    graphs = []
    for job in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(job, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for it in range(20):
        for job in jobs:
            job[2].zero_(), job[3].zero_()
        torch.cuda.synchronize()
        for job, g in zip(jobs, graphs):
            with torch.cuda.stream(job[4]):
                if it % 2:
                    g.replay()
                else:
                    run(job, job[4].cuda_stream)
        torch.cuda.synchronize()
        for job, (out, picked) in zip(jobs, alone):
            assert torch.equal(job[2], out) and torch.equal(job[3], picked)
    s.s.check()
    s.close()


def test_far_offsets(cuda):
    """a cache past 4 GB: the last sequence's last positions, with another sequence's left alone"""
    torch = cuda
    rng = np.random.default_rng(12)
    ctx, n = 1 << 19, 9  # 9 sequences x 8 heads x 2^19 positions x 160 bytes: 6 GB
    s = Session.__new__(Session)
    from trochilus_b200 import moe
    s.torch, s.moe, s.layer, s.heads, s.kv, s.hd, s.ctx, s.keep = torch, moe, 0, 8, 8, 128, ctx, []
    s.s = moe.GpuAttn4(1, n, 8, 8, 128, ctx)
    k, v = _rows(rng, 200, 8, 128)
    dk, dv = (torch.from_numpy(a).to("cuda") for a in (k, v))
    s.s.write_dev(0, s.batch([(n - 1, ctx - 200, 200)]), moe.F32, dk.data_ptr(), 1024, dv.data_ptr(), 1024)
    gk, gv = s.read([(n - 1, ctx - 200, 200), (0, ctx - 200, 200), (n - 2, ctx - 200, 200)])
    assert np.array_equal(gk[:200], orc.held(k)) and np.array_equal(gv[:200], orc.held(v))
    assert not gk[200:].any() and not gv[200:].any()
    # the other positions are zeros: their score is 0, their value 0
    q = rng.normal(size=(1, 8, 128)).astype(np.float32)
    got = s.attend([(n - 1, ctx - 1, 1)], q)[0]
    sc = np.einsum("hd,thd->ht", q[0].astype(np.float64), orc.held(k).astype(np.float64)) * 128 ** -0.5
    top = np.maximum(sc.max(-1), 0)
    w = np.exp(sc - top[:, None])
    want = np.einsum("ht,thd->hd", w, orc.held(v).astype(np.float64))
    want /= (w.sum(-1) + (ctx - 200) * np.exp(-top))[:, None]
    size = float(np.einsum("hd,thd->ht", abs(q[0]), abs(orc.held(k))).max()) * 128 ** -0.5
    assert (abs(got - want) <= orc.tolerance(size, v, want, "f32")).all()
    got, blocks = s.attend([(n - 1, ctx - 1, 1)], q, n_sel=5)
    full = np.zeros((ctx, 8, 128), np.float32)
    full[-200:] = orc.held(k)
    assert np.array_equal(blocks[0], orc.selected(full, q[0], ctx - 1, 5))
    s.close()


def test_host_rows_beside_the_f32_session(cuda):
    """the engine's calls (tr_gpu_attn_write, _decode) and their 4-bit forms on the same prompt and tokens: the 4-bit
    session's output is the oracle's on what it holds, and reads what the device calls read"""
    from trochilus_b200.moe import GpuAttn, GpuAttn4
    rng = np.random.default_rng(13)
    heads, ctx, P = 4, 700, 600  # (more than one chunk of a host write)
    a, f = GpuAttn4(2, 2, heads, heads, 128, ctx), GpuAttn(2, heads, ctx)
    scale = np.float32(128 ** -0.5)
    for layer in range(2):
        k, v = (rng.normal(size=(ctx, heads, 128)).astype(np.float32) for _ in range(2))
        a.write(layer, 1, 0, k[:P], v[:P])
        f.write(layer, 0, orc.held(k)[:P], orc.held(v)[:P])
        for pos in range(P, P + 5):
            q = rng.normal(size=(heads, 128)).astype(np.float32)
            got = a.decode(layer, 1, pos, q, k[pos], v[pos], scale)
            hk, hv = orc.held(k[:pos + 1]), orc.held(v[:pos + 1])
            want, size = orc.attention(q, hk, hv, scale)
            tol = orc.tolerance(size, hv, want, "f32")
            assert (abs(got - want) <= tol).all()
            assert (abs(got - f.decode(layer, pos, q, hk[pos], hv[pos], scale)) <= 2 * tol).all()
    a.check()
    a.close(), f.close()
