"""Calls of the 4-bit KV cache that serving makes and that the other files leave out: many entries, caches of one position,
prompts between other columns and rows, prompts captured and beside each other."""
import numpy as np
import pytest

from tests import attn4_bounds as bnd
from tests import attn4_oracle as orc
from tests.test_gpu_attention4 import KINDS, Session, _kind, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
def test_many_entries(cuda, kind):
    """more entries than a CTA has threads: written at once, read, attended to and selected from; padding among them"""
    rng = np.random.default_rng(71)
    n, ctx = 700, 200
    s = Session(cuda, n, 4, 2, 64, ctx)
    lengths = rng.integers(1, ctx + 1, size=n)
    order = rng.permutation(n)
    s.write([(int(i), 0, int(lengths[i])) for i in order], *_rows(rng, int(lengths.sum()), 2, 64), kind)
    gk, gv = s.read([(i, 0, ctx) for i in range(n)])
    assert np.array_equal(gk, s.k.reshape(gk.shape)) and np.array_equal(gv, s.v.reshape(gv.shape))
    entries = [(int(i) if i % 9 else -1, int(lengths[i]) - 1, 1) for i in order]
    q = bnd.held_in(cuda, kind, rng.normal(size=(n, 4, 64)))
    got, (picked, blocks) = s.attend(entries, q, kind), s.attend(entries, q, kind, n_sel=2)
    for row, (slot, pos, _) in enumerate(entries):
        if slot < 0:
            assert (got[row] == 99).all() and (picked[row] == 99).all() and (blocks[row] == -7).all()
            continue
        k, v = s.k[slot, :pos + 1], s.v[slot, :pos + 1]
        want, tol = bnd.attention(q[row], k, v, 64 ** -0.5, kind)
        assert bnd.far(got[row], want, tol) <= 1, (slot, pos)
        assert np.array_equal(blocks[row], orc.selected(s.k[slot], q[row], pos, 2))
        want, tol = bnd.attention(q[row], k, v, 64 ** -0.5, kind, False, bnd.seen_of(blocks[row], pos))
        assert bnd.far(picked[row], want, tol) <= 1, (slot, pos)
    s.s.check()
    k, v = _rows(rng, n + 1, 2, 64)
    dt, typ = _kind(cuda, s.moe, kind)
    dk, dv = (cuda.from_numpy(x).to("cuda").to(dt) for x in (k, v))
    again = [(int(i), 0, 1) for i in order] + [(int(order[3]), 1, 1)]  # the last names an earlier entry's sequence
    s.s.write_dev(0, s.batch(again), typ, dk.data_ptr(), 128, dv.data_ptr(), 128)
    with pytest.raises(RuntimeError, match="one sequence"):
        s.s.check()
    s.k[order, 0], s.v[order, 0] = (orc.held(x.float().cpu().numpy())[:n] for x in (dk, dv))
    gk, gv = s.read([(i, 0, ctx) for i in range(n)])
    assert np.array_equal(gk, s.k.reshape(gk.shape)) and np.array_equal(gv, s.v.reshape(gv.shape))
    s.close()


@pytest.mark.parametrize("ctx", (1, 2, 33, 65))
def test_small_caches(cuda, ctx):
    rng = np.random.default_rng(72)
    for kind in KINDS:
        s = Session(cuda, 2, 6, 2, 128, ctx)
        s.write([(1, 0, ctx), (0, ctx - 1, 1)], *_rows(rng, ctx + 1, 2, 128), kind)
        gk, gv = s.read([(0, 0, ctx), (1, 0, ctx)])
        assert np.array_equal(gk, s.k.reshape(gk.shape)) and np.array_equal(gv, s.v.reshape(gv.shape))
        q = bnd.held_in(cuda, kind, rng.normal(size=(ctx + 1, 6, 128)))
        entries = [(1, 0, ctx), (0, ctx - 1, 1)]
        for n_sel in (None, 1, 3):
            got = s.attend(entries, q, kind, n_sel=n_sel)
            got, blocks = got if n_sel else (got, None)
            for row in range(ctx + 1):
                slot, pos = (1, row) if row < ctx else (0, ctx - 1)
                seen = bnd.seen_of(blocks[row], pos) if n_sel else None
                want, tol = bnd.attention(q[row], s.k[slot, :pos + 1], s.v[slot, :pos + 1], 128 ** -0.5, kind, False, seen)
                assert bnd.far(got[row], want, tol) <= 1, (slot, pos)
        s.s.check()
        s.close()


def _prompt_job(cuda, rng, s, kind, entries, lead, behind, wide):
    """(batch, packed rows, outputs with a border, call) of a prompt whose rows lie between others"""
    dt, typ = _kind(cuda, s.moe, kind)
    starts = np.cumsum([lead] + [e[2] for e in entries])
    n = int(starts[-1]) + behind
    row = s.heads * s.hd
    packed = cuda.from_numpy(rng.normal(size=(n, row + wide)).astype(np.float32)).to("cuda").to(dt)
    out = cuda.full((n, row + 64), 5.0, dtype=dt, device="cuda")
    b = s.batch(entries, n_tok=n, starts=[int(x) for x in starts])
    es = packed.element_size()

    def call(stream):
        s.s.attend_dev(0, b, typ, packed.data_ptr() + wide * es, row + wide, s.hd ** -0.5, out.data_ptr() + 16 * es, row + 64,
                       stream=stream)
    return packed, out, call


@pytest.mark.parametrize("kind", ("bf16", "f16"))
def test_prompts_between_other_rows_and_columns(cuda, kind):
    """queries inside packed rows, outputs inside wider ones: what lies around them stays; eager, captured and replayed, and
    two prompts of one session on two streams at once"""
    torch = cuda
    rng = np.random.default_rng(73)
    s = Session(torch, 3, 32, 4, 128, 300)
    s.write([(i, 0, 300) for i in range(3)], *_rows(rng, 900, 4, 128), kind)
    jobs = []
    for entries in ([(2, 0, 290), (0, 17, 200)], [(1, 5, 295), (2, 299, 1), (0, 0, 3)]):
        assert bnd.takes_prompt_kernel(torch, len(entries), 295 if entries[0][2] == 295 else 290, 32, 4)
        jobs.append((entries, *_prompt_job(torch, rng, s, kind, entries, 3, 2, 256)))
    alone = []
    for entries, packed, out, call in jobs:
        before = packed.clone()
        call(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        got, row = out.float().cpu().numpy(), 3
        assert torch.equal(packed, before)
        assert (got[:3] == 5).all() and (got[-2:] == 5).all() and (got[:, :16] == 5).all() and (got[:, 16 + 4096:] == 5).all()
        q = packed.float().cpu().numpy()[:, 256:].reshape(-1, 32, 128)
        for slot, pos0, rows in entries:
            for pos in range(pos0, pos0 + rows):
                if pos % 7 == 0 or pos == pos0 + rows - 1:
                    want, tol = bnd.attention(q[row], s.k[slot, :pos + 1], s.v[slot, :pos + 1], 128 ** -0.5, kind, True)
                    assert bnd.far(got[row, 16:16 + 4096].reshape(32, 128), want, tol) <= 1, (slot, pos)
                row += 1
        alone.append(out.clone())
    graphs, streams = [], [torch.cuda.Stream() for _ in jobs]
    for _, _, out, call in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(3):
                call(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for it in range(10):
        for _, _, out, _ in jobs:
            out.fill_(5.0)
        torch.cuda.synchronize()
        for (_, _, _, call), g, st in zip(jobs, graphs, streams):
            with torch.cuda.stream(st):
                if it % 2:
                    g.replay()
                else:
                    for _ in range(3):
                        call(st.cuda_stream)
        torch.cuda.synchronize()
        for (_, _, out, _), want in zip(jobs, alone):
            assert torch.equal(out, want)
    s.s.check()
    s.close()
