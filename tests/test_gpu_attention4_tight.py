"""Decode, drafted rows and selection over the 4-bit KV cache against definitions in 64 bits, each output within a bound of
its own and each row's head within one on its norm (tests/attn4_bounds.py; tests/test_attention4_bounds.py: what they reject)."""
import numpy as np
import pytest

from tests import attn4_bounds as bnd
from tests import attn4_oracle as orc
from tests.test_gpu_attention4 import KINDS, Session

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,hd", ((16, 16, 128), (32, 8, 128), (7, 1, 64), (20, 1, 128), (12, 4, 64), (64, 2, 64)))
def test_decode_drafted_rows_and_selection(cuda, kind, heads, kv, hd):
    rng = np.random.default_rng(51)
    ctx = 1400
    s = Session(cuda, 3, heads, kv, hd, ctx)
    k = rng.normal(size=(3 * ctx, kv, hd)) * np.exp(0.5 * rng.normal(size=(kv, hd))) + (rng.random((kv, hd)) < 0.05) * 4
    s.write([(i, 0, ctx) for i in range(3)], k.astype(np.float32), rng.normal(size=k.shape).astype(np.float32), kind)
    for entries, n_sel in (([(0, 1399, 1), (1, 31, 1), (2, 700, 1), (0, 64, 1), (1, 0, 1)], None), ([(2, 1390, 7), (0, 29, 5)], None),
                           ([(1, 1330, 1)], None), ([(0, 1399, 1), (2, 1200, 4), (1, 63, 2)], 6), ([(1, 1398, 1)], 3)):
        q = bnd.held_in(cuda, kind, 1.5 * rng.normal(size=(sum(e[2] for e in entries), heads, hd)))
        got, row = s.attend(entries, q, kind, n_sel=n_sel), 0
        got, blocks = got if n_sel else (got, None)
        assert not bnd.takes_prompt_kernel(cuda, len(entries), max(e[2] for e in entries), heads, kv)
        for slot, pos0, rows in entries:
            for pos in range(pos0, pos0 + rows):
                seen = None
                if n_sel:
                    assert np.array_equal(blocks[row], orc.selected(s.k[slot], q[row], pos, n_sel))
                    seen = bnd.seen_of(blocks[row], pos)
                want, tol = bnd.attention(q[row], s.k[slot, :pos + 1], s.v[slot, :pos + 1], hd ** -0.5, kind, False, seen)
                assert bnd.far(got[row], want, tol) <= 1, (slot, pos)
                assert bnd.far_in_norm(got[row], want, kind) <= 1, (slot, pos)
                row += 1
    s.s.check()
    s.close()
