"""The bounds that the 4-bit cache's attention is held to (tests/attn4_bounds.py) on the CPU: an exact output passes, zeros, an
output with one record left out, one with a group's scale wrong and one of a wrong sequence length do not."""
import numpy as np
import pytest

from tests import attn4_bounds as bnd
from tests import attn4_oracle as orc


@pytest.mark.parametrize("prompt", (False, True))
@pytest.mark.parametrize("kind", ("f32", "bf16", "f16"))
@pytest.mark.parametrize("n", (33, 129, 1000))
def test_bounds_tell_wrong_outputs(kind, prompt, n):
    rng = np.random.default_rng(n)
    heads, kv, hd = 8, 2, 128
    k, v = (orc.held(rng.normal(size=(n, kv, hd)).astype(np.float32)) for _ in "kv")
    q = rng.normal(size=(heads, hd)).astype(np.float32)
    want, tol = bnd.attention(q, k, v, hd ** -0.5, kind, prompt)
    assert np.allclose(want, orc.attention(q, k, v, hd ** -0.5)[0], rtol=1e-12, atol=1e-14)
    spread = 2 * np.sqrt(128) * hd ** -0.5 if prompt else 0.0

    def passes(x):
        return bnd.far(x, want, tol) <= 1 and bnd.far_in_norm(x, want, kind, spread) <= 1

    assert passes(want) and passes(want.astype(np.float32))
    assert not passes(0 * want)
    seen = np.ones((kv, n), bool)
    seen[:, 32 * (n // 64):32 * (n // 64) + 32] = False
    assert not passes(bnd.attention(q, k, v, hd ** -0.5, kind, prompt, seen)[0])
    assert not passes(bnd.attention(q, k[:-1], v[:-1], hd ** -0.5, kind, prompt)[0]) or n > 129
    other = want.copy()
    other[3, 32:64] *= 1.05
    assert not passes(other)
    assert not passes(bnd.attention(1.01 * q, k, v, hd ** -0.5, kind, prompt)[0]) or kind != "f32"


def test_one_large_value_loosens_its_group_only():
    rng = np.random.default_rng(1)
    k, v = (orc.held(rng.normal(size=(200, 2, 128)).astype(np.float32)) for _ in "kv")
    q = rng.normal(size=(4, 128)).astype(np.float32)
    _, before = bnd.attention(q, k, v, 0.1, "bf16", True)
    v[7, 0, 3] = 8e5
    _, after = bnd.attention(q, k, v, 0.1, "bf16", True)
    assert (after[:2, :32] > 100 * before[:2, :32]).all() and np.allclose(after[:2, 32:], before[:2, 32:])
    assert np.array_equal(after[2:], before[2:])
