"""The 4-bit KV cache at the edges of what its calls allow: values, queries and scales that 16- and 32-bit numbers hold
barely, against definitions in 64 bits with bounds for each value (tests/attn4_bounds.py)."""
import numpy as np
import pytest

from tests.test_gpu_attention4 import Session

pytestmark = pytest.mark.gpu


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
