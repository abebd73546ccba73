"""The 4-bit KV cache without a GPU: what tr_gpu_attn4_* answers on the host (shapes, sizes, missing sessions), and the
oracle's own definitions on values that can be checked by hand."""
import ctypes as C

import numpy as np

from tests import attn4_oracle as orc


def test_host_logic_without_gpu():
    from trochilus_b200 import moe
    L = moe.lib()
    err = C.create_string_buffer(256)

    def refused(*shape):
        assert not L.tr_gpu_attn4_create(None, C.byref(moe.Attn4Config(*shape)), err, 256)
        assert L.tr_gpu_attn4_bytes(C.byref(moe.Attn4Config(*shape))) == 0 or b"no device" in err.value
        return err.value

    assert b"no configuration" in (L.tr_gpu_attn4_create(None, None, err, 256) or err.value)
    assert b"head_dim 96 not supported" in refused(2, 1, 4, 4, 96, 16)
    for shape in ((0, 1, 4, 4, 128, 16), (2, 0, 4, 4, 128, 16), (2, 65536, 4, 4, 128, 16), (2, 1, 4, 4, 128, 0),
                  (2, 1, 4, 4, 128, (1 << 24) + 1), (-1, 1, 4, 4, 128, 16)):
        assert b"bad shape" in refused(*shape)
    for heads in ((4, 3), (0, 1), (4, 0), (4, 8), (257, 1), (-4, 2)):
        assert b"not supported" in refused(2, 1, *heads, 128, 16)
    assert b"no device" in refused(2, 1, 4, 2, 64, 16)
    # 5 bits a value, 64 positions at a time, and the bounds (2 bytes a dim and a unit for 64 positions)
    rows = 16 * 16 * 4096
    n = moe.GpuAttn4.bytes_needed(16, 1, 16, 16, 128, 4096)
    assert rows * 160 + rows // 64 * 260 <= n < rows * 160 + rows // 64 * 260 + (8 << 20)
    assert moe.GpuAttn4.bytes_needed(1, 1, 1, 1, 64, 65) - moe.GpuAttn4.bytes_needed(1, 1, 1, 1, 64, 64) == 5120 + 132
    b = moe.Attn4Batch(1, 1, 1, None, None, None)
    for rc in (L.tr_gpu_attn4_write_dev(None, 0, b, moe.F32, None, 0, None, 0, None),
               L.tr_gpu_attn4_read_dev(None, 0, b, moe.F32, None, 0, None, 0, None),
               L.tr_gpu_attn4_attend_dev(None, 0, b, moe.F32, None, 0, 1.0, None, 0, None),
               L.tr_gpu_attn4_select_dev(None, 0, b, moe.F32, None, 0, 1.0, 1, None, 0, None, None),
               L.tr_gpu_attn4_write(None, 0, 0, 0, 1, None, None),
               L.tr_gpu_attn4_decode(None, 0, 0, 0, None, None, None, 1.0, None), L.tr_gpu_attn4_check(None)):
        assert rc == -1 and "bad arguments" in moe.last_error()
    L.tr_gpu_attn4_free(None)


def test_oracle_by_hand():
    x = np.zeros((1, 64), np.float32)
    x[0, :32] = np.arange(32) % 16              # scale 1, minimum 0: held exactly
    x[0, 32:] = 7.25                            # one value: scale 0
    assert np.array_equal(orc.held(x), x)
    x[0, :2] = 15, 0.5                          # ties go to the even code
    x[0, 2] = 1.5
    assert orc.held(x)[0, 1] == 0 and orc.held(x)[0, 2] == 2
    x[0, 40] = np.inf
    assert np.isnan(orc.held(x)[0, 32:]).all() and np.isfinite(orc.held(x)[0, :32]).all()
    k = np.zeros((130, 1, 64), np.float32)
    k[:64], k[64:128] = 1.0, -2.0
    lo, hi, unit = orc.bounds(k)
    assert unit[:, 0].tolist() == [2 ** -6, 2 ** -5] and hi[0, 0, 0] == 64 and lo[1, 0, 0] == -64
    q = np.ones((1, 64), np.float32)
    assert orc.selected(k, q, 129, 2).tolist() == [[0, 2]] and orc.selected(k, -q, 129, 2).tolist() == [[1, 2]]
    assert orc.selected(k, q, 129, 4).tolist() == [[0, 1, 2, -1]] and orc.selected(k, q, 5, 1).tolist() == [[0]]
    out, size = orc.attention(q, k[:1], k[:1] + 3, 0.5)
    assert np.allclose(out, 4) and size == 32
