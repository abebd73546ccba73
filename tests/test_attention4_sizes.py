"""Shapes of 4-bit KV caches whose bytes pass 64 bits are refused before anything is allocated (no GPU needed)."""
import ctypes as C

from trochilus_b200 import moe


def test_sizes_past_64_bits_are_refused():
    L = moe.lib()
    err = C.create_string_buffer(256)
    k15, ctx = 1 << 15, 1 << 24
    # 2^63 blocks of 10240 bytes: 0 modulo 2^64, so that the sum of the small parts would pass for the size
    for shape in ((k15, k15, k15, k15, 128, ctx), (k15, k15, k15, k15, 64, ctx), (65535, 65535, 65535, 65535, 128, ctx),
                  (k15, k15, 16, 16, 128, ctx), (1 << 14, 1 << 14, 1 << 8, 1 << 8, 128, ctx)):
        cfg = moe.Attn4Config(*shape)
        assert L.tr_gpu_attn4_bytes(C.byref(cfg)) == 0 and "too many" in moe.last_error()
        assert not L.tr_gpu_attn4_create(None, C.byref(cfg), err, 256) and b"too many" in err.value
    # the largest shapes below: sizes in whole blocks (codes, scales, bounds and a unit a block)
    for layers, seqs, kv, n in ((1 << 10, 1 << 10, 1 << 10, ctx), (1 << 14, 1 << 14, 1 << 2, ctx), (1, 65535, 16, ctx)):
        blocks = layers * seqs * kv * (n // 64)
        assert 0 <= moe.GpuAttn4.bytes_needed(layers, seqs, kv, kv, 128, n) - blocks * (10240 + 256 + 4) < 1 << 29
