"""Where the 4-bit KV cache's arrays may lie: on the session's device; host memory is refused before anything is launched."""
import ctypes as C

import numpy as np
import pytest

from tests import attn4_oracle as orc
from tests.test_gpu_attention4 import Session

pytestmark = pytest.mark.gpu


def test_arrays_elsewhere_are_refused(cuda):
    torch = cuda
    s = Session(torch, 2, 4, 2, 64, 130)
    L, a, F32 = s.moe.lib(), s.s.a, s.moe.F32
    d = torch.zeros(8192, device="cuda")
    h = np.zeros(16384, np.float32)
    p, x = d.data_ptr(), (h.ctypes.data + 15) // 16 * 16
    b, out, blocks = s.batch([(0, 3, 2), (1, 7, 1)]), d.data_ptr() + 16384, d.data_ptr() + 24576
    B = s.moe.Attn4Batch
    host = [B(2, 3, 2, x, b.pos0, b.start), B(2, 3, 2, b.slot, x, b.start), B(2, 3, 2, b.slot, b.pos0, x)]
    for f in (lambda b, u, w: L.tr_gpu_attn4_write_dev(a, 0, b, F32, u, 128, w, 128, None),
              lambda b, u, w: L.tr_gpu_attn4_read_dev(a, 0, b, F32, u, 128, w, 128, None),
              lambda b, u, w: L.tr_gpu_attn4_attend_dev(a, 0, b, F32, u, 256, 0.1, w, 256, None),
              lambda b, u, w: L.tr_gpu_attn4_select_dev(a, 0, b, F32, u, 256, 0.1, 1, w, 256, blocks, None)):
        for args in ((b, x, out), (b, p, x), *((w, p, out) for w in host)):
            assert f(*args) == -1 and "memory of the session's device" in s.moe.last_error()
        assert f(b, p, out) == 0
    assert L.tr_gpu_attn4_select_dev(a, 0, b, F32, p, 256, 0.1, 1, out, 256, x, None) == -1
    assert "blocks is not memory" in s.moe.last_error()
    s.s.check()
    s.close()


def test_a_chosen_device(cuda):
    """the same session by the device's number, with pinned rows, and calls inside a capture"""
    torch, moe = cuda, __import__("trochilus_b200.moe", fromlist=["moe"])
    rng = np.random.default_rng(61)
    with pytest.raises(RuntimeError, match="device 99 is none"):
        moe.GpuAttn4(1, 1, 2, 1, 64, 64, device=99)
    a = moe.GpuAttn4(1, 1, 2, 1, 64, 64, device=torch.cuda.current_device())
    k, v = (torch.from_numpy(rng.normal(size=(64, 64)).astype(np.float32)).pin_memory() for _ in "kv")
    at = torch.tensor([0, 0, 0, 64], dtype=torch.int32, device="cuda")
    b = moe.Attn4Batch(1, 64, 64, at.data_ptr(), at.data_ptr() + 4, at.data_ptr() + 8)
    a.write_dev(0, b, moe.F32, k.data_ptr(), 64, v.data_ptr(), 64)
    gk, gv = (torch.zeros((64, 64), device="cuda") for _ in "kv")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.read_dev(0, b, moe.F32, gk.data_ptr(), 64, gv.data_ptr(), 64, stream=torch.cuda.current_stream().cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert np.array_equal(gk.cpu().numpy(), orc.held(k.numpy())) and np.array_equal(gv.cpu().numpy(), orc.held(v.numpy()))
    a.check()
    a.close()


def test_a_refused_launch_is_its_own_call_s_error(cuda):
    """a call on the default stream while a stream that it waits for is captured fails; the calls after it do not"""
    torch = cuda
    rt = C.CDLL("libcudart.so.12")
    s = Session(torch, 1, 4, 2, 64, 130)
    rng = np.random.default_rng(62)
    q, out = torch.ones((1, 256), device="cuda"), torch.zeros((1, 256), device="cuda")
    b, stream, graph = s.batch([(0, 0, 1)]), C.c_void_p(), C.c_void_p()
    assert rt.cudaStreamCreate(C.byref(stream)) == 0
    torch.cuda.synchronize()
    assert rt.cudaStreamBeginCapture(stream, 2) == 0
    L, a, F32 = s.moe.lib(), s.s.a, s.moe.F32
    failed = L.tr_gpu_attn4_attend_dev(a, 0, b, F32, q.data_ptr(), 256, 0.1, out.data_ptr(), 256, None)
    rt.cudaStreamEndCapture(stream, C.byref(graph))
    rt.cudaGetLastError()
    assert failed == -1 and "attention kernel" in s.moe.last_error()
    f = s.moe.GpuAttn(1, 2, 64)  # (another part of the library, which asks for the last error after its launches)
    f.write(0, 0, *rng.normal(size=(2, 3, 2, 128)).astype(np.float32))
    f.close()
    s.write([(0, 0, 130)], *rng.normal(size=(2, 130, 2, 64)).astype(np.float32))  # (raises if the call fails)
    gk, gv = s.read([(0, 0, 130)])
    assert np.array_equal(gk, s.k[0]) and np.array_equal(gv, s.v[0])
    s.s.check()
    assert rt.cudaStreamDestroy(stream) == 0
    s.close()
