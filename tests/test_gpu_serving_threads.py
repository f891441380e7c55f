"""Calls of two host threads at once, each on a stream of its own, whose kernels take very different amounts of shared memory."""
import ctypes as C
import threading

import pytest
import torch

from mingmoe import _lib as L
from mingmoe import fp8, sampling

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def together(calls, times):
    """Each call `times` over in a thread of its own (ctypes lets the others run meanwhile): the statuses other than 0."""
    bad = []
    start = threading.Barrier(len(calls))

    def run(call):
        torch.cuda.synchronize()
        start.wait()
        for i in range(times):
            rc = call()
            if rc != L.MV_OK:
                bad.append((i, rc, L.lib().mv_last_error()))
                return
            if i % 256 == 255:
                torch.cuda.synchronize()

    threads = [threading.Thread(target=run, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return bad


def test_draws(cuda):
    g = torch.Generator(device=cuda).manual_seed(0)
    lib, kept, calls = L.lib(), [], []
    for v in (100, 150000):
        x, u = torch.randn(2, v, generator=g, device=cuda), torch.rand(2, generator=g, device=cuda)
        tokens, stream = torch.empty(2, dtype=torch.int64, device=cuda), torch.cuda.Stream()
        a = L.SampleArgs(x.data_ptr(), u.data_ptr(), 0, 0, 0, 0, tokens.data_ptr(), 0, 0, v, 0, 1.0, 1.0, 0.0, 40, 2, v, L.MV_F32, 0)
        kept.append((x, u, tokens, a, stream))
        calls.append(lambda a=a, st=stream.cuda_stream: lib.mv_sample(C.byref(a), st))
    torch.cuda.synchronize()
    assert together(calls, 50000) == []
    for x, u, tokens, *_ in kept:
        assert torch.equal(tokens, sampling.sample(x, u, top_k=40))


def test_products(cuda):
    g = torch.Generator(device=cuda).manual_seed(1)
    lib, kept, calls = L.lib(), [], []
    for n, k in ((130, 256), (2560, 8192)):
        wq, ws = fp8.quantize_fp8_weight(torch.randn(n, k, generator=g, device=cuda))
        x, y = torch.randn(2, k, generator=g, device=cuda).to(BF), torch.empty(2, n, dtype=F32, device=cuda)
        header, stream = torch.zeros(256, dtype=torch.uint8, device=cuda), torch.cuda.Stream()
        assert lib.mv_fp8_linear_scratch_bytes(2, n, k) == 0
        a = L.Fp8LinearArgs(x.data_ptr(), wq.data_ptr(), ws.data_ptr(), 0, y.data_ptr(), 0, k, wq.stride(0), ws.stride(0), 0, n, 0, 2, n, k,
                            L.MV_BF16, L.MV_F32, 0)
        kept.append((x, wq, ws, y, a, header, stream))
        calls.append(lambda a=a, h=header.data_ptr(), st=stream.cuda_stream: lib.mv_fp8_linear(C.byref(a), h, 256, st))
    torch.cuda.synchronize()
    assert together(calls, 50000) == []
    for x, wq, ws, y, *_ in kept:
        assert torch.equal(y, fp8.fp8_linear(x, wq, ws, out_dtype=F32))
