"""Products whose weights, scales and activations are written by the kernel right in front of them."""
import pytest
import torch

from mingmoe import fp8 as F

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("t", [1, 4, 16, 100, 700])
def test_weights_written_right_before(cuda, t):
    g = torch.Generator(device=cuda).manual_seed(0)
    ws_ = [torch.randn(2560, 2048, generator=g, device=cuda) for _ in range(3)]
    x = torch.randn(t, 2048, generator=g, device=cuda).to(BF)
    packed = [F.quantize_fp8_weight(w) for w in ws_]
    want = [F.fp8_linear(x, *p) for p in packed]
    torch.cuda.synchronize()
    wq, ws = torch.empty(2560, 2048, dtype=torch.uint8, device=cuda), torch.empty_like(packed[0][1])
    for i in range(60):
        q, s = packed[i % 3]
        ws.copy_(s)
        wq.copy_(q.view(torch.uint8))
        a = F.fp8_linear(x, wq.view(F.E4M3), ws)
        b = F.fp8_linear(x, *F.quantize_fp8_weight(ws_[i % 3]))
        y = torch.zeros_like(x)
        y.copy_(x)
        c = F.fp8_linear(y, q, s)
        assert torch.equal(a, want[i % 3]) and torch.equal(b, want[i % 3]) and torch.equal(c, want[i % 3])
