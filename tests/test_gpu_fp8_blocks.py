"""GPU parity of products with 8-bit weights over many blocks of K, whose scales all differ: each block of a tile meets its own, in
tiles that follow one another through the same stages, and behind the 32 scales that a lane's register holds."""
import pytest
import torch

from mingmoe import _lib as L
from mingmoe import fp8 as F
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def uneven(dev, rows, k, seed):
    """Values whose blocks of 128 columns differ by powers of 2^8, in every row its own."""
    g = torch.Generator(device=dev).manual_seed(seed)
    blocks = -(-k // 128)
    e = torch.randint(-3, 4, (rows, blocks), generator=g, device=dev)
    x = torch.randn(rows, blocks * 128, generator=g, device=dev) * torch.exp2(8.0 * e).repeat_interleave(128, 1)
    return x[:, :k].contiguous()


@pytest.mark.parametrize("t,n,k", [(3, 2560, 8192), (20, 900, 4225), (61, 9000, 4225), (100, 20000, 1100), (300, 2048, 8320),
                                   (700, 5632, 4225), (700, 5632, 8320), (2100, 5632, 4225), (5000, 2300, 640)])
def test_every_block_meets_its_scales(cuda, t, n, k):
    x = uneven(cuda, t, k, 1).to(BF)
    wq, ws = F.quantize_fp8_weight(uneven(cuda, n, k, 2) * 0.02)
    y = F.fp8_linear(x, wq, ws, out_dtype=F32)
    for i in range(0, t, 700):
        ref, mag = O.fp8_linear(x[i:i + 700], wq, ws)
        assert bool(((y[i:i + 700].double() - ref).abs() <= O.fp8_bound(ref, mag, k, F32)).all())
    for _ in range(3):
        assert torch.equal(F.fp8_linear(x, wq, ws, out_dtype=F32), y)
    torch.cuda.synchronize()
    assert not L.all_workspace_errors()
