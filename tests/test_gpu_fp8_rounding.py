"""GPU parity of the rounding to e4m3 blocks at the ends of the types and at sizes that take four blocks a thread."""
import math

import pytest
import torch

from mingmoe import fp8 as F
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_weights_at_the_end_of_the_type(cuda, dtype):
    """Only infinities and NaNs make a block not finite: the type's largest numbers do not."""
    top = torch.finfo(dtype).max
    w = torch.randn(384, 256, generator=torch.Generator(device=cuda).manual_seed(0), device=cuda).to(dtype)
    w[5, 7], w[200, 130], w[300, 0] = top, -top, math.inf
    w[310, 200] = math.nan
    q, s = F.quantize_fp8_weight(w)
    assert torch.isnan(s).tolist() == [[False, False], [False, False], [True, True]]
    big = (torch.tensor(top, dtype=torch.float64) / 448).float().item()
    assert s[0, 0].item() == s[1, 1].item() == big
    # quotients of fp32 numbers, rounded to fp32: 448 and what lies that far below
    for i, j in ((0, 0), (1, 1), (0, 1), (1, 0)):
        rows, cols = slice(i * 128, i * 128 + 128), slice(j * 128, j * 128 + 128)
        want = O.round_e4m3((w[rows, cols].double() / s[i, j].double()).float().double().clamp(-448, 448))
        assert torch.equal(q[rows, cols].double(), want)
    assert q[5, 7].float().item() == 448 and q[200, 130].float().item() == -448


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("t,k,off,st", [(40001, 256, 0, 256), (80000, 100, 4, 104), (8001, 1281, 1, 1283), (1300, 8000, 0, 8000), (77000, 4, 0, 4),
                                        (4737, 2044, 0, 2044)])
def test_more_blocks_than_threads_take_one_by_one(cuda, dtype, t, k, off, st):
    """From 64 x 8 blocks for each SM on a thread takes four, 16 apart; rows at every alignment, ragged last blocks."""
    assert t * -(-k // 128) > 64 * 8 * torch.cuda.get_device_properties(0).multi_processor_count
    g = torch.Generator(device=cuda).manual_seed(1)
    flat = torch.randn(t * st + 16, generator=g, device=cuda) * torch.exp2(torch.randint(-8, 9, (t * st + 16,), generator=g, device=cuda).float())
    x = torch.as_strided(flat.to(dtype), (t, k), (st, 1), off)
    q, scale = F.quantize_fp8(x)
    for i in range(0, t, 8000):
        rq, rs = O.quantize(x[i:i + 8000])
        assert torch.equal(scale[i:i + 8000].double(), rs) and torch.equal(q[i:i + 8000].double(), rq)


@pytest.mark.parametrize("off", [0, 1])
def test_products_of_as_many_blocks(cuda, off):
    """The same rounding in front of a product: the rows' results are those of the rows by themselves."""
    x = torch.randn(9600, 1026, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda).to(BF)[:, off:off + 1025]
    wq, ws = F.quantize_fp8_weight(torch.randn(600, 1025, generator=torch.Generator(device=cuda).manual_seed(3), device=cuda))
    y = F.fp8_linear(x, wq, ws, out_dtype=F32)
    for i in range(0, 9600, 2400):
        ref, mag = O.fp8_linear(x[i:i + 2400], wq, ws)
        assert bool(((y[i:i + 2400].double() - ref).abs() <= O.fp8_bound(ref, mag, 1025, F32)).all())
