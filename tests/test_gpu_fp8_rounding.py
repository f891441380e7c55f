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
