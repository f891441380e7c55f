"""Calls that are the first of their thread to reach the GPU, as a server's worker threads make them: the same results."""
import threading

import pytest
import torch

from mingmoe import _lib as L
from mingmoe import attention, fp8
from mingmoe.block import MoeBlock
from oracle import moe_oracle as MO

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def in_a_new_thread(call):
    result = []

    def run():
        try:
            result.append(call())
        except Exception as e:  # the thread's error is the test's
            result.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    if isinstance(result[0], Exception):
        raise result[0]
    return result[0]


@pytest.mark.parametrize("t", [1, 30, 700])
def test_products(cuda, t):
    g = torch.Generator(device=cuda).manual_seed(0)
    wq, ws = fp8.quantize_fp8_weight(torch.randn(5000, 512, generator=g, device=cuda))
    x = torch.randn(t, 512, generator=g, device=cuda).to(BF)
    want = fp8.fp8_linear(x, wq, ws)
    torch.cuda.synchronize()
    assert torch.equal(in_a_new_thread(lambda: fp8.fp8_linear(x, wq, ws)), want)


@pytest.mark.parametrize("t", [1, 300])
def test_attention(cuda, t):
    g = torch.Generator(device=cuda).manual_seed(1)
    q, k, v = (torch.randn(t, h, 64, generator=g, device=cuda).to(BF) for h in (4, 2, 2))
    cu = torch.tensor([0, t], dtype=torch.int32, device=cuda)
    cache = attention.PagedKV.empty(20, 16, 2, 64, BF, cuda)
    table, lens = torch.arange(20, dtype=torch.int32, device=cuda)[None], torch.tensor([t], dtype=torch.int32, device=cuda)
    attention.kv_append(cache, k, v, table, cu, lens)
    for call in (lambda: attention.prompt_attention(q, k, v, cu, max_q=t), lambda: attention.paged_attention(q, cache, table, cu, lens, max_q=t)):
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(in_a_new_thread(call), want)


def test_blocks(cuda):
    block = MoeBlock.from_params(MO.make_block_params(seed=0, H=256, I=128, E=16, I_s=256), top_k=4)
    x = torch.randn(40, 256, generator=torch.Generator(device=cuda).manual_seed(2), device=cuda).to(BF)
    for call in (lambda: block.decode(x[:8]), lambda: block.decode(x[:1]), lambda: block.prefill(x)):
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(in_a_new_thread(call), want)
    assert not L.all_workspace_errors()
