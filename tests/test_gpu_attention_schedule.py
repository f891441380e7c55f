"""GPU parity of the attention calls over batches that stretch the split of their work over the SMs, against the plain 64-bit
implementation with its derived bounds (oracle.attention_oracle)."""
import pytest
import torch

from mingmoe import attention as A
from oracle import attention_oracle as O
from test_gpu_attention import BF, FP, cu_of, errors, randn

pytestmark = pytest.mark.gpu


def check_rows(q, k, v, out, lse, rows, heads):
    """Rows [a, e) of one causal sequence, some heads: a row sees the keys up to its own, so keys behind e do not matter."""
    G = q.shape[1] // k.shape[1]
    for a, e in rows:
        for h in heads:
            o, s, to, ts = O.attention_fast(q[a:e, h:h + 1], k[:e, h // G:h // G + 1], v[:e, h // G:h // G + 1], True)
            assert bool(((out[a:e, h:h + 1].double() - o).abs() <= to).all()), (a, h)
            assert bool(((lse[a:e, h:h + 1].double() - s).abs() <= ts).all()), (a, h)


# hq, hkv, tokens, hint: 2.2 and 2.3 million key tiles in one of 1024 sequences
@pytest.mark.parametrize("hq,hkv,n,hint", [(256, 4, 16384, None), (128, 8, 4096, 1)])
def test_one_long_prompt_among_empty_sequences(cuda, hq, hkv, n, hint):
    q, k, v = (randn((n, h, 64), BF, cuda, i) for i, h in enumerate((hq, hkv, hkv)))
    cu = cu_of([0] * 700 + [n] + [0] * 323, cuda)
    out, lse = A.prompt_attention(q, k, v, cu, max_q=hint, return_lse=True)
    assert errors() == []
    check_rows(q, k, v, out, lse, [(0, 200), (n // 2 - 77, n // 2), (n - 130, n)], (0, hq // hkv, hq - 1))


def test_more_key_tiles_than_the_schedule_counts(cuda):
    """65536 tokens of 32 key heads, taken a token at a time: up to 2.15e9 key tiles."""
    n, hq, hkv = 65536, 256, 32
    q, k, v = (randn((n, h, 64), FP, cuda, i) for i, h in enumerate((hq, hkv, hkv)))
    out, lse = A.prompt_attention(q, k, v, cu_of([n], cuda), max_q=1, return_lse=True)
    assert errors() == []
    check_rows(q, k, v, out, lse, [(0, 100), (n // 3, n // 3 + 9), (n - 20, n)], (0, 9, 100, hq - 1))
