"""GPU parity of the attention calls on arguments at the edge of what they take, against the plain 64-bit implementation."""
import pytest
import torch

from mingmoe import attention as A
from oracle import attention_oracle as O
from test_gpu_attention import BF, Paged, check, cu_of, errors, randn

pytestmark = pytest.mark.gpu


def off(t, n):
    """The tensor's values in a contiguous tensor that begins n elements behind a 16-byte address."""
    flat = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)
    return flat[n:n + t.numel()].view(t.shape).copy_(t)


@pytest.mark.parametrize("n", [1, 4])
def test_operands_off_a_16_byte_address(cuda, n):
    new, kv = [3, 2], [40, 2]
    P = Paged(cuda, BF, 2, 128, 16, kv)
    cu = cu_of(new, cuda)
    q, k, v = (randn((5, h, 128), BF, cuda, i) for i, h in enumerate((8, 2, 2)))
    refs = [O.attention(q[cu[b]:cu[b + 1]], P.k[b], P.v[b], True) for b in range(2)]
    check(A.paged_attention(off(q, n), P.cache, P.table, cu, P.lens), None, refs, cu)
    refs = [O.attention(q[cu[b]:cu[b + 1]], k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]], True) for b in range(2)]
    check(A.prompt_attention(off(q, n), off(k, n), off(v, n), cu), None, refs, cu)
    assert torch.equal(A.kv_append(P.cache, off(k, n), off(v, n), P.table, cu, P.lens, q=off(q, n)), q)
    assert torch.equal(O.gather(P.kc, P.table[0], 40)[37:], k[:3]) and torch.equal(O.gather(P.vc, P.table[1], 2), v[3:])
    assert errors() == []


def test_page_table_without_columns(cuda):
    """Sequences that have no page yet: rows without a key."""
    P = Paged(cuda, BF, 2, 128, 16, [0, 0])
    q = randn((3, 8, 128), BF, cuda, 1)
    for hint in (2, 1000):
        for causal in (True, False):
            out, lse = A.paged_attention(q, P.cache, P.table[:, :0].contiguous(), cu_of([1, 2], cuda), P.lens, max_q=hint,
                                         causal=causal, return_lse=True)
            assert bool((out == 0).all()) and bool((lse == -torch.inf).all())
    assert errors() == []
    # a length that has no page is clamped to none and reported
    out = A.paged_attention(q, P.cache, P.table[:, :0].contiguous(), cu_of([1, 2], cuda), P.lens + 1)
    assert bool((out == 0).all()) and errors() == [5]


@pytest.mark.parametrize("name", ["causal", "return_lse"])
def test_flag_without_a_truth_value(cuda, name):
    """A flag whose truth value raises: that error, and nothing is launched."""
    P = Paged(cuda, BF, 2, 128, 16, [3])
    q, cu, out = randn((1, 8, 128), BF, cuda, 1), cu_of([1], cuda), torch.full((1, 8, 128), 7.0, dtype=BF, device=cuda)
    A.paged_attention(q, P.cache, P.table, cu, P.lens)  # the stream's workspace exists: calls go through the host module
    for flag in (torch.ones(2), torch.ones(2, device=cuda)):
        with pytest.raises(RuntimeError, match="ambiguous"):
            A.paged_attention(q, P.cache, P.table, cu, P.lens, out=out, **{name: flag})
        with pytest.raises(RuntimeError, match="ambiguous"):
            A.prompt_attention(q, q, q, cu, out=out, **{name: flag})
    assert bool((out == 7).all())
    k = randn((1, 2, 128), BF, cuda, 2)
    before = P.kc.clone()
    with pytest.raises(RuntimeError, match="ambiguous"):
        A.kv_append(P.cache, k, k, P.table, cu, P.lens, interleaved=torch.ones(2))
    assert torch.equal(before.view(torch.int16), P.kc.view(torch.int16))
