"""GPU parity of the attention calls over batches that stretch the split of their work over the SMs, against the plain 64-bit
implementation with its derived bounds (oracle.attention_oracle)."""
import pytest
import torch

from mingmoe import attention as A
from oracle import attention_oracle as O
from test_gpu_attention import BF, FP, Paged, check, cu_of, errors, randn

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


# Batches whose items are cut under each of the rules that a kernel has for it (attn_split.cu, attn_tile.cu): many items of
# single tokens, few of them, packed short prompts with a longer one among them, other prompts and chunks.

def gathered(cuda, dtype, hkv, d, page, kv, seed):
    P = Paged(cuda, dtype, hkv, d, page, kv, seed=seed)
    return P, [O.gather(P.kc, P.table[b], n) for b, n in enumerate(kv)], [O.gather(P.vc, P.table[b], n) for b, n in enumerate(kv)]


@pytest.mark.parametrize("dtype,d,hq,hkv,B", [(BF, 128, 16, 4, 61), (FP, 64, 14, 2, 90), (FP, 128, 12, 1, 200), (BF, 128, 8, 4, 5)])
def test_single_tokens_over_uneven_lengths(cuda, dtype, d, hq, hkv, B):
    kv = [1 + (b * b * 997 + 61 * b) % (4001 if b % 5 else 200) for b in range(B)]
    P, ks, vs = gathered(cuda, dtype, hkv, d, 32, kv, seed=B)
    cu = cu_of([1] * B, cuda)
    q = randn((B, hq, d), dtype, cuda, 8, 2.0)
    out, lse = A.paged_attention(q, P.cache, P.table, cu, P.lens, max_q=1, return_lse=True)
    check(out, lse, [O.attention_fast(q[b:b + 1], ks[b], vs[b], True) for b in range(B)], cu)
    assert torch.equal(out, A.paged_attention(q, P.cache, P.table, cu, P.lens, max_q=1))
    assert errors() == []


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,d,hq,hkv", [(BF, 128, 16, 4), (FP, 64, 8, 8)])
def test_longer_prompt_among_short_ones(cuda, dtype, d, hq, hkv, causal):
    lens = [100, 1500, 33, 260, 64, 1, 700, 390, 128, 200]
    T = sum(lens)
    q, k, v = (randn((T, h, d), dtype, cuda, 30 + i, 1.5) for i, h in enumerate((hq, hkv, hkv)))
    cu = cu_of(lens, cuda)
    refs = [O.attention_fast(q[cu[b]:cu[b + 1]], k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]], causal) for b in range(len(lens))]
    out, lse = A.prompt_attention(q, k, v, cu, causal=causal, return_lse=True)
    check(out, lse, refs, cu)
    assert errors() == []


@pytest.mark.parametrize("hint", [None, 1])
@pytest.mark.parametrize("dtype,d,hq,hkv", [(BF, 128, 16, 4), (FP, 64, 14, 2)])
def test_chunk_beside_single_tokens(cuda, dtype, d, hq, hkv, hint):
    new = [1] * 20 + [500] + [1] * 19 + [0, 3]
    kv = [n + (137 * b * b) % 2500 for b, n in enumerate(new)]
    P, ks, vs = gathered(cuda, dtype, hkv, d, 16, kv, seed=3)
    cu = cu_of(new, cuda)
    q = randn((sum(new), hq, d), dtype, cuda, 9, 1.5)
    refs = [O.attention_fast(q[cu[b]:cu[b + 1]], ks[b], vs[b], True) for b in range(len(new))]
    out, lse = A.paged_attention(q, P.cache, P.table, cu, P.lens, max_q=hint, return_lse=True)
    check(out, lse, refs, cu)
    assert errors() == []


@pytest.mark.parametrize("interleaved", [False, True])
def test_both_host_paths_give_the_same(cuda, monkeypatch, interleaved):
    """The same plain arguments through the C++ host module and through the Python code behind it: equal bits."""
    new, kv = [3, 1, 40], [30, 200, 40]
    P, R = (Paged(cuda, BF, 2, 128, 16, kv, seed=4) for _ in range(2))
    qkv = randn((44, 12, 128), BF, cuda, 2)
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    cu, cs = cu_of(new, cuda), A.rotation_table(256, 64, device=cuda)
    cuk = cu_of([44, 0, 0], cuda)
    where = torch.arange(44, dtype=torch.int32, device=cuda)

    def calls(X):
        qr = A.kv_append(X.cache, k, v, X.table, cu, X.lens, q=q, cos_sin=cs, positions=where, interleaved=interleaved)
        into = torch.zeros_like(qr)
        assert A.kv_append(X.cache, k, v, X.table, cu, X.lens, q=q, q_out=into, cos_sin=cs) is into
        o = A.paged_attention(qr, X.cache, X.table, cu, X.lens, max_q=40, scale=0.2, causal=False, return_lse=True)
        p = A.prompt_attention(q, k, v, cu, cu_seqlens_k=cuk, scale=0.1, causal=False, return_lse=True)
        return [qr, into, *o, *p, A.paged_attention(qr, X.cache, X.table, cu, X.lens), A.prompt_attention(q, k, v, cu),
                X.kc, X.vc]

    calls(P)
    native = calls(P)

    class Nothing:
        kv_append = paged_attention = prompt_attention = staticmethod(lambda *a: NotImplemented)

    monkeypatch.setattr(A, "_module", Nothing)
    for a, b in zip(native, calls(R)):
        assert torch.equal(a.contiguous().view(torch.int16), b.contiguous().view(torch.int16))
    assert errors() == []
