"""GPU parity: appending to the paged cache, attention over it, attention over packed prompts, against the plain
64-bit implementation.

Bar: copied values (v, unrotated parts, untouched cache slots) are bit-equal. Everything else lies within the bound
that oracle.attention_oracle derives for each element from the promised arithmetic: one rounding of the result to the
element type, one of each softmax weight (u = 2^-8 bf16, 2^-11 f16), fp32 everywhere else."""
import math
import random

import pytest
import torch

from mingmoe import _lib as L
from mingmoe import attention as A
from oracle import attention_oracle as O

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16
NAN = float("nan")


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def cu_of(lens, dev):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return ints(c, dev)


def errors():
    torch.cuda.synchronize()
    return sorted(c for c, _ in L.all_workspace_errors().values())


def randn(shape, dtype, dev, seed, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)


class Paged:
    """A batch of sequences in a shuffled cache whose every other slot is NaN; unused page ids are nonsense."""

    def __init__(self, dev, dtype, hkv, d, page, kv, hnd=False, seed=0, spare=3):
        need = [-(-n // page) for n in kv]
        n_pages = sum(need) + spare
        order = list(range(n_pages))
        random.Random(seed).shuffle(order)
        width = max(need + [1]) + 2
        shape = (n_pages, hkv, page, d) if hnd else (n_pages, page, hkv, d)
        self.kc, self.vc = (torch.full(shape, NAN, dtype=dtype, device=dev) for _ in range(2))
        if hnd:
            self.kc, self.vc = self.kc.transpose(1, 2), self.vc.transpose(1, 2)
        rows, at = [], 0
        self.k, self.v = [], []
        for b, n in enumerate(kv):
            ids = order[at:at + need[b]]
            at += need[b]
            rows.append(ids + [-(10 ** 6) if i % 2 else 10 ** 9 for i in range(width - len(ids))])
            k, v = randn((n, hkv, d), dtype, dev, 100 * seed + b), randn((n, hkv, d), dtype, dev, 100 * seed + b + 50)
            j = torch.arange(n, device=dev)
            pg = torch.tensor(ids + [0], device=dev)[j // page]
            self.kc[pg, j % page], self.vc[pg, j % page] = k, v
            self.k.append(k)
            self.v.append(v)
        self.table = ints(rows, dev).reshape(len(kv), width)
        self.lens = ints(kv, dev)
        self.cache = A.PagedKV(self.kc, self.vc)


def check(out, lse, refs, cu):
    for b, (o, s, to, ts) in enumerate(refs):
        a, e = int(cu[b]), int(cu[b + 1])
        d = (out[a:e].double() - o).abs()
        assert bool((d <= to).all()), (b, d.max().item(), (d - to).max().item())
        if lse is not None:
            empty = torch.isinf(s)
            assert torch.equal(lse[a:e][empty].double(), s[empty])
            assert bool(((lse[a:e].double() - s).abs()[~empty] <= ts[~empty]).all()), b


# ------------------------------------------------------------------------------------------------ kv_append

@pytest.mark.parametrize("dtype,d,hq,hkv,page,rot,inter,hnd", [
    (BF, 128, 16, 4, 16, 128, False, False), (FP, 64, 14, 2, 8, 32, True, False), (BF, 64, 5, 5, 32, 64, False, True),
    (FP, 128, 12, 1, 256, 48, False, False), (BF, 128, 3, 3, 64, 0, False, False), (BF, 128, 32, 2, 128, 128, True, True)])
def test_append(cuda, dtype, d, hq, hkv, page, rot, inter, hnd):
    new, kv = [3, 0, 1, 17, 5], [3, 9, 70, 300, 5]
    T = sum(new)
    P = Paged(cuda, dtype, hkv, d, page, kv, hnd=hnd, seed=d + page)
    kc0, vc0 = P.kc.clone(), P.vc.clone()
    qkv = randn((T + 2, hq + 2 * hkv, d), dtype, cuda, 7)[1:-1]
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    cs = A.rotation_table(301, rot, device=cuda) if rot else None
    cu = cu_of(new, cuda)
    qo = A.kv_append(P.cache, k, v, P.table, cu, P.lens, q=q, cos_sin=cs, interleaved=inter)
    pos = torch.cat([torch.arange(n - m, n) for m, n in zip(new, kv)]).to(cuda)
    seq = torch.cat([torch.full((m,), b) for b, m in enumerate(new)]).to(cuda)
    pg = P.table[seq, pos // page].long()
    if rot:
        for got, x in ((qo, q), (P.kc[pg, pos % page], k)):
            y, tol = O.rotate(x, cs, pos, inter)
            assert bool(((got.double() - y).abs() <= tol).all())
            assert torch.equal(got[..., rot:], x[..., rot:])
    else:
        assert torch.equal(qo, q) and torch.equal(P.kc[pg, pos % page], k)
    assert torch.equal(P.vc[pg, pos % page], v)
    # nothing else changed
    kc0[pg, pos % page], vc0[pg, pos % page] = P.kc[pg, pos % page], P.vc[pg, pos % page]
    bits = torch.int16
    assert torch.equal(P.kc.contiguous().view(bits), kc0.contiguous().view(bits))
    assert torch.equal(P.vc.contiguous().view(bits), vc0.contiguous().view(bits))
    assert errors() == []


@pytest.mark.parametrize("B", [1, 31, 32, 33, 200, 1100])
def test_append_many_sequences(cuda, B):
    rnd = random.Random(B)
    new = [rnd.choice([0, 1, 1, 2, 5]) for _ in range(B - 1)] + [2]
    kv = [n + rnd.randrange(0, 40) for n in new]
    P = Paged(cuda, BF, 1, 64, 16, kv, seed=B % 7)
    T = sum(new)
    k, v = randn((T, 1, 64), BF, cuda, 1), randn((T, 1, 64), BF, cuda, 2)
    assert A.kv_append(P.cache, k, v, P.table, cu_of(new, cuda), P.lens) is None
    pos = torch.cat([torch.arange(n - m, n) for m, n in zip(new, kv)]).to(cuda)
    seq = torch.cat([torch.full((m,), b) for b, m in enumerate(new)]).to(cuda)
    pg = P.table[seq, pos // 16].long()
    assert torch.equal(P.kc[pg, pos % 16], k) and torch.equal(P.vc[pg, pos % 16], v)
    assert errors() == []


def test_append_positions_and_in_place_q(cuda):
    new, kv = [4, 2], [4, 30]
    P = Paged(cuda, BF, 2, 128, 16, kv)
    q, k, v = (randn((6, h, 128), BF, cuda, i) for i, h in enumerate((8, 2, 2)))
    q0 = q.clone()
    cs = A.rotation_table(50, 64, device=cuda)
    where = ints([0, 49, 3, 3, 17, 8], cuda)
    qo = A.kv_append(P.cache, k, v, P.table, cu_of(new, cuda), P.lens, q=q, q_out=q, cos_sin=cs, positions=where)
    assert qo is q
    y, tol = O.rotate(q0, cs, where, False)
    assert bool(((q.double() - y).abs() <= tol).all())
    y, tol = O.rotate(k, cs, where, False)
    got = torch.cat([O.gather(P.kc, P.table[0, :1], 4), O.gather(P.kc, P.table[1, :2], 30)[28:]])
    assert bool(((got.double() - y).abs() <= tol).all())
    assert errors() == []


def test_append_skips_what_is_outside(cuda):
    """A token whose page id, length or position does not fit is skipped and reported; its neighbours are written."""
    P = Paged(cuda, BF, 1, 64, 16, [20, 20, 20])
    kc0 = P.kc.clone()
    table = P.table.clone()
    table[1, 1] = P.cache.num_pages  # page of tokens 16.. of sequence 1
    k, v, q = (randn((9, 1, 64), BF, cuda, i) for i in range(3))
    cs = A.rotation_table(19, 64, device=cuda)  # position 19 is outside
    qo = torch.zeros_like(q)
    cu = ints([0, 2, 7, 8], cuda)  # row 8 belongs to nobody
    A.kv_append(P.cache, k, v, table, cu, ints([19, 19, 1], cuda), q=q, q_out=qo, cos_sin=cs)
    written = {0, 1, 2, 3, 7}  # sequence 1: positions 14, 15 in its first page, 16.. in the bad one
    for t in range(9):
        assert bool(qo[t].abs().sum() > 0) == (t in written), t
    kc = kc0.view(torch.int16) != P.kc.view(torch.int16)
    assert int(kc.flatten(2).any(-1).sum()) == len(written)
    assert errors() == [4]
    A.kv_append(P.cache, k[:3], v[:3], P.table, ints([0, 3, 3, 3], cuda), ints([2, 0, 0], cuda))  # shorter than its chunk
    assert errors() == [4]
    A.kv_append(P.cache, k[:1], v[:1], P.table, ints([0, 1, 1, 1], cuda), ints([20], cuda).expand(3).contiguous(),
                cos_sin=cs)
    assert errors() == [4]


# ------------------------------------------------------------------------------------------------ paged_attention

PAGED = [  # dtype, d, hq, hkv, page, new, kv
    (BF, 128, 16, 4, 16, [1], [1]),
    (BF, 128, 16, 4, 16, [1, 1, 1, 1], [63, 64, 65, 700]),
    (FP, 64, 14, 2, 8, [1, 1, 1], [7, 129, 1000]),
    (FP, 128, 8, 8, 32, [1, 2, 1], [40, 256, 31]),
    (BF, 64, 16, 1, 64, [1, 3], [200, 90]),
    (BF, 128, 32, 1, 128, [1, 2], [500, 127]),
    (BF, 128, 12, 2, 256, [5, 1, 0, 9], [5, 300, 12, 1200]),
    (FP, 128, 15, 5, 16, [8, 2], [77, 515]),
    (BF, 128, 16, 4, 64, [130, 17, 1], [130, 400, 333]),
    (FP, 64, 28, 4, 32, [65, 256], [300, 256]),
    (BF, 128, 64, 1, 128, [1, 5], [500, 127]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(PAGED)))
def test_paged(cuda, case, causal):
    dtype, d, hq, hkv, page, new, kv = PAGED[case]
    P = Paged(cuda, dtype, hkv, d, page, kv, seed=case)
    cu = cu_of(new, cuda)
    q = randn((sum(new), hq, d), dtype, cuda, 11, 2.0)
    refs = [O.attention(q[cu[b]:cu[b + 1]], P.k[b], P.v[b], causal) for b in range(len(new))]
    # the hint only chooses the kernel: every choice gives the result
    for hint in (None, max(new), 1, 4, 1000):
        out, lse = A.paged_attention(q, P.cache, P.table, cu, P.lens, max_q=hint, causal=causal, return_lse=True)
        check(out, lse, refs, cu)
    assert errors() == []


@pytest.mark.parametrize("hint", [1, 1000])
def test_paged_empty_rows(cuda, hint):
    """Sequences shorter in the cache than their chunk, and empty ones: rows without a key are 0 / -inf."""
    new, kv = [3, 2, 1, 0, 40], [0, 1, 0, 5, 33]
    P = Paged(cuda, BF, 2, 128, 16, kv)
    cu = cu_of(new, cuda)
    q = randn((sum(new), 8, 128), BF, cuda, 3)
    for causal in (True, False):
        out, lse = A.paged_attention(q, P.cache, P.table, cu, P.lens, max_q=hint, causal=causal, return_lse=True)
        check(out, lse, [O.attention(q[cu[b]:cu[b + 1]], P.k[b], P.v[b], causal) for b in range(5)], cu)
        assert bool((out[:3] == 0).all())
    assert errors() == []


@pytest.mark.parametrize("dtype,d,hq,hkv,page,new,n", [(BF, 128, 12, 2, 16, 1, 20011), (FP, 64, 8, 1, 64, 3, 33333),
                                                       (BF, 128, 16, 4, 32, 70, 9001), (FP, 64, 7, 1, 16, 300, 5000)])
def test_paged_long(cuda, dtype, d, hq, hkv, page, new, n):
    """One sequence over the whole card: its key range is cut into pieces that are joined."""
    P = Paged(cuda, dtype, hkv, d, page, [n], seed=5)
    cu = cu_of([new], cuda)
    q = randn((new, hq, d), dtype, cuda, 12, 2.0)
    # a key far above the rest early on, a larger one late: the running maximum has to move and pieces to differ
    P.kc[P.table[0, 2].long(), 3] *= 3
    P.kc[P.table[0, (n - 9 - new) // page].long(), (n - 9 - new) % page] *= 4
    k = O.gather(P.kc, P.table[0], n)
    ref = O.attention_fast(q, k, P.v[0], True)
    for hint in (new, 1, 1000):
        out, lse = A.paged_attention(q, P.cache, P.table, cu, P.lens, max_q=hint, return_lse=True)
        check(out, lse, [ref], cu)
        again = A.paged_attention(q, P.cache, P.table, cu, P.lens, max_q=hint)
        assert torch.equal(again, out)  # fixed order of sums
    assert errors() == []


def test_paged_many_sequences(cuda):
    """More sequences than one launch takes."""
    rnd = random.Random(3)
    new = [rnd.choice([0, 1, 1, 2]) for _ in range(1300)]
    kv = [n + rnd.randrange(0, 20) for n in new]
    P = Paged(cuda, BF, 1, 64, 8, kv)
    cu = cu_of(new, cuda)
    q = randn((sum(new), 2, 64), BF, cuda, 4)
    refs = [O.attention(q[cu[b]:cu[b + 1]], P.k[b], P.v[b], True) for b in range(1300)]
    for hint in (2, 1000):
        out, lse = A.paged_attention(q, P.cache, P.table, cu, P.lens, max_q=hint, return_lse=True)
        check(out, lse, refs, cu)
    assert errors() == []


@pytest.mark.parametrize("hint", [1, 1000])
def test_paged_layouts(cuda, hint):
    """A [page, head, token, d] cache, strided queries, an output inside a wider tensor, a given scale."""
    new, kv = [2, 1], [100, 37]
    P = Paged(cuda, FP, 4, 128, 16, kv, hnd=True)
    cu = cu_of(new, cuda)
    q = randn((3, 20, 128), FP, cuda, 5)[:, 3:11]
    big = torch.full((3, 12, 128), 7.0, dtype=FP, device=cuda)
    out = A.paged_attention(q, P.cache, P.table, cu, P.lens, max_q=hint, scale=0.3, out=big[:, 2:10])
    check(out, None, [O.attention(q[cu[b]:cu[b + 1]], P.k[b], P.v[b], True, 0.3) for b in range(2)], cu)
    assert bool((big[:, :2] == 7).all()) and bool((big[:, 10:] == 7).all())
    qt = randn((8, 3, 128), FP, cuda, 6).transpose(0, 1)  # heads outermost
    out = A.paged_attention(qt, P.cache, P.table, cu, P.lens, max_q=hint)
    check(out, None, [O.attention(qt[cu[b]:cu[b + 1]], P.k[b], P.v[b], True) for b in range(2)], cu)
    assert errors() == []


@pytest.mark.parametrize("hint", [1, 1000])
def test_paged_offsets_past_32_bits(cuda, hint):
    """Pages beyond 2^32 elements of the cache."""
    pages = (1 << 32) // (64 * 4 * 128) + 40
    kc, vc = (torch.empty(pages, 64, 4, 128, dtype=BF, device=cuda) for _ in range(2))
    kc[-2:], vc[-2:] = randn((2, 64, 4, 128), BF, cuda, 1), randn((2, 64, 4, 128), BF, cuda, 2)
    cache = A.PagedKV(kc, vc)
    table = ints([[pages - 1, pages - 2]], cuda)
    k, v, q = (randn((3, h, 128), BF, cuda, 3 + h) for h in (4, 4, 16))
    cu, lens = ints([0, 3], cuda), ints([100], cuda)
    A.kv_append(cache, k, v, table, cu, lens)
    out = A.paged_attention(q, cache, table, cu, lens, max_q=hint)
    kk, vv = O.gather(kc, table[0], 100), O.gather(vc, table[0], 100)
    assert torch.equal(kk[97:], k) and torch.equal(vv[97:], v)
    check(out, None, [O.attention(q, kk, vv, True)], cu)
    assert errors() == []


@pytest.mark.parametrize("hint", [1, 1000])
def test_paged_bad_page_is_reported(cuda, hint):
    P = Paged(cuda, BF, 2, 128, 16, [40, 40])
    q = randn((2, 8, 128), BF, cuda, 1)
    cu = cu_of([1, 1], cuda)
    good = A.paged_attention(q, P.cache, P.table, cu, P.lens, max_q=hint)
    for bad in (-1, P.cache.num_pages, 2 ** 31 - 1):
        table = P.table.clone()
        table[0, 1] = bad
        out = A.paged_attention(q, P.cache, table, cu, P.lens, max_q=hint)
        assert errors() == [4]
        assert torch.equal(out[1], good[1])
    # lengths and bounds that do not fit are clamped and reported
    lens = P.lens.clone()
    lens[0] = 10 ** 6
    A.paged_attention(q, P.cache, torch.zeros_like(P.table), cu, lens, max_q=hint)
    assert errors() == [5]
    A.paged_attention(q, P.cache, P.table, ints([0, 1, 50], cuda), P.lens, max_q=hint)
    assert errors() == [5]


@pytest.mark.parametrize("hint", [1, 1000])
def test_paged_stream_and_graph(cuda, hint):
    """On another stream, and replayed in a graph after the lengths, pages and contents changed."""
    P = Paged(cuda, BF, 4, 128, 16, [300, 90], seed=1)
    R = Paged(cuda, BF, 4, 128, 16, [17, 371], seed=2)
    cu = cu_of([1, 1], cuda)
    q = randn((2, 16, 128), BF, cuda, 1)
    cs = A.rotation_table(400, 128, device=cuda)
    k, v = randn((2, 4, 128), BF, cuda, 2), randn((2, 4, 128), BF, cuda, 3)

    def step(cache, table, lens):
        qr = A.kv_append(cache, k, v, table, cu, lens, q=q, cos_sin=cs)
        return A.paged_attention(qr, cache, table, cu, lens, max_q=hint)

    n = max(P.kc.shape[0], R.kc.shape[0])
    w = max(P.table.shape[1], R.table.shape[1])
    kc, vc = (torch.zeros(n, 16, 4, 128, dtype=BF, device=cuda) for _ in range(2))
    table, lens = torch.zeros(2, w, dtype=torch.int32, device=cuda), torch.ones(2, dtype=torch.int32, device=cuda)
    cache = A.PagedKV(kc, vc)

    def load(X):
        kc[:X.kc.shape[0]], vc[:X.vc.shape[0]] = X.kc, X.vc
        table[:, :X.table.shape[1]] = X.table
        lens.copy_(X.lens)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        load(P)
        eager = step(cache, table, lens)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = step(cache, table, lens)
    torch.cuda.current_stream().wait_stream(s)
    for X in (P, R):
        load(X)
        g.replay()
        torch.cuda.synchronize()
        want = step(X.cache, X.table, X.lens)
        assert torch.equal(out, want)
        if X is P:
            assert torch.equal(eager, want)
    assert errors() == []


# ------------------------------------------------------------------------------------------------ prompt_attention

PROMPTS = [  # dtype, d, hq, hkv, lens
    (BF, 128, 16, 4, [1]),
    (BF, 128, 16, 4, [37]),
    (BF, 128, 16, 4, [64, 1, 0, 127, 129, 30]),
    (FP, 64, 14, 2, [200, 17, 128]),
    (BF, 64, 4, 4, [130, 256, 5]),
    (FP, 128, 6, 2, [63, 65]),
    (BF, 128, 20, 1, [33, 150]),
    (FP, 128, 32, 1, [5, 20]),
    (BF, 64, 80, 2, [33, 150]),
    (FP, 128, 64, 1, [5, 20]),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_prompt(cuda, case, causal):
    dtype, d, hq, hkv, lens = PROMPTS[case]
    T = sum(lens)
    # rows of nobody before and behind the sequences hold NaN
    qkv = randn((T + 9, hq + 2 * hkv, d), dtype, cuda, case)
    qkv[:4], qkv[T + 4:] = NAN, NAN
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    cu = cu_of([4] + lens, cuda)[1:]
    refs = []
    for b in range(len(lens)):
        a, e = int(cu[b]), int(cu[b + 1])
        refs.append(O.attention(q[a:e], k[a:e], v[a:e], causal))
    for hint in (None, 1):
        out0 = torch.full((T + 9, hq, d), 5.0, dtype=dtype, device=cuda)
        out, lse = A.prompt_attention(q, k, v, cu, max_q=hint, causal=causal, return_lse=True, out=out0)
        check(out, lse, refs, cu)
        assert bool((out[:4] == 5).all()) and bool((out[T + 4:] == 5).all())
    assert errors() == []


@pytest.mark.parametrize("causal", [True, False])
def test_prompt_key_lengths_of_their_own(cuda, causal):
    """More keys than queries, fewer (rows without a key), none at all."""
    nq, nk = [5, 140, 3, 70, 0], [200, 90, 0, 70, 8]
    q = randn((sum(nq), 8, 128), BF, cuda, 1)
    k, v = randn((sum(nk), 2, 128), BF, cuda, 2), randn((sum(nk), 2, 128), BF, cuda, 3)
    cu, cuk = cu_of(nq, cuda), cu_of(nk, cuda)
    refs = [O.attention(q[cu[b]:cu[b + 1]], k[cuk[b]:cuk[b + 1]], v[cuk[b]:cuk[b + 1]], causal) for b in range(5)]
    for hint in (None, 1):
        out, lse = A.prompt_attention(q, k, v, cu, cu_seqlens_k=cuk, max_q=hint, causal=causal, return_lse=True)
        check(out, lse, refs, cu)
    none = A.prompt_attention(q, k[:0], v[:0], cu, cu_seqlens_k=torch.zeros_like(cuk), causal=causal)
    assert bool((none == 0).all())
    assert errors() == []


@pytest.mark.parametrize("dtype,d,hq,hkv,lens,causal", [(BF, 128, 8, 2, [1500, 700], True), (FP, 64, 6, 2, [1111], False),
                                                        (FP, 128, 5, 5, [900, 900], True), (BF, 64, 7, 1, [2043], True)])
def test_prompt_long(cuda, dtype, d, hq, hkv, lens, causal):
    T = sum(lens)
    q, k, v = (randn((T, h, d), dtype, cuda, 20 + i, 1.5) for i, h in enumerate((hq, hkv, hkv)))
    k[lens[0] // 2] *= 4
    cu = cu_of(lens, cuda)
    refs = [O.attention_fast(q[cu[b]:cu[b + 1]], k[cu[b]:cu[b + 1]], v[cu[b]:cu[b + 1]], causal) for b in range(len(lens))]
    out, lse = A.prompt_attention(q, k, v, cu, causal=causal, return_lse=True)
    check(out, lse, refs, cu)
    assert torch.equal(out, A.prompt_attention(q, k, v, cu, causal=causal))
    assert errors() == []


def test_prompt_layouts(cuda):
    """Operands without 16-byte rows or with other orders are taken as they are or copied, never misread."""
    base = randn((50, 6, 136), BF, cuda, 1)
    cu = cu_of([50], cuda)
    odd = base[:, :, 1:129]           # rows not 16-byte aligned
    q, k, v = odd[:, :4], odd[:, 4:5], odd[:, 5:]
    ref = O.attention(q, k, v, True)
    check(A.prompt_attention(q, k, v, cu), None, [ref], cu)
    inner = randn((50, 128, 6), BF, cuda, 2).transpose(1, 2)  # inner stride not 1
    q, k, v = inner[:, :4], inner[:, 4:5], inner[:, 5:]
    check(A.prompt_attention(q, k, v, cu), None, [O.attention(q, k, v, True)], cu)
    kx = randn((50, 1, 128), BF, cuda, 3).expand(50, 4, 128)  # one key head broadcast to all
    check(A.prompt_attention(q, kx, kx, cu), None, [O.attention(q, kx, kx, True)], cu)


def test_extreme_scores(cuda):
    """Scores near fp32's exp limits, equal scores, and one row whose scores all tie at a huge value."""
    n = 300
    q = torch.zeros(n, 4, 128, dtype=BF, device=cuda)
    k, v = torch.zeros(n, 1, 128, dtype=BF, device=cuda), randn((n, 1, 128), BF, cuda, 1)
    q[:, 0, 0], q[:, 1, 0], q[:, 2, 0] = 1e4, -1e4, 3e18
    k[:, 0, 0] = torch.linspace(-5, 5, n, device=cuda).to(BF)
    k[7, 0, 0] = 5.0
    cu = cu_of([n], cuda)
    for hint in (None, 1):
        out, lse = A.prompt_attention(q, k, v, cu, max_q=hint, return_lse=True)
        assert bool(torch.isfinite(out).all())
        check(out, lse, [O.attention(q, k, v, True)], cu)


def test_no_tokens(cuda):
    P = Paged(cuda, BF, 2, 128, 16, [5])
    e = torch.empty(0, 2, 128, dtype=BF, device=cuda)
    q = torch.empty(0, 8, 128, dtype=BF, device=cuda)
    cu = ints([0, 0], cuda)
    assert A.kv_append(P.cache, e, e, P.table, cu, P.lens, q=q).shape == q.shape
    assert A.paged_attention(q, P.cache, P.table, cu, P.lens).shape == q.shape
    out, lse = A.prompt_attention(q, e, e, cu, return_lse=True)
    assert out.shape == q.shape and lse.shape == (0, 8)
    assert A.prompt_attention(q, e, e, ints([0], cuda)).shape == q.shape


# ------------------------------------------------------------------------------------------------ refusals

def test_refusals(cuda):
    dev = cuda
    P = Paged(dev, BF, 2, 128, 16, [20])
    cu = ints([0, 1], dev)
    q, k = randn((1, 8, 128), BF, dev, 1), randn((1, 2, 128), BF, dev, 2)
    ok = dict(page_table=P.table, cu_seqlens=cu, kv_lens=P.lens)
    for exc, kw in ((TypeError, dict(page_table=P.table.long())), (TypeError, dict(kv_lens=P.lens.float())),
                    (ValueError, dict(cu_seqlens=ints([0, 1, 1], dev))), (ValueError, dict(page_table=P.table[0])),
                    (RuntimeError, dict(kv_lens=P.lens.cpu()))):
        with pytest.raises(exc):
            A.paged_attention(q, P.cache, **{**ok, **kw})
        with pytest.raises(exc):
            A.kv_append(P.cache, k, k, **{**ok, **kw})
    args = (P.cache, P.table, cu, P.lens)
    for exc, bad in ((TypeError, q.half()), (ValueError, q[..., :64]), (RuntimeError, q.cpu()), (ValueError, q[0]),
                     (RuntimeError, q[:, :7])):  # 7 query heads over 2 key heads
        with pytest.raises(exc):
            A.paged_attention(bad, *args)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError):
            A.paged_attention(q, *args, scale=scale)
    with pytest.raises(ValueError):
        A.paged_attention(q, *args, out=torch.empty(2, 8, 128, dtype=BF, device=dev))
    with pytest.raises(RuntimeError):
        A.paged_attention(randn((1, 130, 128), BF, dev, 1), *args)  # 65 query heads to a key head
    with pytest.raises(ValueError):
        A.kv_append(P.cache, k, k[:, :1], P.table, cu, P.lens)
    with pytest.raises(RuntimeError):
        A.kv_append(P.cache, k, k, P.table, cu, P.lens, cos_sin=A.rotation_table(30, 24, device=dev))
    with pytest.raises(TypeError):
        A.kv_append(P.cache, k, k, P.table, cu, P.lens, cos_sin=A.rotation_table(30, 32, device=dev).to(BF))
    with pytest.raises(ValueError):
        A.kv_append(P.cache, k, k, P.table, cu, P.lens, q_out=q)
    with pytest.raises(TypeError):
        A.prompt_attention(q.float(), q.float(), q.float(), cu)
    with pytest.raises(ValueError):
        A.prompt_attention(q, torch.cat([k, k]), torch.cat([k, k]), cu)
    with pytest.raises(RuntimeError):
        A.prompt_attention(*(randn((1, 2, 96), BF, dev, 1),) * 3, cu)
    for shape, dtype, exc in (((2, 12, 2, 128), BF, RuntimeError), ((2, 4, 2, 128), BF, RuntimeError),
                              ((2, 512, 2, 128), BF, RuntimeError), ((2, 16, 2, 80), BF, RuntimeError),
                              ((2, 16, 2, 128), torch.float32, TypeError)):
        with pytest.raises(exc):
            c = A.PagedKV(torch.zeros(shape, dtype=dtype, device=dev), torch.zeros(shape, dtype=dtype, device=dev))
            A.paged_attention(torch.zeros(1, 8, shape[-1], dtype=BF, device=dev), c, P.table, cu, P.lens)
    assert math.isfinite(float(A.paged_attention(q, *args).float().abs().max()))
    assert errors() == []
