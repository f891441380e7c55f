"""Measured cases of the attention operators: appending to a paged cache with the position rotation, attention of new
tokens over the paged cache, and attention over packed prompts.

`run` computes them in plain torch operations (fp32, rounded once) where `own` is false, and through the public
entry points of `mingmoe.attention` where it is true. Sequence lengths of a case are drawn from its own `lens` number,
so a case stays a dict of plain values.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one token of one conversation: the smallest call of a decode step, all launch and latency
        dict(name="append_token", op="append", dtype="bf16", hq=16, hkv=4, d=128, page=16, batch=1, new=1, ctx=700,
             rot=128, interleaved=False, lens=1),
        # one decode step of a full server batch, half of each head rotated, interleaved pairs
        dict(name="append_batch", op="append", dtype="f16", hq=14, hkv=2, d=64, page=32, batch=192, new=192,
             ctx=100000, rot=32, interleaved=True, lens=2),
        # a packed batch of long prompts going into the cache
        dict(name="append_prompts", op="append", dtype="bf16", hq=16, hkv=4, d=128, page=64, batch=9, new=16001,
             ctx=5000, rot=128, interleaved=False, lens=3),
        # decode of one short conversation: latency
        dict(name="decode_short", op="paged", dtype="bf16", hq=16, hkv=4, d=128, page=16, batch=1, new=1, ctx=811,
             causal=True, lse=False, lens=4),
        # decode of one very long conversation: the cache has to be split over the whole card
        dict(name="decode_long", op="paged", dtype="bf16", hq=12, hkv=2, d=128, page=64, batch=1, new=1, ctx=130500,
             causal=True, lse=True, lens=5),
        # decode step of a server batch with conversations of very different lengths: the cache's bandwidth
        dict(name="decode_batch", op="paged", dtype="f16", hq=16, hkv=4, d=128, page=32, batch=61, new=61, ctx=301000,
             causal=True, lse=False, lens=6),
        # a few tokens per sequence checked at once (drafted tokens), small heads, 7 query heads to a key head
        dict(name="drafts", op="paged", dtype="f16", hq=14, hkv=2, d=64, page=16, batch=24, new=120, ctx=60000,
             causal=True, lse=False, lens=7),
        # chunked prefill: new pieces of four conversations over what is in the cache already
        dict(name="chunk", op="paged", dtype="bf16", hq=16, hkv=4, d=128, page=64, batch=4, new=2043, ctx=45000,
             causal=True, lse=True, lens=8),
        # one spoken sentence as a prompt
        dict(name="prompt_short", op="prompt", dtype="bf16", hq=16, hkv=4, d=128, batch=1, new=37, causal=True,
             lse=False, lens=9),
        # the ragged packed prefill batch of this repository's benchmark (2043 tokens)
        dict(name="prompt_packed", op="prompt", dtype="bf16", hq=16, hkv=4, d=128, batch=8, new=2043, causal=True,
             lse=True, lens=10),
        # an encoder's pass over audio frames: every frame sees every other, small heads, one key head per query head
        dict(name="prompt_full", op="prompt", dtype="f16", hq=16, hkv=16, d=64, batch=5, new=9999, causal=False,
             lse=False, lens=11),
        # long documents
        dict(name="prompt_long", op="prompt", dtype="bf16", hq=16, hkv=4, d=128, batch=2, new=20000, causal=True,
             lse=False, lens=12),
    ]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    v = min(hi, max(lo, v))
    return v + 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(["append", "paged", "paged", "paged", "prompt", "prompt"])
    d = rng.choice([64, 128, 128])
    hq, hkv = rng.choice([(16, 4), (16, 16), (12, 2), (14, 2), (16, 2), (16, 1), (8, 8), (15, 5)])
    c = dict(op=op, dtype=rng.choice(["bf16", "f16"]), hq=hq, hkv=hkv, d=d)
    lens = rng.randrange(1, 1 << 30)
    if op == "append":
        batch = _log_int(rng, 1, 192)
        new = max(batch, _log_int(rng, 1, 16001))
        c.update(page=rng.choice([16, 32, 64, 128]), batch=batch, new=new, ctx=_log_int(rng, batch, 100000),
                 rot=rng.choice([0, d // 2, d, d]), interleaved=rng.random() < 0.5, lens=lens)
    elif op == "paged":
        kind = rng.choice(["decode", "decode", "drafts", "chunk"])
        if kind == "chunk":
            batch = _log_int(rng, 1, 6)
            new = max(batch, _log_int(rng, 17, 2043))
            ctx = _log_int(rng, 100, 45000)
        else:
            batch = _log_int(rng, 1, 61)
            new = batch if kind == "decode" else batch * rng.randrange(2, 8)
            ctx = max(batch, _log_int(rng, 100, 2400000 // (hkv * d)))
        c.update(page=rng.choice([16, 32, 64, 128]), batch=batch, new=new, ctx=ctx, causal=rng.random() < 0.9,
                 lse=rng.random() < 0.3, lens=lens)
    else:
        batch = _log_int(rng, 1, 16)
        c.update(batch=batch, new=max(batch, _log_int(rng, 17, 11001)), causal=rng.random() < 0.75,
                 lse=rng.random() < 0.3, lens=lens)
    return c


def _split(total, n, rnd):
    """`total` tokens over n sequences of very different lengths, at least one each."""
    w = [math.exp(rnd.gauss(0.0, 0.7)) for _ in range(n)]
    s = sum(w)
    lens = [1 + int((total - n) * x / s) for x in w]
    lens[rnd.randrange(n)] += total - sum(lens)
    return [v + 1 if v == 3072 else v for v in lens]


def _lens(case):
    """(new tokens, tokens already in the cache) of every sequence."""
    rnd = random.Random(case["lens"])
    new = _split(case["new"], case["batch"], rnd)
    if case["op"] == "prompt":
        return new, [0] * len(new)
    ctx = _split(max(case["ctx"], case["batch"]), case["batch"], rnd)
    return new, [c + 2 if a + c == 3072 or c + 2 == 3072 else c for a, c in zip(new, ctx)]


# ------------------------------------------------------------------------------------------------ inputs

def _cu(lens, device=DEV):
    cu = [0]
    for v in lens:
        cu.append(cu[-1] + v)
    return torch.tensor(cu, dtype=torch.int32, device=device)


def _table(max_pos, rot):
    """cos (first half of a row) and sin (second half) of the positions' angles, fp32."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=DEV) / rot)
    a = torch.arange(max_pos, dtype=torch.float64, device=DEV)[:, None] * inv[None]
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def _randn(g, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).mul_(scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = random.Random(seed)
    dtype = DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    new, ctx = _lens(case)
    T = sum(new)
    st = dict(case=case, new=new, ctx=ctx, cu=_cu(new))
    # one projection writes a token's query, key and value heads side by side: the operators get strided views of it
    qkv = _randn(g, (T, hq + 2 * hkv, d), dtype)
    qkv[:, :hq] *= 2.0  # trained queries give logits well away from uniform
    st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    if case["op"] == "prompt":
        if own:
            import_attention()
        return st
    page = case["page"]
    total = [a + b for a, b in zip(new, ctx)]
    npages = [-(-n // page) for n in total]
    n_all = sum(npages) + 3  # the pool holds a few pages nobody owns
    order = list(range(n_all))
    rnd.shuffle(order)
    table, at = [], 0
    for n in npages:
        table.append(order[at:at + n] + [0] * (max(npages) - n))
        at += n
    st["page_table"] = torch.tensor(table, dtype=torch.int32, device=DEV)
    st["kv_lens"] = torch.tensor(total, dtype=torch.int32, device=DEV)
    # pages are recycled: slots that hold no token of this batch hold older values
    st["k_cache"] = _randn(g, (n_all, page, hkv, d), dtype)
    st["v_cache"] = _randn(g, (n_all, page, hkv, d), dtype)
    if case["op"] == "append" and case["rot"]:
        st["cos_sin"] = _table(max(total), case["rot"])
    if own:
        st["cache"] = import_attention().PagedKV(st["k_cache"], st["v_cache"])
    return st


def import_attention():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ming-voice_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from mingmoe import attention
    return attention


# ------------------------------------------------------------------------------------------------ one pass

def run(st):
    case = st["case"]
    if own:
        A = import_attention()
        if case["op"] == "append":
            q = A.kv_append(st["cache"], st["k"], st["v"], st["page_table"], st["cu"], st["kv_lens"], q=st["q"],
                            cos_sin=st.get("cos_sin"), interleaved=case["interleaved"])
            return dict(q=q, k_cache=st["k_cache"], v_cache=st["v_cache"])
        if case["op"] == "paged":
            r = A.paged_attention(st["q"], st["cache"], st["page_table"], st["cu"], st["kv_lens"],
                                  max_q=max(st["new"]), causal=case["causal"], return_lse=case["lse"])
        else:
            r = A.prompt_attention(st["q"], st["k"], st["v"], st["cu"], max_q=max(st["new"]), causal=case["causal"],
                                   return_lse=case["lse"])
        return dict(out=r[0], lse=r[1]) if case["lse"] else dict(out=r)
    if case["op"] == "append":
        return _plain_append(st)
    return _plain_attention(st)


def _plain_rotate(x, cos, sin, interleaved):
    """x [T, heads, d] fp32, cos / sin [T, rot / 2]."""
    rot = 2 * cos.shape[1]
    c, s = cos[:, None], sin[:, None]
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        r = torch.stack([a * c - b * s, b * c + a * s], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        r = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    return torch.cat([r, x[..., rot:]], dim=-1)


def _plain_append(st):
    case, cu, k_cache, v_cache = st["case"], st["cu"], st["k_cache"], st["v_cache"]
    T, page, dtype = st["q"].shape[0], case["page"], st["q"].dtype
    tok = torch.arange(T, device=DEV)
    seq = torch.searchsorted(cu[1:].contiguous(), tok, right=True)
    start = st["kv_lens"] - (cu[1:] - cu[:-1])
    pos = (start[seq] + tok - cu[seq]).long()
    slot = st["page_table"][seq, pos // page].long() * page + pos % page
    q, k = st["q"].float(), st["k"].float()
    if case["rot"]:
        cs = st["cos_sin"][pos]
        cos, sin = cs[:, :case["rot"] // 2], cs[:, case["rot"] // 2:]
        q = _plain_rotate(q, cos, sin, case["interleaved"])
        k = _plain_rotate(k, cos, sin, case["interleaved"])
    k_cache.view(-1, *k_cache.shape[2:])[slot] = k.to(dtype)
    v_cache.view(-1, *v_cache.shape[2:])[slot] = st["v"]
    return dict(q=q.to(dtype), k_cache=k_cache, v_cache=v_cache)


def _plain_attention(st):
    case = st["case"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    G, scale, dtype = hq // hkv, 1.0 / math.sqrt(d), st["q"].dtype
    outs, lses, at = [], [], 0
    for b, (nq, nc) in enumerate(zip(st["new"], st["ctx"])):
        n = nq + nc
        if case["op"] == "prompt":
            k, v = st["k"][at:at + nq], st["v"][at:at + nq]
        else:
            pages = st["page_table"][b, :-(-n // case["page"])]
            k = st["k_cache"][pages].flatten(0, 1)[:n]
            v = st["v_cache"][pages].flatten(0, 1)[:n]
        k = k.float().permute(1, 2, 0)                                    # [hkv, d, n]
        v = v.float().transpose(0, 1)                                     # [hkv, n, d]
        step = max(1, min(nq, (1 << 28) // (hq * n)))                     # bounds the score matrix
        for i0 in range(0, nq, step):
            i1 = min(nq, i0 + step)
            q = st["q"][at + i0:at + i1].float().view(i1 - i0, hkv, G, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
            s = torch.matmul(q, k).mul_(scale).view(hkv, G, i1 - i0, n)
            if case["causal"]:
                row = torch.arange(n - nq + i0, n - nq + i1, device=DEV)
                s.masked_fill_(torch.arange(n, device=DEV)[None] > row[:, None], float("-inf"))
            m = s.amax(dim=-1, keepdim=True)
            p = s.sub_(m).exp_()
            l = p.sum(dim=-1, keepdim=True)
            o = torch.matmul(p.view(hkv, -1, n), v).view(hkv, G, i1 - i0, d) / l
            outs.append(o.permute(2, 0, 1, 3).reshape(i1 - i0, hq, d).to(dtype))
            if case["lse"]:
                lses.append((m + l.log()).squeeze(-1).permute(2, 0, 1).reshape(i1 - i0, hq))
        at += nq
    out = dict(out=torch.cat(outs))
    if case["lse"]:
        out["lse"] = torch.cat(lses)
    return out


# ------------------------------------------------------------------------------------------------ definition in fp64

def exact(case, seed):
    st = prepare(case, seed)
    new, ctx, hq, hkv, d = st["new"], st["ctx"], case["hq"], case["hkv"], case["d"]
    group = hq // hkv
    if case["op"] == "append":
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        qo = torch.empty(sum(new), hq, d, dtype=torch.float64, device=DEV)
        at = 0
        for b in range(len(new)):
            p = torch.arange(ctx[b], ctx[b] + new[b], device=DEV)
            rows = st["page_table"][b].long()[torch.div(p, case["page"], rounding_mode="floor")]
            cols = torch.remainder(p, case["page"])
            parts = []
            for x in (st["q"], st["k"]):
                x = x[at:at + new[b]].double()
                if case["rot"]:
                    half = case["rot"] // 2
                    # each pair as a complex number times exp(i angle), the angle's cos and sin from the call's table
                    w = torch.complex(st["cos_sin"][p, :half].double(), st["cos_sin"][p, half:].double())[:, None]
                    y = x.clone()
                    if case["interleaved"]:
                        z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) * w
                        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = z.real, z.imag
                    else:
                        z = torch.complex(x[..., :half], x[..., half:2 * half]) * w
                        y[..., :half], y[..., half:2 * half] = z.real, z.imag
                    x = y
                parts.append(x)
            qo[at:at + new[b]] = parts[0]
            kc[rows, cols] = parts[1]
            vc[rows, cols] = st["v"][at:at + new[b]].double()
            at += new[b]
        return dict(q=qo, k_cache=kc, v_cache=vc)
    out = torch.empty(sum(new), hq, d, dtype=torch.float64, device=DEV)
    lse = torch.empty(sum(new), hq, dtype=torch.float64, device=DEV)
    at = 0
    for b in range(len(new)):
        n = new[b] + ctx[b]
        j = torch.arange(n, device=DEV)
        if case["op"] == "paged":
            rows = st["page_table"][b].long()[torch.div(j, case["page"], rounding_mode="floor")]
            keys, vals = (st[c][rows, torch.remainder(j, case["page"])].double() for c in ("k_cache", "v_cache"))
        else:
            keys, vals = st["k"][at:at + n].double(), st["v"][at:at + n].double()
        step = max(1, (1 << 26) // n)
        for h in range(hq):
            kh, vh = keys[:, h // group], vals[:, h // group]
            for i0 in range(0, new[b], step):
                i = torch.arange(i0, min(new[b], i0 + step), device=DEV)
                s = torch.einsum("id,jd->ij", st["q"][at + i, h].double(), kh) * d ** -0.5
                if case["causal"]:
                    s = torch.where(j[None, :] <= ctx[b] + i[:, None], s, torch.full_like(s, -math.inf))
                z = torch.logsumexp(s, dim=1)
                lse[at + i, h] = z
                out[at + i, h] = torch.exp(s - z[:, None]) @ vh
        at += new[b]
    return dict(out=out, lse=lse) if case["lse"] else dict(out=out)


# ------------------------------------------------------------------------------------------------ floor

def work(case):
    new, ctx = _lens(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    T = sum(new)
    ints = 4 * (2 * len(new) + 1)
    if case["op"] == "append":
        pages = sum(-(-(a + b) // case["page"]) - b // case["page"] for a, b in zip(new, ctx))
        values = T * (hq + 2 * hkv) * d
        table = T * case["rot"] * 4
        return dict(bytes=4 * values + table + 4 * pages + ints, flops=3 * T * (hq + hkv) * case["rot"])
    pairs, pages = 0, 0
    for a, b in zip(new, ctx):
        n = a + b
        pairs += a * n - (a * (a - 1) // 2 if case["causal"] else 0)
        pages += -(-n // case["page"]) if case["op"] == "paged" else 0
    keys = T + sum(ctx)
    nbytes = 2 * d * (2 * T * hq + 2 * keys * hkv) + 4 * pages + ints + (4 * T * hq if case["lse"] else 0)
    return dict(bytes=nbytes, flops=4 * d * hq * pairs)
