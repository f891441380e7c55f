"""Measured cases of the operators between a decoder layer's output and the next step's cache slots: products with
8-bit floating-point weights (a scale for each block of 128), drawing tokens from logits, and planning a step's pages.

`run` computes them in plain torch operations where `own` is false, and through the public entry points of
`mingmoe.fp8`, `mingmoe.sampling` and `mingmoe.paging` where it is true.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"
BLOCK = 128


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one token through the query / key / value projection: launches and latency
        dict(name="proj_token", op="linear", dtype="bf16", out="bf16", m=1, n=2560, k=2048, residual=False),
        # the vocabulary head of one conversation: the weights' bandwidth
        dict(name="head_token", op="linear", dtype="bf16", out="f32", m=1, n=131072, k=2048, residual=False),
        # the head of a server batch; the last tile of rows and the last block of columns are ragged
        dict(name="head_batch", op="linear", dtype="f16", out="f32", m=61, n=100277, k=1500, residual=False),
        # the output projection of the packed prefill batch of this repository's benchmark (2043 tokens), residual added
        dict(name="proj_prompt", op="linear", dtype="bf16", out="bf16", m=2043, n=2048, k=2048, residual=True),
        # the shared expert's gate and up rows over long prompts: the tensor cores' rate
        dict(name="wide_prompt", op="linear", dtype="bf16", out="bf16", m=16001, n=5632, k=2048, residual=False),
        # one conversation's next token, all filters on: latency
        dict(name="draw_token", op="sample", dtype="f32", batch=1, vocab=131072, temp=0.8, top_k=50, top_p=0.95,
             min_p=0.02, flat=2.0, masked=False, mixed=False),
        # a server batch without filters but the floor min_p: one pass over all logits
        dict(name="draw_plain", op="sample", dtype="bf16", batch=192, vocab=131072, temp=1.0, top_k=0, top_p=1.0,
             min_p=0.01, flat=2.5, masked=False, mixed=False),
        # flat distributions, where the nucleus holds tens of thousands of tokens
        dict(name="draw_nucleus", op="sample", dtype="f32", batch=48, vocab=100277, temp=1.3, top_k=0, top_p=0.9,
             min_p=0.0, flat=1.2, masked=False, mixed=False),
        # every request has settings of its own, greedy ones among them, and a grammar masks most of the vocabulary
        dict(name="draw_mixed", op="sample", dtype="bf16", batch=128, vocab=50257, temp=0.7, top_k=200, top_p=0.9,
             min_p=0.05, flat=2.0, masked=True, mixed=True),
        # one new token for each running sequence of a server: few need a page
        dict(name="plan_tokens", op="plan", batch=61, max_seqs=61, max_len=16384, page=32, new=61, ctx=301000, rows=False,
             lens=1),
        # long prompts begin beside running sequences: many pages, a slot for each packed token
        dict(name="plan_prompts", op="plan", batch=9, max_seqs=64, max_len=20000, page=16, new=16001, ctx=5000, rows=True,
             lens=2),
        # a large server's step in an order of its own: the sequences' rows of the page table are gathered
        dict(name="plan_server", op="plan", batch=1000, max_seqs=1024, max_len=33000, page=64, new=2000, ctx=3000000,
             rows=True, lens=3),
    ]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, v))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "sample", "sample", "sample", "plan"])
    if op == "linear":
        k = rng.choice([_log_int(rng, 64, 4096), 128 * rng.randrange(1, 33), 2048])
        if rng.random() < 0.5:  # few tokens, up to a vocabulary of rows
            m, n = _log_int(rng, 1, 200), _log_int(rng, 100, 131072)
            while m * n * k > (1 << 35) or n * k > (1 << 28):
                n //= 2
        else:
            m, n = _log_int(rng, 1, 16001), _log_int(rng, 100, 6000)
            while m * n * k > 16001 * 5632 * 2048:
                m //= 2
        out = rng.choice(["bf16", "f16", "f32"])
        dtype = rng.choice(["bf16", "f16"])
        return dict(op=op, dtype=dtype, out=out, m=m, n=n, k=k, residual=out == dtype and rng.random() < 0.5)
    if op == "sample":
        vocab = _log_int(rng, 1000, 131072)
        batch = min(_log_int(rng, 1, 256), max(1, (128 * 50257) // vocab))
        return dict(op=op, dtype=rng.choice(["bf16", "f16", "f32"]), batch=batch, vocab=vocab,
                    temp=rng.choice([0.3, 0.7, 1.0, 1.0, 1.5]), top_k=rng.choice([0, 0, 1, _log_int(rng, 2, 2000)]),
                    top_p=rng.choice([1.0, 1.0, 0.95, 0.8, 0.3]), min_p=rng.choice([0.0, 0.0, 0.001, 0.05, 0.3]),
                    flat=rng.choice([0.5, 1.5, 2.0, 3.0]), masked=rng.random() < 0.3, mixed=rng.random() < 0.3)
    max_seqs = _log_int(rng, 1, 1024)
    batch = _log_int(rng, 1, max_seqs)
    max_len = rng.randrange(2000, 33000)
    rows = batch < max_seqs or rng.random() < 0.5
    return dict(op=op, batch=batch, max_seqs=max_seqs, max_len=max_len, page=rng.choice([8, 16, 32, 64, 128, 256]),
                new=min(batch * max_len // 8, max(batch, _log_int(rng, 1, 16001))),
                ctx=_log_int(rng, batch, batch * max_len // 8), rows=rows, lens=rng.randrange(1, 1 << 30))


def _split(total, n, most, rnd):
    """`total` tokens over n sequences of very different lengths, none above `most`."""
    w = [math.exp(rnd.gauss(0.0, 0.7)) for _ in range(n)]
    s = sum(w)
    lens = [min(most, int(total * x / s)) for x in w]
    short = total - sum(lens)
    for i in range(n):
        more = min(short, most - lens[i])
        lens[i] += more
        short -= more
    return lens


# ------------------------------------------------------------------------------------------------ inputs

def _ceil_div(a, b):
    return -(-a // b)


def _quantize_weight(w):
    """Blocks of 128 x 128 with the scale max / 448, as a checkpoint holds them; rows start at whole 16 bytes."""
    n, k = w.shape
    nb, kb = _ceil_div(n, BLOCK), _ceil_div(k, BLOCK)
    pad = torch.zeros(nb * BLOCK, kb * BLOCK, device=DEV)
    pad[:n, :k] = w
    tiles = pad.view(nb, BLOCK, kb, BLOCK)
    scale = tiles.abs().amax(dim=(1, 3)).clamp_(min=1e-30) / 448.0
    q = (tiles / scale[:, None, :, None]).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn)
    return q.view(nb * BLOCK, kb * BLOCK)[:n, :k], scale


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = random.Random(seed)
    st = dict(case=case)
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        x = torch.randn(m, k, generator=g, device=DEV)
        # a few columns of a trained model's hidden states are much larger than the rest
        loud = torch.randperm(k, generator=g, device=DEV)[:max(1, k // 200)]
        x[:, loud] *= 20.0
        st["x"] = x.to(DTYPES[case["dtype"]])
        st["wq"], st["ws"] = _quantize_weight(torch.randn(n, k, generator=g, device=DEV) * 0.02)
        if case["residual"]:
            st["residual"] = torch.randn(m, n, generator=g, device=DEV).to(DTYPES[case["dtype"]])
        return st
    if case["op"] == "sample":
        b, v = case["batch"], case["vocab"]
        logits = torch.randn(b, v, generator=g, device=DEV) * case["flat"]
        # the likely tokens stand out from the bulk, fewer and fewer of them
        peaks = torch.randint(0, v, (b, 40), generator=g, device=DEV)
        logits.scatter_add_(1, peaks, -2.0 * case["flat"] * torch.rand(b, 40, generator=g, device=DEV).log())
        if case["masked"]:
            logits[torch.rand(b, v, generator=g, device=DEV) < 0.8] = -math.inf
            logits[:, 0] = 0.0  # something is always allowed
        st["logits"] = logits.to(DTYPES[case["dtype"]])
        st["u"] = torch.rand(b, generator=g, device=DEV)

        def setting(value, others, dtype):
            pick = torch.tensor([rnd.choice([value, *others]) if case["mixed"] else value for _ in range(b)], dtype=dtype)
            return pick.to(DEV)

        st["temperature"] = setting(case["temp"], [0.0, 0.3, 1.0, 1.7], torch.float32)
        st["top_k"] = setting(case["top_k"], [0, 1, 40, v // 3], torch.int32)
        st["top_p"] = setting(case["top_p"], [1.0, 0.5, 0.99], torch.float32)
        st["min_p"] = setting(case["min_p"], [0.0, 0.1], torch.float32)
        return st
    lens_rnd = random.Random(case["lens"])
    s, b, page = case["max_seqs"], case["batch"], case["page"]
    columns = _ceil_div(case["max_len"], page)
    order = list(range(s))
    if case["rows"]:
        rnd.shuffle(order)
    order = order[:b]
    new = _split(case["new"], b, case["max_len"] // 2, lens_rnd)
    ctx = _split(case["ctx"], b, case["max_len"] // 2, lens_rnd)
    lens = [0] * s
    for i, c in zip(order, ctx):
        lens[i] = c
    owned = [_ceil_div(c, page) for c in lens]
    need = sum(_ceil_div(c + a, page) - _ceil_div(c, page) for a, c in zip(new, ctx))
    ids = torch.randperm(sum(owned) + need + 5, generator=g, device=DEV).int()
    used = torch.tensor(owned, device=DEV)
    cell = torch.arange(columns, device=DEV)[None] < used[:, None]
    st["pages"] = torch.zeros(s, columns, dtype=torch.int32, device=DEV)
    st["pages"][cell] = ids[:sum(owned)]
    st["free"] = torch.cat([ids[sum(owned):], torch.zeros(sum(owned), dtype=torch.int32, device=DEV)])
    st["n_free"] = torch.tensor([need + 5], dtype=torch.int32, device=DEV)
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    st["new"] = torch.tensor(new, dtype=torch.int32, device=DEV)
    st["seqs"] = torch.tensor(order, dtype=torch.int32, device=DEV) if case["rows"] else None
    # the counters after the step go to buffers of their own, so that the step can be planned again
    st["lens_out"], st["n_free_out"] = torch.empty_like(st["lens"]), torch.empty_like(st["n_free"])
    st["tokens"] = sum(new)
    return st


# ------------------------------------------------------------------------------------------------ one pass

def import_own(name):
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ming-voice_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import importlib
    return importlib.import_module("mingmoe." + name)


def run(st):
    case = st["case"]
    if case["op"] == "linear":
        if own:
            return import_own("fp8").fp8_linear(st["x"], st["wq"], st["ws"], residual=st.get("residual"),
                                                out_dtype=DTYPES[case["out"]])
        return _plain_linear(st)
    if case["op"] == "sample":
        if own:
            tokens, logprob = import_own("sampling").sample(
                st["logits"], st["u"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                min_p=st["min_p"], return_logprob=True)
            return dict(tokens=tokens, logprob=logprob)
        return _plain_sample(st)
    if own:
        step = import_own("paging").plan_step(st["new"], st["lens"], st["pages"], st["free"], st["n_free"],
                                              page_size=case["page"], num_tokens=st["tokens"], seqs=st["seqs"],
                                              lens_out=st["lens_out"], n_free_out=st["n_free_out"])
        return dict(cu_seqlens=step.cu_seqlens, kv_lens=step.kv_lens, page_table=step.page_table, slots=step.slots,
                    positions=step.positions, lens=st["lens_out"], n_free=st["n_free_out"])
    return _plain_plan(st)


def _plain_quantize(x):
    """Values that e4m3 holds and their blocks' powers of two, both fp32: x [m, k], k a multiple of 128."""
    tiles = x.view(x.shape[0], -1, BLOCK)
    fraction, exponent = torch.frexp(tiles.abs().amax(dim=2))
    e = torch.where(fraction <= 0.875, exponent - 9, exponent - 8).clamp_(min=-126)
    scale = torch.ldexp(torch.ones_like(fraction), e)
    return (tiles / scale[..., None]).to(torch.float8_e4m3fn).float(), scale


def _plain_linear(st):
    x, wq, ws = st["x"].float(), st["wq"], st["ws"]
    n, k = wq.shape
    pad = ws.shape[1] * BLOCK - k
    q, scale = _plain_quantize(torch.nn.functional.pad(x, (0, pad)))
    xd = (q * scale[..., None]).flatten(1)[:, :k]
    wd = wq.float() * ws.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = xd @ wd.t()
    if "residual" in st:
        y += st["residual"].float()
    return y.to(DTYPES[st["case"]["out"]])


def _plain_sample(st):
    """64 bits: a token next to the nucleus' border, or next to the drawn number, must not depend on a sum's rounding."""
    b, v = st["logits"].shape
    order_l, order_i = torch.sort(st["logits"], dim=1, descending=True, stable=True)
    greedy = st["temperature"] <= 0
    t = torch.where(greedy, 1.0, st["temperature"]).double()[:, None]
    x = order_l.double()
    w = ((x - x[:, :1]) / t).exp()
    rank = torch.arange(v, device=DEV)[None]
    k = torch.where(st["top_k"] > 0, st["top_k"], v)[:, None]
    w_k = torch.where(rank < k, w, 0.0)
    before = w_k.cumsum(1) - w_k
    p = st["top_p"].double()[:, None]
    kept = (rank < k) & ((before < p * w_k.sum(1, keepdim=True)) | (p >= 1)) & (w >= st["min_p"].double()[:, None])
    kept &= ~greedy[:, None]
    kept[:, 0] = True
    by_index = torch.zeros(b, v, dtype=torch.float64, device=DEV).scatter_(1, order_i, torch.where(kept, w, 0.0))
    run_sum = by_index.cumsum(1)
    total = run_sum[:, -1:]
    tokens = (run_sum > st["u"].double()[:, None] * total).int().argmax(1)
    logprob = (by_index.gather(1, tokens[:, None]) / total).log().squeeze(1)
    return dict(tokens=tokens, logprob=logprob.float())


def _plain_plan(st):
    page, t, seqs = st["case"]["page"], st["tokens"], st["seqs"]
    new, pages = st["new"], st["pages"]
    old = st["lens"] if seqs is None else st["lens"][seqs]
    kv_lens = old + new
    cu = torch.nn.functional.pad(new.cumsum(0), (1, 0)).int()
    have, need = (old + page - 1) // page, (kv_lens + page - 1) // page
    more = need - have
    first = more.cumsum(0) - more
    column = torch.arange(pages.shape[1], device=DEV)[None]
    taken = (column >= have[:, None]) & (column < need[:, None])
    at = st["n_free"] - 1 - first[:, None] - (column - have[:, None])
    table = pages if seqs is None else pages[seqs]
    table = torch.where(taken, st["free"][at.clamp(0, st["free"].shape[0] - 1)], table)
    table = torch.where(column < need[:, None], table, 0)
    if seqs is None:
        pages.copy_(table)
        st["lens_out"].copy_(kv_lens)
    else:
        pages[seqs] = table
        st["lens_out"].copy_(st["lens"])
        st["lens_out"][seqs] = kv_lens
    st["n_free_out"].copy_(st["n_free"] - more.sum())
    token = torch.arange(t, device=DEV)
    owner = torch.searchsorted(cu[1:].contiguous(), token, right=True)
    positions = old[owner] + token - cu[owner]
    slots = table[owner, positions // page].long() * page + positions % page
    return dict(cu_seqlens=cu, kv_lens=kv_lens, page_table=table, slots=slots, positions=positions.int(),
                lens=st["lens_out"], n_free=st["n_free_out"])


# ------------------------------------------------------------------------------------------------ definition in fp64

def _e4m3(v):
    """The nearest value with 4 significant bits and exponents of at least -6, ties to the even one, of fp64 values."""
    exponent = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3.0)
    return torch.round(v / step) * step


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        if m * n * k > 1 << 39:
            return None
        y = torch.zeros(m, n, dtype=torch.float64, device=DEV)
        for b in range(_ceil_div(k, BLOCK)):
            cols = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
            x = st["x"][:, cols].double()
            top = x.abs().amax(1, keepdim=True)
            e = torch.where(top > 0, torch.ceil(torch.log2(top / 448.0)), torch.full_like(top, -126.0)).clamp(min=-126.0)
            values = _e4m3(x * torch.exp2(-e)) * torch.exp2(e)
            for i in range(0, n, 128 * BLOCK):
                w = st["wq"][i:i + 128 * BLOCK, cols].double()
                row_scale = st["ws"][torch.arange(i, i + w.shape[0], device=DEV) // BLOCK, b].double()
                y[:, i:i + w.shape[0]] += values @ w.t() * row_scale
        if case["residual"]:
            y += st["residual"].double()
        return y
    if case["op"] == "plan":
        return None  # whole numbers only
    b, v = st["logits"].shape
    tokens = torch.empty(b, dtype=torch.int64, device=DEV)
    logprob = torch.empty(b, dtype=torch.float64, device=DEV)
    for r in range(b):
        l = st["logits"][r].double()
        # ranks by two keys: ascending index within equal logits
        order = torch.argsort(-l, stable=True)
        temp, k, p, floor = (float(st[key][r]) for key in ("temperature", "top_k", "top_p", "min_p"))
        if temp <= 0:
            tokens[r], logprob[r] = order[0], 0.0
            continue
        z = (l[order] - l[order[0]]) / temp
        n = v if k <= 0 else min(v, int(k))
        mass = torch.exp(z[:n])
        if p < 1:
            n = min(n, max(1, int(torch.searchsorted(torch.cumsum(mass, 0), p * mass.sum())) + 1))
        n = max(1, int((torch.exp(z[:n]) >= floor).sum()))
        chosen, _ = torch.sort(order[:n])
        share = torch.exp((l[chosen] - l[order[0]]) / temp)
        share = share / share.sum()
        i = int(torch.searchsorted(torch.cumsum(share, 0), st["u"][r].double(), right=True).clamp(max=n - 1))
        tokens[r], logprob[r] = chosen[i], torch.log(share[i])
    return dict(tokens=tokens, logprob=logprob)


# ------------------------------------------------------------------------------------------------ floor

def work(case):
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        nbytes = size[case["dtype"]] * m * k + n * k + 4 * _ceil_div(n, BLOCK) * _ceil_div(k, BLOCK)
        nbytes += size[case["out"]] * m * n * (2 if case["residual"] else 1)
        return dict(bytes=nbytes, flops=2 * m * n * k)
    if case["op"] == "sample":
        b, v = case["batch"], case["vocab"]
        return dict(bytes=size[case["dtype"]] * b * v + b * (5 * 4 + 8 + 4), flops=4 * b * v)
    rnd = random.Random(case["lens"])
    b, s, page = case["batch"], case["max_seqs"], case["page"]
    new = _split(case["new"], b, case["max_len"] // 2, rnd)
    ctx = _split(case["ctx"], b, case["max_len"] // 2, rnd)
    taken = sum(_ceil_div(a + c, page) - _ceil_div(c, page) for a, c in zip(new, ctx))
    held = sum(_ceil_div(a + c, page) for a, c in zip(new, ctx))
    gathered = held - taken + b * _ceil_div(case["max_len"], page) if case["rows"] else 0
    nbytes = 4 * (2 * b + s) + 4 * (b + 1 + b + s) + 8 * taken + 4 * gathered + 12 * sum(new)
    return dict(bytes=nbytes, flops=sum(new) + b)
