"""Plain 64-bit restatement of the attention entry points (test infrastructure only; product code never imports it).

Each function also returns what a rounding-error bound of its results needs, so that the tests' tolerances follow
from the arithmetic that include/mingmoe.h promises: fp32 scores, sums and outputs, weights rounded once to the
element type, results rounded once."""
import math

import torch

# relative rounding error of the element types: half the spacing at 1 (bf16 2^-8, f16 2^-11)
UNIT = {d: torch.finfo(d).eps / 2 for d in (torch.bfloat16, torch.float16)}


def gather(cache, pages, n):
    """The first n rows [n, Hkv, D] of a sequence whose page ids are `pages` in a [pages, page, Hkv, D] cache."""
    page = cache.shape[1]
    j = torch.arange(n, device=cache.device)
    return cache[pages.long()[j // page], j % page]


def attention(q, k, v, causal, scale=None):
    """One sequence: q [nq, Hq, D], k, v [n, Hkv, D] -> (out, lse, tol_out, tol_lse), all fp64."""
    nq, Hq, D = q.shape
    n, Hkv = k.shape[0], k.shape[1]
    u = UNIT[q.dtype]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.zeros(nq, Hq, D, dtype=torch.float64, device=q.device)
    lse = torch.full((nq, Hq), -math.inf, dtype=torch.float64, device=q.device)
    tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    see = torch.ones(nq, n, dtype=torch.bool, device=q.device)
    if causal:
        see = torch.arange(n, device=q.device)[None] <= (n - nq + torch.arange(nq, device=q.device))[:, None]
    for h in range(Hq):
        kh, vh = k[:, h // (Hq // Hkv)].double(), v[:, h // (Hq // Hkv)].double()
        qh = q[:, h].double()
        for i in range(nq):
            idx = see[i].nonzero().flatten()
            if idx.numel() == 0:
                continue
            s = (kh[idx] @ qh[i]) * scale
            m = s.max()
            p = (s - m).exp()
            z = p.sum()
            p = p / z
            out[i, h] = p @ vh[idx]
            lse[i, h] = m + z.log()
            # a score is a sum of D products in fp32 (at most D roundings of the sum of magnitudes), then scaled
            ds = (kh[idx].abs() @ qh[i].abs()).max() * scale * (D + 4) * 2.0 ** -24 + s.abs().max() * 2.0 ** -22
            spread = p @ vh[idx].abs()
            cnt = idx.numel()
            tol[i, h] = u * out[i, h].abs() + spread * (u + 2 * ds + (cnt + 64) * 2.0 ** -24 + 2.0 ** -20)
            if q.dtype == torch.float16:  # weights and results below the smallest normal number
                tol[i, h] += cnt * 2.0 ** -25 * vh[idx].abs().max() + 2.0 ** -25
            tol_lse[i, h] = ds + (cnt + 64) * 2.0 ** -24 + 2.0 ** -20 + lse[i, h].abs() * 2.0 ** -22
    return out, lse, tol, tol_lse


def attention_fast(q, k, v, causal, scale=None):
    """The same, a head at a time, for long sequences whose rows all see a key."""
    nq, Hq, D = q.shape
    n, Hkv = k.shape[0], k.shape[1]
    u = UNIT[q.dtype]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    res = [torch.empty(nq, Hq, D, dtype=torch.float64, device=q.device) for _ in range(2)]
    ls = [torch.empty(nq, Hq, dtype=torch.float64, device=q.device) for _ in range(2)]
    hide = None
    if causal:
        hide = torch.arange(n, device=q.device)[None] > (n - nq + torch.arange(nq, device=q.device))[:, None]
    for h in range(Hq):
        kh, vh, qh = k[:, h // (Hq // Hkv)].double(), v[:, h // (Hq // Hkv)].double(), q[:, h].double()
        s = qh @ kh.T * scale
        ds = (qh.abs() @ kh.abs().T).amax(1) * scale * (D + 4) * 2.0 ** -24 + s.abs().amax(1) * 2.0 ** -22
        if hide is not None:
            s = s.masked_fill(hide, -math.inf)
        lse = torch.logsumexp(s, 1)
        p = (s - lse[:, None]).exp()
        o = p @ vh
        res[0][:, h] = o
        res[1][:, h] = u * o.abs() + (p @ vh.abs()) * (u + 2 * ds + (n + 64) * 2.0 ** -24 + 2.0 ** -20)[:, None]
        if q.dtype == torch.float16:
            res[1][:, h] += n * 2.0 ** -25 * vh.abs().max() + 2.0 ** -25
        ls[0][:, h] = lse
        ls[1][:, h] = ds + (n + 64) * 2.0 ** -24 + 2.0 ** -20 + lse.abs() * 2.0 ** -22
    return res[0], ls[0], res[1], ls[1]


def rotate(x, cos_sin, pos, interleaved):
    """x [T, heads, D] by cos_sin [max_pos, rot] at rows pos -> (y, tol) in fp64."""
    x64 = x.double()
    rot = cos_sin.shape[1]
    half = rot // 2
    c, s = cos_sin[pos.long(), :half].double()[:, None], cos_sin[pos.long(), half:].double()[:, None]
    a_idx = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    b_idx = a_idx + (1 if interleaved else half)
    a, b = x64[..., a_idx], x64[..., b_idx]
    y, tol = x64.clone(), torch.zeros_like(x64)
    y[..., a_idx], y[..., b_idx] = a * c - b * s, b * c + a * s
    for i, (p, r) in ((a_idx, (a * c, b * s)), (b_idx, (b * c, a * s))):
        tol[..., i] = UNIT[x.dtype] * y[..., i].abs() + 2.0 ** -22 * (p.abs() + r.abs())
    if x.dtype == torch.float16:
        tol[..., :rot] += 2.0 ** -25  # half of the spacing below the smallest normal number
    return y, tol
