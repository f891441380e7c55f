"""Plain 64-bit restatements of the 8-bit products, of drawing tokens and of planning a step's pages (test infrastructure only;
product code never imports it). include/mingmoe.h has the definitions."""
import math

import torch

BLOCK = 128
# relative rounding error of the result types: half the spacing at 1
UNIT = {d: torch.finfo(d).eps / 2 for d in (torch.bfloat16, torch.float16, torch.float32)}


def round_e4m3(v):
    """fp64 values of magnitude up to 448 to the nearest e4m3 value, ties to even: 4 significant bits, spacing 2^-9 at least."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(v / step) * step


def quantize(x):
    """x [T, K] -> (values [T, K], scale [T, blocks]), fp64; a block that is not finite has scale NaN and values 0."""
    x = x.double()
    T, K = x.shape
    blocks = -(-K // BLOCK)
    q, scale = torch.zeros_like(x), torch.zeros(T, blocks, dtype=torch.float64, device=x.device)
    for b in range(blocks):
        part = x[:, b * BLOCK:(b + 1) * BLOCK]
        top = part.abs().amax(1)
        good = torch.isfinite(top)
        m, e = torch.frexp(torch.where(good, top, 1.0))
        e = torch.where(m > 0.875, e - 8, e - 9)  # the smallest with top <= 448 2^e
        e = torch.where(top == 0, -126, e).clamp(min=-126)
        s = torch.ldexp(torch.ones_like(top), e)
        scale[:, b] = torch.where(good, s, math.nan)
        q[:, b * BLOCK:(b + 1) * BLOCK] = torch.where(good[:, None], round_e4m3(part / s[:, None]), 0.0)
    return q, scale


def fp8_linear(x, wq, ws, residual=None):
    """(y, magnitudes): fp64 results, and the sums of the products' magnitudes."""
    q, scale = quantize(x)
    N, K = wq.shape
    w = wq.double()
    y = torch.zeros(x.shape[0], N, dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(y)
    rows = torch.arange(N, device=x.device) // BLOCK
    for b in range(scale.shape[1]):
        c = slice(b * BLOCK, (b + 1) * BLOCK)
        f = scale[:, b, None] * ws.double()[rows, b][None]
        y += f * (q[:, c] @ w[:, c].t())
        mag += f.abs() * (q[:, c].abs() @ w[:, c].abs().t())
    if residual is not None:
        y += residual.double()
        mag += residual.double().abs()
    return y, mag


def fp8_bound(y, mag, K, dtype):
    """What the promised arithmetic allows: products of e4m3 values are exact in fp32; up to 128 additions of a block, one per
    block and the residual's, each off by at most 2^-23 of the magnitudes so far (an fp32 unit: tensor cores may cut instead
    of rounding), two roundings of a block's factor and its product; one rounding to the result's type."""
    blocks = -(-K // BLOCK)
    tol = mag * (min(K, BLOCK) + blocks + 4) * 2.0 ** -23 + y.abs() * UNIT[dtype]
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # half the spacing below the smallest normal number
    return tol


def sample(logits, u, temperature, top_k, top_p, min_p):
    """One row: (token, log-probability), from Python numbers."""
    l = logits.double().cpu() + 0.0
    if l.numel() == 0 or torch.isnan(l).any() or l.max() == -math.inf:
        return -1, -math.inf
    V = l.numel()
    order = torch.argsort(-l, stable=True)  # equal logits: the lower index first
    m = l[order[0]]
    if not temperature > 0:
        return int(order[0]), 0.0
    # infinitely far below the first of the order is no weight, at an infinite temperature too (inf / inf has no value)
    z = torch.where(l == m, 0.0, torch.where((l - m).isinf(), -math.inf, (l - m) / temperature))
    w = torch.exp(z)[order]
    n = min(V, top_k) if top_k > 0 else V
    if top_p < 1:
        before = torch.cumsum(w[:n], 0) - w[:n]
        n = max(1, int((before < top_p * w[:n].sum()).sum()))
    if min_p > 0:
        n = max(1, int((w[:n] >= min_p).sum())) if min_p <= 1 else 1
    chosen = torch.sort(order[:n]).values
    mass = torch.exp(z[chosen])
    run = torch.cumsum(mass, 0)
    u = min(max(u, 0.0), 1.0 - 2.0 ** -24) if u == u else 0.0
    over = run > u * run[-1]
    i = int(over.int().argmax())
    return int(chosen[i]), float(torch.log(mass[i] / run[-1]))


class Pages:
    """A sequence state in Python lists: what plan_step and release_pages do to it."""

    def __init__(self, lens, pages, free, page_size):
        self.lens, self.pages, self.free, self.page = list(lens), [list(p) for p in pages], list(free), page_size

    def step(self, new, seqs, T, max_len, columns):
        """(cu, kv_lens, table, slots, positions, ok)"""
        limit = min(max_len, columns * self.page)
        known = [0 <= s < len(self.lens) for s in seqs]
        lens = [self.lens[s] if k else 0 for s, k in zip(seqs, known)]
        ok = all(known) and len(set(seqs)) == len(seqs) and all(n >= 0 and (n == 0 or l + n <= limit) for l, n in zip(lens, new))
        ok = ok and sum(new) <= T
        more = [-(-(l + n) // self.page) - -(-l // self.page) for l, n in zip(lens, new)] if ok else []
        ok = ok and sum(more) <= len(self.free)
        if not ok:
            table = [(self.pages[s] if k else []) for s, k in zip(seqs, known)]
            return [0] * (len(seqs) + 1), lens, table, [-1] * T, [0] * T, 0
        cu, slots, positions = [0], [], []
        for s, n, m in zip(seqs, new, more):
            self.pages[s] += [self.free.pop() for _ in range(m)]
            for p in range(self.lens[s], self.lens[s] + n):
                slots.append(self.pages[s][p // self.page] * self.page + p % self.page)
                positions.append(p)
            self.lens[s] += n
            cu.append(cu[-1] + n)
        rest = T - cu[-1]
        return (cu, [self.lens[s] for s in seqs], [list(self.pages[s]) for s in seqs], slots + [-1] * rest,
                positions + [0] * rest, 1)

    def release(self, seqs, room):
        known = all(0 <= s < len(self.lens) for s in seqs) and len(set(seqs)) == len(seqs)
        if not known or len(self.free) + sum(len(self.pages[s]) for s in seqs) > room:
            return 0
        for s in seqs:
            self.free += self.pages[s]
            self.pages[s], self.lens[s] = [], 0
        return 1
