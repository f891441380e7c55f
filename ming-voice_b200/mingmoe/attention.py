"""Attention beside the MoE block: a paged key / value cache, attention of new tokens over it, attention over packed
prompts (mv_kv_append, mv_paged_attention, mv_prompt_attention; formulas and rules in include/mingmoe.h).

    cache = PagedKV(k_cache, v_cache)                       # [num_pages, page_size, Hkv, D], once
    q = kv_append(cache, k, v, page_table, cu_seqlens, kv_lens, q=q, cos_sin=table)
    o = paged_attention(q, cache, page_table, cu_seqlens, kv_lens, max_q=1)

Token tensors are packed [T, heads, D] (any row and head stride): sequence b owns rows cu_seqlens[b]:cu_seqlens[b + 1].
Lengths, bounds and page ids are int32 device tensors, read on the device: no call synchronises the host, and a
captured graph serves whatever lengths its buffers hold at the replay.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib as L

_DTYPES = (torch.bfloat16, torch.float16)


class PagedKV:
    """A paged cache: k, v [num_pages, page_size, n_kv_heads, head_dim], bf16 or f16, page_size a power of two in
    8..256, head_dim 64 or 128. Any page, token and head strides (a permuted [num_pages, n_kv_heads, page_size,
    head_dim] tensor is fine), inner stride 1. The tensors stay the caller's: the cache holds references to them."""

    def __init__(self, k, v):
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError(f"k and v must both be [pages, page_size, heads, head_dim], got {tuple(k.shape)} / {tuple(v.shape)}")
        if k.dtype != v.dtype or k.dtype not in _DTYPES:
            raise TypeError("the cache must be bf16 or f16, k and v alike")
        if k.stride(3) != 1 or v.stride(3) != 1:
            raise ValueError("the cache needs a unit inner stride")
        L.require_cuda(k, v)
        if k.device != v.device:
            raise ValueError("k and v are on different devices")
        self.k, self.v = k, v
        self.num_pages, self.page_size, self.n_kv_heads, self.head_dim = k.shape
        self.dtype, self.device = k.dtype, k.device
        c = L.PagedKV()
        c.k, c.v, c.dtype = k.data_ptr(), v.data_ptr(), L.dt(k)
        c.num_pages, c.page_size, c.n_kv_heads, c.head_dim = k.shape
        c.k_sp, c.k_st, c.k_sh = k.stride()[:3]
        c.v_sp, c.v_st, c.v_sh = v.stride()[:3]
        self._c = c
        self._ref = C.byref(c)

    @classmethod
    def empty(cls, num_pages, page_size, n_kv_heads, head_dim, dtype=torch.bfloat16, device="cuda"):
        shape = (num_pages, page_size, n_kv_heads, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))


def _rows(t, name, heads, d, dtype, device):
    """A [T, heads, d] operand as the kernels take it (copied only where its layout has no 16-byte vectors)."""
    if t.dim() != 3 or t.shape[2] != d or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} must be [T, {'heads' if heads is None else heads}, {d}], got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")
    st, sh, s1 = t.stride()
    if s1 != 1 or (st | sh) & 7 or st < d or sh < d or t.data_ptr() & 15:
        t = t.contiguous()
    return t


def _out(t, name, like_shape, d, dtype, device):
    if t is None:
        return torch.empty(like_shape, dtype=dtype, device=device)
    if t.shape != like_shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {tuple(like_shape)} {dtype} on {device}")
    if t.stride(2) != 1:
        raise ValueError(f"{name} needs a unit inner stride")
    return t


def _ints(t, name, shape, device):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    if t.dim() != len(shape) or any(n is not None and a != n for a, n in zip(t.shape, shape)):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError(f"{name} needs a unit inner stride")
    return t.data_ptr()


def _batch(page_table, cu_seqlens, kv_lens, device):
    B = kv_lens.shape[0] if kv_lens.dim() == 1 else -1
    lens = _ints(kv_lens, "kv_lens", (None,), device)
    cu = _ints(cu_seqlens, "cu_seqlens", (B + 1,), device)
    table = _ints(page_table, "page_table", (B, None), device)
    return B, cu, lens, table


def _workspace(device):
    global _ws_bytes
    if _ws_bytes == 0:
        _ws_bytes = L.lib().mv_attention_workspace_bytes()
    return L.workspace("attention", _ws_bytes, device)


_ws_bytes = 0


def kv_append(cache, k, v, page_table, cu_seqlens, kv_lens, *, q=None, q_out=None, cos_sin=None, positions=None,
              interleaved=False):
    """Appends k, v [T, Hkv, D] of T packed new tokens to `cache`, rotating k (and q) by their positions on the way;
    returns the rotated q ([T, Hq, D]; None without q). kv_lens [B] are the lengths with the new tokens in them:
    new token i of n lands at position kv_lens[b] - n + i.

    cos_sin: fp32 [max_pos, rot_dim], a position's rot_dim / 2 cosines then its sines (rotation_table); None copies
    without rotating. rot_dim is a multiple of 16 up to D. Pairs are (i, i + rot_dim / 2), or (2i, 2i + 1) when
    `interleaved`. positions: int32 [T] rows of cos_sin, if not the cache positions. q_out may be q itself."""
    dev, d, dtype = cache.device, cache.head_dim, cache.dtype
    k = _rows(k, "k", cache.n_kv_heads, d, dtype, dev)
    v = _rows(v, "v", cache.n_kv_heads, d, dtype, dev)
    T = k.shape[0]
    if v.shape[0] != T:
        raise ValueError("k and v have different numbers of tokens")
    B, cu, lens, table = _batch(page_table, cu_seqlens, kv_lens, dev)
    Hq = 0
    qp = qo = None
    qs = qos = (0, 0)
    if q is not None:
        q = _rows(q, "q", None, d, dtype, dev)
        if q.shape[0] != T:
            raise ValueError("q and k have different numbers of tokens")
        Hq = q.shape[1]
        q_out = _out(q_out, "q_out", q.shape, d, dtype, dev)
        qp, qo, qs, qos = q.data_ptr(), q_out.data_ptr(), q.stride(), q_out.stride()
    elif q_out is not None:
        raise ValueError("q_out without q")
    cs, cs_stride, max_pos, rot = None, 0, 0, 0
    if cos_sin is not None:
        if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or cos_sin.device != dev:
            raise TypeError(f"cos_sin must be fp32 [max_pos, rot_dim] on {dev}")
        if cos_sin.stride(1) != 1:
            raise ValueError("cos_sin needs a unit inner stride")
        cs, cs_stride, (max_pos, rot) = cos_sin.data_ptr(), cos_sin.stride(0), cos_sin.shape
        if max_pos == 1:
            cs_stride = rot
    pos = None if positions is None else _ints(positions, "positions", (T,), dev)
    ws = _workspace(dev)
    L.check(L.lib().mv_kv_append(cache._ref, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                                 v.stride(1), qp, qs[0], qs[1], Hq, qo, qos[0], qos[1], T, table,
                                 page_table.stride(0), page_table.shape[1], cu, lens, B, cs, cs_stride, max_pos, rot,
                                 interleaved, pos, ws.data_ptr(), ws.numel(),
                                 torch.cuda.current_stream(dev).cuda_stream), "kv_append")
    return q_out


def paged_attention(q, cache, page_table, cu_seqlens, kv_lens, *, max_q=None, scale=None, causal=True, out=None,
                    return_lse=False):
    """Attention of the packed new tokens q [T, Hq, D] over the cache, which holds their keys and values already
    (kv_append): out [T, Hq, D], and with return_lse also lse [T, Hq] fp32 (ln of the sum of exp scores; -inf for a
    row that sees no key, whose out is 0). max_q: the largest number of new tokens of a sequence, where the caller
    knows it; it only chooses the kernel. scale defaults to 1 / sqrt(D)."""
    dev, d, dtype = cache.device, cache.head_dim, cache.dtype
    q = _rows(q, "q", None, d, dtype, dev)
    T, Hq = q.shape[0], q.shape[1]
    B, cu, lens, table = _batch(page_table, cu_seqlens, kv_lens, dev)
    out = _out(out, "out", q.shape, d, dtype, dev)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=dev) if return_lse else None
    ws = _workspace(dev)
    L.check(L.lib().mv_paged_attention(cache._ref, q.data_ptr(), q.stride(0), q.stride(1), Hq, T, table,
                                       page_table.stride(0), page_table.shape[1], cu, lens, B,
                                       T if max_q is None else max_q, 1.0 / math.sqrt(d) if scale is None else scale,
                                       causal, out.data_ptr(), out.stride(0), out.stride(1),
                                       lse.data_ptr() if return_lse else None, ws.data_ptr(), ws.numel(),
                                       torch.cuda.current_stream(dev).cuda_stream), "paged_attention")
    return (out, lse) if return_lse else out


def prompt_attention(q, k, v, cu_seqlens, *, cu_seqlens_k=None, max_q=None, scale=None, causal=True, out=None,
                     return_lse=False):
    """Attention over packed prompts: q [Tq, Hq, D], k, v [Tk, Hkv, D], sequence b's queries in rows
    cu_seqlens[b]:cu_seqlens[b + 1] and its keys in the same rows of k and v (or in cu_seqlens_k's). Causal masks
    align the ends: token i of n sees keys j <= n_keys - n + i. Returns as paged_attention."""
    if q.dim() != 3 or k.dim() != 3:
        raise ValueError("q, k, v must be [T, heads, D]")
    L.require_cuda(q)
    dev, d, dtype = q.device, q.shape[2], q.dtype
    if dtype not in _DTYPES:
        raise TypeError("prompt_attention: tensors must be bf16 or f16")
    q = _rows(q, "q", None, d, dtype, dev)
    k = _rows(k, "k", None, d, dtype, dev)
    v = _rows(v, "v", k.shape[1], d, dtype, dev)
    if v.shape[0] != k.shape[0]:
        raise ValueError("k and v have different numbers of tokens")
    T, Hq = q.shape[0], q.shape[1]
    B = cu_seqlens.shape[0] - 1
    cu = _ints(cu_seqlens, "cu_seqlens", (None,), dev)
    if B < 0:
        raise ValueError("cu_seqlens needs at least one entry")
    cuk = None
    if cu_seqlens_k is not None:
        cuk = _ints(cu_seqlens_k, "cu_seqlens_k", (B + 1,), dev)
    elif k.shape[0] != T:
        raise ValueError("q and k have different numbers of tokens: cu_seqlens_k is needed")
    out = _out(out, "out", q.shape, d, dtype, dev)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=dev) if return_lse else None
    ws = _workspace(dev)
    L.check(L.lib().mv_prompt_attention(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                                        v.data_ptr(), v.stride(0), v.stride(1), L.dt(dtype), T, k.shape[0], Hq,
                                        k.shape[1], d, cu, cuk, B, T if max_q is None else max_q,
                                        1.0 / math.sqrt(d) if scale is None else scale, causal, out.data_ptr(),
                                        out.stride(0), out.stride(1), lse.data_ptr() if return_lse else None,
                                        ws.data_ptr(), ws.numel(), torch.cuda.current_stream(dev).cuda_stream),
            "prompt_attention")
    return (out, lse) if return_lse else out


def rotation_table(max_pos, rot_dim, base=10000.0, device="cuda"):
    """cos_sin of kv_append: fp32 [max_pos, rot_dim], angles pos * base ** (-2 i / rot_dim) taken in fp64."""
    inv = float(base) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    a = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv[None]
    return torch.cat([a.cos(), a.sin()], dim=1).float()
