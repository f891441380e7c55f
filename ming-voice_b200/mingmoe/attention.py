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
import struct

import torch

from . import _lib as L

_DTYPES = (torch.bfloat16, torch.float16)

# The argument structs of the C entry points, packed in one step: a call of a few microseconds is bounded by its host
# side, where filling a ctypes structure field by field takes several times as long.
_APPEND = struct.Struct("@10P10q8i")
_ATTN = struct.Struct("@10P9q10ifi")
assert _APPEND.size == C.sizeof(L.KVAppendArgs) and _ATTN.size == C.sizeof(L.AttentionArgs)


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
        self._ptr = C.addressof(c)

    @classmethod
    def empty(cls, num_pages, page_size, n_kv_heads, head_dim, dtype=torch.bfloat16, device="cuda"):
        shape = (num_pages, page_size, n_kv_heads, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))


def _rows(t, name, d, dtype, device):
    """A [T, heads, d] operand as the kernels take it (copied only where its layout has no 16-byte vectors), its
    shape and its strides."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != d:
        raise ValueError(f"{name} must be [T, heads, {d}], got {tuple(shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")
    st, sh, s1 = strides = t.stride()
    if s1 != 1 or (st | sh) & 7 or st < d or sh < d or t.data_ptr() & 15:
        t = t.contiguous()
        strides = t.stride()
    return t, shape, strides


def _out(t, name, like, shape, dtype, device):
    if t is None:
        t = torch.empty_like(like)
    elif t.shape != shape or t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {tuple(shape)} {dtype} on {device}")
    strides = t.stride()
    if strides[2] != 1:
        raise ValueError(f"{name} needs a unit inner stride")
    return t, strides


def _ints(t, name, device):
    """Shape of an int32 index tensor."""
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")
    shape = t.shape
    if len(shape) == 0 or (t.stride()[-1] != 1 and shape[-1] > 1):
        raise ValueError(f"{name} needs a unit inner stride")
    return shape


def _batch(page_table, cu_seqlens, kv_lens, device):
    """(sequences, columns and row stride of the page table)"""
    lens, cu, table = (_ints(kv_lens, "kv_lens", device), _ints(cu_seqlens, "cu_seqlens", device),
                       _ints(page_table, "page_table", device))
    B = lens[0]
    if len(lens) != 1 or len(cu) != 1 or cu[0] != B + 1 or len(table) != 2 or table[0] != B:
        raise ValueError(f"kv_lens [B], cu_seqlens [B + 1] and page_table [B, max_pages] do not agree: {tuple(lens)}, "
                         f"{tuple(cu)}, {tuple(table)}")
    return B, table[1], page_table.stride()[0]


def _call(fn, args, device, what):
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    ws = _ws.get((device.index, stream))
    if ws is None:
        buf = L.workspace("attention", L.lib().mv_attention_workspace_bytes(), device)
        ws = _ws[(device.index, stream)] = (buf.data_ptr(), buf.numel())
    rc = fn(args, ws[0], ws[1], stream)
    if rc:
        L.check(rc, what)


_ws: dict = {}  # (device, stream) -> address and size of the "attention" workspace (its size never changes)


def kv_append(cache, k, v, page_table, cu_seqlens, kv_lens, *, q=None, q_out=None, cos_sin=None, positions=None,
              interleaved=False):
    """Appends k, v [T, Hkv, D] of T packed new tokens to `cache`, rotating k (and q) by their positions on the way;
    returns the rotated q ([T, Hq, D]; None without q). kv_lens [B] are the lengths with the new tokens in them:
    new token i of n lands at position kv_lens[b] - n + i.

    cos_sin: fp32 [max_pos, rot_dim], a position's rot_dim / 2 cosines then its sines (rotation_table); None copies
    without rotating. rot_dim is a multiple of 16 up to D. Pairs are (i, i + rot_dim / 2), or (2i, 2i + 1) when
    `interleaved`. positions: int32 [T] rows of cos_sin, if not the cache positions. q_out may be q itself."""
    dev, d, dtype = cache.device, cache.head_dim, cache.dtype
    k, k_shape, ks = _rows(k, "k", d, dtype, dev)
    v, v_shape, vs = _rows(v, "v", d, dtype, dev)
    T = k_shape[0]
    if k_shape[1] != cache.n_kv_heads or v_shape != k_shape:
        raise ValueError(f"k and v must be [T, {cache.n_kv_heads}, {d}], got {tuple(k_shape)} / {tuple(v_shape)}")
    B, max_pages, pt_stride = _batch(page_table, cu_seqlens, kv_lens, dev)
    Hq = qp = qo = 0
    qs = qos = (0, 0)
    if q is not None:
        q, q_shape, qs = _rows(q, "q", d, dtype, dev)
        if q_shape[0] != T:
            raise ValueError("q and k have different numbers of tokens")
        Hq = q_shape[1]
        q_out, qos = _out(q_out, "q_out", q, q_shape, dtype, dev)
        qp, qo = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    cs = cs_stride = max_pos = rot = pos = 0
    if cos_sin is not None:
        if cos_sin.dtype != torch.float32 or cos_sin.ndim != 2 or cos_sin.device != dev:
            raise TypeError(f"cos_sin must be fp32 [max_pos, rot_dim] on {dev}")
        cs_stride, inner = cos_sin.stride()
        if inner != 1:
            raise ValueError("cos_sin needs a unit inner stride")
        cs, (max_pos, rot) = cos_sin.data_ptr(), cos_sin.shape
    if positions is not None:
        if tuple(_ints(positions, "positions", dev)) != (T,):
            raise ValueError(f"positions must be [{T}]")
        pos = positions.data_ptr()
    _call(L.lib().mv_kv_append,
          _APPEND.pack(cache._ptr, k.data_ptr(), v.data_ptr(), qp, qo, page_table.data_ptr(), cu_seqlens.data_ptr(),
                       kv_lens.data_ptr(), pos, cs, ks[0], ks[1], vs[0], vs[1], qs[0], qs[1], qos[0], qos[1],
                       pt_stride, cs_stride, T, B, Hq, max_pages, max_pos, rot, bool(interleaved), 0), dev, "kv_append")
    return q_out


def paged_attention(q, cache, page_table, cu_seqlens, kv_lens, *, max_q=None, scale=None, causal=True, out=None,
                    return_lse=False):
    """Attention of the packed new tokens q [T, Hq, D] over the cache, which holds their keys and values already
    (kv_append): out [T, Hq, D], and with return_lse also lse [T, Hq] fp32 (ln of the sum of exp scores; -inf for a
    row that sees no key, whose out is 0). max_q: the largest number of new tokens of a sequence, where the caller
    knows it; it only chooses the kernel. scale defaults to 1 / sqrt(D)."""
    dev, d, dtype = cache.device, cache.head_dim, cache.dtype
    q, shape, qs = _rows(q, "q", d, dtype, dev)
    T, Hq = shape[0], shape[1]
    B, max_pages, pt_stride = _batch(page_table, cu_seqlens, kv_lens, dev)
    out, os_ = _out(out, "out", q, shape, dtype, dev)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=dev) if return_lse else None
    _call(L.lib().mv_paged_attention,
          _ATTN.pack(cache._ptr, q.data_ptr(), 0, 0, out.data_ptr(), lse.data_ptr() if return_lse else 0,
                     cu_seqlens.data_ptr(), 0, page_table.data_ptr(), kv_lens.data_ptr(), qs[0], qs[1], 0, 0, 0, 0,
                     os_[0], os_[1], pt_stride, T, B, Hq, T if max_q is None else max_q, bool(causal), max_pages, 0, 0,
                     0, 0, 1.0 / math.sqrt(d) if scale is None else scale, 0), dev, "paged_attention")
    return (out, lse) if return_lse else out


def prompt_attention(q, k, v, cu_seqlens, *, cu_seqlens_k=None, max_q=None, scale=None, causal=True, out=None,
                     return_lse=False):
    """Attention over packed prompts: q [Tq, Hq, D], k, v [Tk, Hkv, D], sequence b's queries in rows
    cu_seqlens[b]:cu_seqlens[b + 1] and its keys in the same rows of k and v (or in cu_seqlens_k's). Causal masks
    align the ends: token i of n sees keys j <= n_keys - n + i. Returns as paged_attention."""
    if q.ndim != 3:
        raise ValueError("q, k, v must be [T, heads, D]")
    if not q.is_cuda:
        L.require_cuda(q)
    dev, d, dtype = q.device, q.shape[2], q.dtype
    if dtype not in _DTYPES:
        raise TypeError("prompt_attention: tensors must be bf16 or f16")
    q, shape, qs = _rows(q, "q", d, dtype, dev)
    k, k_shape, ks = _rows(k, "k", d, dtype, dev)
    v, v_shape, vs = _rows(v, "v", d, dtype, dev)
    if v_shape != k_shape:
        raise ValueError(f"k and v differ: {tuple(k_shape)} / {tuple(v_shape)}")
    T, Hq = shape[0], shape[1]
    cu = _ints(cu_seqlens, "cu_seqlens", dev)
    B = cu[0] - 1
    if len(cu) != 1 or B < 0:
        raise ValueError("cu_seqlens must be [B + 1]")
    cuk = 0
    if cu_seqlens_k is not None:
        if _ints(cu_seqlens_k, "cu_seqlens_k", dev) != cu:
            raise ValueError(f"cu_seqlens_k must be [{B + 1}]")
        cuk = cu_seqlens_k.data_ptr()
    elif k_shape[0] != T:
        raise ValueError("q and k have different numbers of tokens: cu_seqlens_k is needed")
    out, os_ = _out(out, "out", q, shape, dtype, dev)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=dev) if return_lse else None
    _call(L.lib().mv_prompt_attention,
          _ATTN.pack(0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0,
                     cu_seqlens.data_ptr(), cuk, 0, 0, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1], 0, T,
                     B, Hq, T if max_q is None else max_q, bool(causal), 0, k_shape[0], k_shape[1], d, L.dt(dtype),
                     1.0 / math.sqrt(d) if scale is None else scale, 0), dev, "prompt_attention")
    return (out, lse) if return_lse else out


def rotation_table(max_pos, rot_dim, base=10000.0, device="cuda"):
    """cos_sin of kv_append: fp32 [max_pos, rot_dim], angles pos * base ** (-2 i / rot_dim) taken in fp64."""
    inv = float(base) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    a = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv[None]
    return torch.cat([a.cos(), a.sin()], dim=1).float()
