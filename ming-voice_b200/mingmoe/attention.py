"""Attention beside the MoE block: a paged key / value cache, attention of new tokens over it, attention over packed
prompts (mv_kv_append, mv_paged_attention, mv_prompt_attention; formulas and rules in include/mingmoe.h).

    cache = PagedKV(k_cache, v_cache)                       # [num_pages, page_size, Hkv, D], once
    q = kv_append(cache, k, v, page_table, cu_seqlens, kv_lens, q=q, cos_sin=table)
    o = paged_attention(q, cache, page_table, cu_seqlens, kv_lens, max_q=1)

Token tensors are packed [T, heads, D] (any row and head stride): sequence b owns rows cu_seqlens[b]:cu_seqlens[b + 1].
The calls read their arguments in C++ (csrc/attention_host.cpp) where these are as the kernels take them; the Python code
below it refuses what does not fit and copies what only needs another layout.

Lengths, bounds and page ids are int32 device tensors, read on the device: no call synchronises the host, and a
captured graph serves whatever lengths its buffers hold at the replay. A call runs on its tensors' device, on that device's
current stream, whichever device is current. Inference only: the results of inputs that require a gradient have no history.
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
        # what every call needs, read in one step
        self._key = (C.addressof(c), k.device, k.get_device(), k.dtype, self.n_kv_heads, self.head_dim)

    @classmethod
    def empty(cls, num_pages, page_size, n_kv_heads, head_dim, dtype=torch.bfloat16, device="cuda"):
        shape = (num_pages, page_size, n_kv_heads, head_dim)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))


def _fit(t, name, d, dtype, device):
    """A [T, heads, d] operand that the kernels cannot take as it is: refused, or copied where only its layout or address
    has no 16-byte vectors."""
    if t.ndim != 3 or t.shape[2] != d:
        raise ValueError(f"{name} must be [T, heads, {d}], got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")
    return t.clone(memory_format=torch.contiguous_format)


def _rows(t, name, d, dtype, device, index):
    """(operand, tokens, heads, token stride, head stride, address)"""
    p, s = t.data_ptr(), t.stride()
    if len(s) == 3:
        st, sh, s1 = s
        T, H, n = t.shape
        if (s1 == 1 and n == d and t.dtype is dtype and t.get_device() == index and not (st | sh) & 7 and st >= d
                and sh >= d and not p & 15):
            return t, T, H, st, sh, p
    t = _fit(t, name, d, dtype, device)
    st, sh, _ = t.stride()
    return t, t.shape[0], t.shape[1], st, sh, t.data_ptr()


def _out(t, name, like, device):
    """The result buffer: a new one, or the caller's. (buffer, token stride, head stride, address)"""
    if t is None:
        t = torch.empty_like(like)
    elif t.shape != like.shape or t.dtype != like.dtype or t.device != device:
        raise ValueError(f"{name} must be {tuple(like.shape)} {like.dtype} on {device}")
    st, sh, s1 = t.stride()
    if s1 != 1:
        raise ValueError(f"{name} needs a unit inner stride")
    return t, st, sh, t.data_ptr()


def _ints(t, name, device, index):
    """Shape of an int32 index tensor."""
    if t.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32")
    if t.get_device() != index:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")
    shape = t.shape
    if len(shape) == 0 or (shape[-1] > 1 and t.stride()[-1] != 1):
        raise ValueError(f"{name} needs a unit inner stride")
    return shape


def _batch(page_table, cu_seqlens, kv_lens, device, index):
    """(sequences, columns and row stride of the page table)"""
    lens, cu, table = (_ints(kv_lens, "kv_lens", device, index), _ints(cu_seqlens, "cu_seqlens", device, index),
                       _ints(page_table, "page_table", device, index))
    B = lens[0]
    if len(lens) != 1 or len(cu) != 1 or cu[0] != B + 1 or len(table) != 2 or table[0] != B:
        raise ValueError(f"kv_lens [B], cu_seqlens [B + 1] and page_table [B, max_pages] do not agree: {tuple(lens)}, "
                         f"{tuple(cu)}, {tuple(table)}")
    return B, table[1], page_table.stride()[0]


def _call(name, args, device, index):
    stream = torch._C._cuda_getCurrentRawStream(index)
    ws = _ws.get((index, stream))
    if ws is None:
        buf = L.workspace("attention", L.lib().mv_attention_workspace_bytes(), device)
        ws = _ws[(index, stream)] = (buf.data_ptr(), buf.numel())
        _host().workspace(index, stream, *ws)
    rc = getattr(L.lib(), name)(args, ws[0], ws[1], stream)
    if rc:
        L.check(rc, name)


def _host():
    """The C++ host module, bound to the loaded library's entry points."""
    global _module
    if _module is None:
        try:
            from . import _attention_host as m
        except ImportError as e:
            raise ImportError(f"mingmoe/_attention_host.so is missing or does not load ({e}): build it with "
                              "`python ming-voice_b200/mingmoe/build.py` (or __graft_entry__.build())") from e
        lib = L.lib()
        m.bind(*(C.cast(f, C.c_void_p).value for f in (lib.mv_kv_append, lib.mv_paged_attention,
                                                       lib.mv_prompt_attention)))
        _module = m
    return _module


_module = None
_ws: dict = {}  # (device, stream) -> address and size of the "attention" workspace (its size never changes)


def kv_append(cache, k, v, page_table, cu_seqlens, kv_lens, *, q=None, q_out=None, cos_sin=None, positions=None,
              interleaved=False):
    """Appends k, v [T, Hkv, D] of T packed new tokens to `cache`, rotating k (and q) by their positions on the way;
    returns the rotated q ([T, Hq, D]; None without q), without a gradient. kv_lens [B] are the lengths with the new tokens
    in them: new token i of n lands at position kv_lens[b] - n + i.

    cos_sin: fp32 [max_pos, rot_dim], a position's rot_dim / 2 cosines then its sines (rotation_table); None copies
    without rotating. rot_dim is a multiple of 16 up to D. Pairs are (i, i + rot_dim / 2), or (2i, 2i + 1) when
    `interleaved`. positions: int32 [T] rows of cos_sin, if not the cache positions. q_out may be q itself."""
    r = (_module or _host()).kv_append(cache._key[0], cache._key[2], k, v, page_table, cu_seqlens, kv_lens, q, q_out,
                                       cos_sin, positions, interleaved)
    if type(r) is int:
        L.check(r, "kv_append")
    if r is not NotImplemented:
        return r
    c_ptr, dev, index, dtype, n_kv, d = cache._key
    if torch._C._cuda_getDevice() != index:  # launches go to the current one
        with torch.cuda.device(index):
            return kv_append(cache, k, v, page_table, cu_seqlens, kv_lens, q=q, q_out=q_out, cos_sin=cos_sin,
                             positions=positions, interleaved=interleaved)
    k, T, H, k_st, k_sh, kp = _rows(k, "k", d, dtype, dev, index)
    v, Tv, Hv, v_st, v_sh, vp = _rows(v, "v", d, dtype, dev, index)
    if H != n_kv or Hv != n_kv or Tv != T:
        raise ValueError(f"k and v must be [T, {n_kv}, {d}], got {tuple(k.shape)} / {tuple(v.shape)}")
    B, max_pages, pt_stride = _batch(page_table, cu_seqlens, kv_lens, dev, index)
    Hq = q_st = q_sh = qp = qo_st = qo_sh = qop = 0
    if q is not None:
        q, Tq, Hq, q_st, q_sh, qp = _rows(q, "q", d, dtype, dev, index)
        if Tq != T:
            raise ValueError("q and k have different numbers of tokens")
        q_out, qo_st, qo_sh, qop = _out(q_out, "q_out", q, dev)
    elif q_out is not None:
        raise ValueError("q_out without q")
    cs = cs_stride = max_pos = rot = pos = 0
    if cos_sin is not None:
        if cos_sin.dtype is not torch.float32 or cos_sin.ndim != 2 or cos_sin.get_device() != index:
            raise TypeError(f"cos_sin must be fp32 [max_pos, rot_dim] on {dev}")
        cs_stride, inner = cos_sin.stride()
        if inner != 1:
            raise ValueError("cos_sin needs a unit inner stride")
        cs, (max_pos, rot) = cos_sin.data_ptr(), cos_sin.shape
    if positions is not None:
        if tuple(_ints(positions, "positions", dev, index)) != (T,):
            raise ValueError(f"positions must be [{T}]")
        pos = positions.data_ptr()
    _call("mv_kv_append",
          _APPEND.pack(c_ptr, kp, vp, qp, qop, page_table.data_ptr(), cu_seqlens.data_ptr(), kv_lens.data_ptr(), pos,
                       cs, k_st, k_sh, v_st, v_sh, q_st, q_sh, qo_st, qo_sh, pt_stride, cs_stride, T, B, Hq, max_pages,
                       max_pos, rot, bool(interleaved), 0), dev, index)
    return q_out


def paged_attention(q, cache, page_table, cu_seqlens, kv_lens, *, max_q=None, scale=None, causal=True, out=None,
                    return_lse=False):
    """Attention of the packed new tokens q [T, Hq, D] over the cache, which holds their keys and values already
    (kv_append): out [T, Hq, D], and with return_lse also lse [T, Hq] fp32 (ln of the sum of exp scores; -inf for a
    row that sees no key, whose out is 0), without a gradient. max_q: the largest number of new tokens of a sequence,
    where the caller knows it; it only chooses the kernel. scale defaults to 1 / sqrt(D)."""
    r = (_module or _host()).paged_attention(cache._key[0], cache._key[2], q, page_table, cu_seqlens, kv_lens, max_q,
                                             scale, causal, out, return_lse)
    if type(r) is int:
        L.check(r, "paged_attention")
    if r is not NotImplemented:
        return r
    c_ptr, dev, index, dtype, _, d = cache._key
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return paged_attention(q, cache, page_table, cu_seqlens, kv_lens, max_q=max_q, scale=scale, causal=causal,
                                   out=out, return_lse=return_lse)
    q, T, Hq, q_st, q_sh, qp = _rows(q, "q", d, dtype, dev, index)
    B, max_pages, pt_stride = _batch(page_table, cu_seqlens, kv_lens, dev, index)
    out, o_st, o_sh, op = _out(out, "out", q, dev)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=dev) if return_lse else None
    _call("mv_paged_attention",
          _ATTN.pack(c_ptr, qp, 0, 0, op, lse.data_ptr() if return_lse else 0, cu_seqlens.data_ptr(), 0,
                     page_table.data_ptr(), kv_lens.data_ptr(), q_st, q_sh, 0, 0, 0, 0, o_st, o_sh, pt_stride, T, B, Hq,
                     T if max_q is None else max_q, bool(causal), max_pages, 0, 0, 0, 0,
                     1.0 / math.sqrt(d) if scale is None else scale, 0), dev, index)
    return (out, lse) if return_lse else out


def prompt_attention(q, k, v, cu_seqlens, *, cu_seqlens_k=None, max_q=None, scale=None, causal=True, out=None,
                     return_lse=False):
    """Attention over packed prompts: q [Tq, Hq, D], k, v [Tk, Hkv, D], sequence b's queries in rows
    cu_seqlens[b]:cu_seqlens[b + 1] and its keys in the same rows of k and v (or in cu_seqlens_k's). Causal masks
    align the ends: token i of n sees keys j <= n_keys - n + i. Returns as paged_attention, without a gradient."""
    r = (_module or _host()).prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k, max_q, scale, causal, out, return_lse)
    if type(r) is int:
        L.check(r, "prompt_attention")
    if r is not NotImplemented:
        return r
    dtype, index, dev = q.dtype, q.get_device(), q.device
    if index < 0:
        L.require_cuda(q)
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return prompt_attention(q, k, v, cu_seqlens, cu_seqlens_k=cu_seqlens_k, max_q=max_q, scale=scale, causal=causal,
                                    out=out, return_lse=return_lse)
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError("prompt_attention: tensors must be bf16 or f16")
    if q.ndim != 3:
        raise ValueError("q, k, v must be [T, heads, D]")
    d = q.shape[2]
    q, T, Hq, q_st, q_sh, qp = _rows(q, "q", d, dtype, dev, index)
    k, Tk, Hkv, k_st, k_sh, kp = _rows(k, "k", d, dtype, dev, index)
    v, Tv, Hv, v_st, v_sh, vp = _rows(v, "v", d, dtype, dev, index)
    if Tv != Tk or Hv != Hkv:
        raise ValueError(f"k and v differ: {tuple(k.shape)} / {tuple(v.shape)}")
    cu = _ints(cu_seqlens, "cu_seqlens", dev, index)
    B = cu[0] - 1
    if len(cu) != 1 or B < 0:
        raise ValueError("cu_seqlens must be [B + 1]")
    cuk = 0
    if cu_seqlens_k is not None:
        if _ints(cu_seqlens_k, "cu_seqlens_k", dev, index) != cu:
            raise ValueError(f"cu_seqlens_k must be [{B + 1}]")
        cuk = cu_seqlens_k.data_ptr()
    elif Tk != T:
        raise ValueError("q and k have different numbers of tokens: cu_seqlens_k is needed")
    out, o_st, o_sh, op = _out(out, "out", q, dev)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=dev) if return_lse else None
    _call("mv_prompt_attention",
          _ATTN.pack(0, qp, kp, vp, op, lse.data_ptr() if return_lse else 0, cu_seqlens.data_ptr(), cuk, 0, 0, q_st, q_sh,
                     k_st, k_sh, v_st, v_sh, o_st, o_sh, 0, T, B, Hq, T if max_q is None else max_q, bool(causal), 0, Tk,
                     Hkv, d, L.dt(dtype), 1.0 / math.sqrt(d) if scale is None else scale, 0), dev, index)
    return (out, lse) if return_lse else out


def rotation_table(max_pos, rot_dim, base=10000.0, device="cuda"):
    """cos_sin of kv_append: fp32 [max_pos, rot_dim], angles pos * base ** (-2 i / rot_dim) taken in fp64."""
    inv = float(base) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    a = torch.arange(max_pos, dtype=torch.float64, device=device)[:, None] * inv[None]
    return torch.cat([a.cos(), a.sin()], dim=1).float()
