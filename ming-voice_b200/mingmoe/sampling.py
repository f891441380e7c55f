"""Drawing tokens from logits (mv_sample; the filters' definitions in include/mingmoe.h).

    tokens = sample(logits, torch.rand(B, device="cuda"), temperature=0.8, top_k=50, top_p=0.95)

One pass over the logits [B, V], on the device, from random numbers that the caller draws: no host synchronisation, and a
captured graph draws anew at each replay from whatever its buffers hold.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from . import _serving


def _setting(v, name, dtype, b, dev):
    """(tensor or None, value): one number for all rows, or one for each."""
    if not isinstance(v, torch.Tensor):
        return None, v
    if tuple(v.shape) != (b,) or v.dtype != dtype:
        raise ValueError(f"{name} must be a number or {dtype} [{b}], got {v.dtype} {tuple(v.shape)}")
    if v.device != dev:
        raise RuntimeError(f"{name} is on {v.device}, expected {dev}")
    return v.contiguous(), 0


def sample(logits, u, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, return_logprob=False):
    """One token (int64 [B]) for each row of logits [B, V] (bf16 / f16 / f32, any row stride). u [B] fp32: uniform random
    numbers in [0, 1). temperature, top_p, min_p: numbers or fp32 [B]; top_k: a number or int32 [B]. Off: top_k 0, top_p 1,
    min_p 0. temperature 0 takes the largest logit (the lowest index of equal ones). With return_logprob also fp32 [B]: ln of the
    probability with which the token was drawn. A row with a NaN, or of -inf alone, gives -1 (and -inf)."""
    r = (_serving._module or _serving.host()).sample(logits, u, temperature, top_k, top_p, min_p, out, return_logprob)
    if type(r) is int:
        L.check(r, "sample")
    if r is not NotImplemented:
        return r
    L.require_cuda(logits, u)
    dev = logits.device
    if logits.dim() != 2:
        raise ValueError(f"logits must be [B, V], got {tuple(logits.shape)}")
    if logits.dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise TypeError(f"logits are {logits.dtype}: bf16, f16 or f32")
    b, v = logits.shape
    if tuple(u.shape) != (b,) or u.dtype != torch.float32:
        raise ValueError(f"u must be float32 [{b}], got {u.dtype} {tuple(u.shape)}")
    if u.device != dev:
        raise RuntimeError(f"u is on {u.device}, expected {dev}")
    if v > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    f32 = torch.float32
    t, tv = _setting(temperature, "temperature", f32, b, dev)
    k, kv = _setting(top_k, "top_k", torch.int32, b, dev)
    p, pv = _setting(top_p, "top_p", f32, b, dev)
    m, mv = _setting(min_p, "min_p", f32, b, dev)
    if out is None:
        out = torch.empty(b, dtype=torch.int64, device=dev)
    elif tuple(out.shape) != (b,) or out.dtype != torch.int64 or out.device != dev or not out.is_contiguous():
        raise ValueError(f"out must be contiguous int64 [{b}] on {dev}")
    u = u.contiguous()
    logprob = torch.empty(b, dtype=f32, device=dev) if return_logprob else None
    with torch.cuda.device(dev):
        a = L.SampleArgs(logits.data_ptr(), u.data_ptr(), *(x.data_ptr() if x is not None else 0 for x in (t, p, m, k)),
                         out.data_ptr(), logprob.data_ptr() if return_logprob else 0, 0, logits.stride(0),
                         0, tv, pv, mv, min(max(int(kv), 0), 0x7fffffff), b, v, L.dt(logits), 0)
        L.check(L.lib().mv_sample(C.byref(a), L.stream_ptr(dev)), "sample")
    return (out, logprob) if return_logprob else out
