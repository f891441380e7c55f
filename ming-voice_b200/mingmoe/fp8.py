"""Linear layers with 8-bit floating-point weights (mv_fp8_linear; formulas and rules in include/mingmoe.h).

    wq, ws = quantize_fp8_weight(w)                         # once: e4m3 [N, K], fp32 [ceil(N / 128), ceil(K / 128)]
    y = fp8_linear(x, wq, ws, residual=r)                   # x [..., K] bf16 / f16

Weights with one scale for each block of 128 x 128, as block-scaled checkpoints hold them (weight = wq * scale); activations
are rounded to e4m3 on the way in, with a power of two for each token and block of 128 columns. Products of the blocks are
added in fp32 and the result is rounded once. Any number of tokens, from one token's weight streaming to the tensor cores'
rate for prompts. A call runs on its tensors' device, on that device's current stream. Inference only.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from . import _serving

BLOCK = 128
_DTYPES = (torch.bfloat16, torch.float16)
E4M3 = torch.float8_e4m3fn


def _matrix(t, name):
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name} must be a matrix with a unit inner stride, got {tuple(t.shape)} / {t.stride()}")


def _header(dev):
    """The error word of a stream's calls, which the C++ module learns of too."""
    stream = torch.cuda.current_stream(dev).cuda_stream
    index = dev.index if dev.index is not None else torch.cuda.current_device()
    buf = _headers.get((index, stream))
    if buf is None:
        buf = _headers[(index, stream)] = L.workspace("fp8", 256, dev)
        _serving.host().workspace(index, stream, buf.data_ptr(), buf.numel())
    return buf


_headers: dict = {}


def quantize_fp8_weight(w):
    """w [N, K] bf16 / f16 / f32 -> (wq [N, K] e4m3, ws fp32): ws = max / 448 of each block of 128 x 128. The rows of wq start at
    whole 16 bytes, as fp8_linear takes them (wq is a view where K is not a multiple of 16)."""
    L.require_cuda(w)
    _matrix(w, "w")
    if w.dtype not in (*_DTYPES, torch.float32):
        raise TypeError(f"w is {w.dtype}: bf16, f16 or f32")
    n, k = w.shape
    q = torch.zeros(n, -(-k // 16) * 16, dtype=torch.uint8, device=w.device).view(E4M3)[:, :k]
    ws = torch.empty(-(-n // BLOCK), -(-k // BLOCK), dtype=torch.float32, device=w.device)
    with torch.cuda.device(w.device):
        L.check(L.lib().mv_quantize_fp8_weight(L.ptr(w), L.dt(w), w.stride(0), n, k, L.ptr(q), q.stride(0), L.ptr(ws),
                                               max(ws.stride(0), 1), L.stream_ptr(w.device)), "quantize_fp8_weight")
    return q, ws


def quantize_fp8(x):
    """x [T, K] bf16 / f16 / f32 -> (q [T, K] e4m3, scale [T, ceil(K / 128)] fp32), q * scale ~ x: what fp8_linear makes of its
    activations. scale is a view: a block's scales of all tokens lie side by side."""
    L.require_cuda(x)
    _matrix(x, "x")
    if x.dtype not in (*_DTYPES, torch.float32):
        raise TypeError(f"x is {x.dtype}: bf16, f16 or f32")
    t, k = x.shape
    blocks = -(-k // BLOCK)
    q = torch.empty(t, blocks * BLOCK, dtype=E4M3, device=x.device)
    scale = torch.empty(blocks, t, dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        L.check(L.lib().mv_quantize_fp8(L.ptr(x), L.dt(x), x.stride(0), t, k, L.ptr(q), blocks * BLOCK, L.ptr(scale), t,
                                        L.stream_ptr(x.device)), "quantize_fp8")
    return q[:, :k], scale.t()


def fp8_linear(x, wq, ws, *, residual=None, out=None, out_dtype=None):
    """x W^T (+ residual): x [..., K] bf16 / f16, wq [N, K] e4m3 whose rows start at whole 16 bytes, ws as above. The result has
    out_dtype (bf16, f16 or f32; that of x by default), and residual [..., N] the same type. `out` may be the residual."""
    r = (_serving._module or _serving.host()).fp8_linear(x, wq, ws, residual, out, out_dtype)
    if type(r) is int:
        L.check(r, "fp8_linear")
    if r is not NotImplemented:
        return r
    dev = x.device
    L.require_cuda(x, wq, ws, residual, out)
    if x.dtype not in _DTYPES:
        raise TypeError(f"x is {x.dtype}: bf16 or f16")
    if wq.dtype != E4M3 or ws.dtype != torch.float32:
        raise TypeError(f"wq must be float8_e4m3fn and ws float32, got {wq.dtype} / {ws.dtype}")
    _matrix(wq, "wq")
    _matrix(ws, "ws")
    n, k = wq.shape
    if x.dim() < 1 or x.shape[-1] != k or k < 1:
        raise ValueError(f"x {tuple(x.shape)} does not fit wq {tuple(wq.shape)}")
    if tuple(ws.shape) != (-(-n // BLOCK), -(-k // BLOCK)):
        raise ValueError(f"ws must be {(-(-n // BLOCK), -(-k // BLOCK))}, got {tuple(ws.shape)}")
    dtype = x.dtype if out_dtype is None else out_dtype
    if dtype not in (*_DTYPES, torch.float32):
        raise TypeError(f"out_dtype is {dtype}: bf16, f16 or f32")
    shape = (*x.shape[:-1], n)
    for name, t in (("residual", residual), ("out", out)):
        if t is not None and (tuple(t.shape) != shape or t.dtype != dtype):
            raise ValueError(f"{name} must be {shape} {dtype}, got {tuple(t.shape)} {t.dtype}")
    for t in (wq, ws, residual, out):
        if t is not None and t.device != dev:
            raise RuntimeError(f"tensors on {t.device} and {dev}")
    x2 = x.reshape(-1, k)
    if k > 1 and x2.stride(1) != 1:
        x2 = x2.contiguous()
    rows = x2.shape[0]
    r2 = None
    if residual is not None:
        r2 = residual.reshape(rows, n)
        if n > 1 and r2.stride(1) != 1:
            r2 = r2.contiguous()
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=dev)
    o2 = out.view(rows, n)
    if n > 1 and o2.stride(1) != 1:
        raise ValueError("out needs a unit inner stride")
    with torch.cuda.device(dev):
        lib = L.lib()
        ws_bytes = lib.mv_fp8_linear_scratch_bytes(rows, n, k)
        scratch = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        header = _header(dev)
        a = L.Fp8LinearArgs(x2.data_ptr(), wq.data_ptr(), ws.data_ptr(), r2.data_ptr() if r2 is not None else 0,
                            o2.data_ptr(), scratch.data_ptr(), x2.stride(0), wq.stride(0), ws.stride(0),
                            r2.stride(0) if r2 is not None else 0, o2.stride(0), ws_bytes, rows, n, k, L.dt(x.dtype),
                            L.dt(dtype), 0)
        L.check(lib.mv_fp8_linear(C.byref(a), L.ptr(header), header.numel(), L.stream_ptr(dev)), "fp8_linear")
    return out
