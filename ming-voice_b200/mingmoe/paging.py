"""Pages of the next step, on the device (mv_plan_step, mv_release_pages; rules in include/mingmoe.h).

DeviceSequences is layer.Sequences with its state on the GPU: a step is planned by a kernel from tensors, so a decode loop
needs nothing from the host, and a captured step plans anew at each replay. plan_step and release_pages are the operators by
themselves, on the caller's own state:

    lens [S] int32      tokens of each sequence in the cache
    pages [S, P] int32  their page ids (any row stride): the first ceil(lens / page_size) of a row
    free [F] int32      a stack of free page ids: the first n_free[0], the last of them on top
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L
from . import _serving
from .attention import PagedKV


class Step:
    """One step's packed tokens, all on the device: cu_seqlens [B + 1], kv_lens [B] (with the new tokens), page_table [B, P],
    slots [T] int64 (rows of the cache as [num_pages * page_size, ...]; -1 behind the last token), positions [T], and ok [1]:
    0 where the step was refused. max_q and prompts are what the host knows, as in layer.Batch."""

    __slots__ = ("cu_seqlens", "kv_lens", "page_table", "slots", "positions", "ok", "max_q", "prompts")

    def __init__(self, cu_seqlens, kv_lens, page_table, slots, positions, ok, max_q=None, prompts=False):
        self.cu_seqlens, self.kv_lens, self.page_table = cu_seqlens, kv_lens, page_table
        self.slots, self.positions, self.ok = slots, positions, ok
        self.max_q, self.prompts = max_q, prompts


def _ints(t, name, dev, shape=None, contiguous=True):
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32")
    if t.device != dev:
        raise RuntimeError(f"{name} is on {t.device}, expected {dev}")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _state(lens, pages, free, n_free, lens_out, n_free_out, page_size):
    """The state's part of the argument struct."""
    L.require_cuda(lens, pages, free, n_free, lens_out, n_free_out)
    dev = lens.device
    if lens.dim() != 1 or pages.dim() != 2 or free.dim() != 1:
        raise ValueError("lens must be [S], pages [S, P] and free [F]")
    s = lens.shape[0]
    _ints(lens, "lens", dev)
    _ints(pages, "pages", dev, (s, pages.shape[1]), contiguous=False)
    if pages.shape[1] > 1 and pages.stride(1) != 1:
        raise ValueError("pages needs a unit inner stride")
    _ints(free, "free", dev)
    _ints(n_free, "n_free", dev, (1,))
    lens_out = lens if lens_out is None else lens_out
    n_free_out = n_free if n_free_out is None else n_free_out
    _ints(lens_out, "lens_out", dev, (s,))
    _ints(n_free_out, "n_free_out", dev, (1,))
    a = L.PlanArgs()
    a.lens, a.pages, a.free_pages, a.n_free = lens.data_ptr(), pages.data_ptr(), free.data_ptr(), n_free.data_ptr()
    a.lens_out, a.n_free_out = lens_out.data_ptr(), n_free_out.data_ptr()
    a.pages_st, a.max_seqs, a.max_pages, a.num_pages, a.page_size = (pages.stride(0), s, pages.shape[1], free.shape[0],
                                                                      page_size)
    return a, dev


def plan_step(new, lens, pages, free, n_free, *, page_size, num_tokens, seqs=None, max_len=None, lens_out=None,
              n_free_out=None, max_q=None, prompts=False):
    """The Step of new[b] more tokens for each sequence seqs[b] (None: for sequence b, new [S], and the page table is `pages`
    itself), packed into num_tokens rows. Their pages come from the top of the free stack. pages is written in place; the
    counters go to lens_out and n_free_out, or in place too. A step that does not fit (no room, a sequence unknown or twice, a
    negative count, more tokens than num_tokens or max_len, with `prompts` tokens of a sequence that has some already) changes nothing: ok is 0 and the step has no token."""
    r = (_serving._module or _serving.host()).plan_step(new, lens, pages, free, n_free, page_size, num_tokens, seqs, max_len,
                                                        lens_out, n_free_out, prompts)
    if type(r) is int:
        L.check(r, "plan_step")
    if r is not NotImplemented:
        return Step(*r, max_q, prompts)
    a, dev = _state(lens, pages, free, n_free, lens_out, n_free_out, page_size)
    L.require_cuda(new, seqs)
    if new.dim() != 1:
        raise ValueError(f"new must be [B], got {list(new.shape)}")
    b, p = new.shape[0], pages.shape[1]
    _ints(new, "new", dev)
    if seqs is None:
        if b != lens.shape[0]:
            raise ValueError(f"new must be [{lens.shape[0]}] without seqs, got [{b}]")
        table = pages
    else:
        _ints(seqs, "seqs", dev, (b,))
        table = torch.empty(b, p, dtype=torch.int32, device=dev)
        a.seqs, a.table, a.table_st = seqs.data_ptr(), table.data_ptr(), p
    ints = torch.empty(3 * b + 4 + num_tokens, dtype=torch.int32, device=dev)
    cu, kv_lens, ok, scratch, positions = ints.split([b + 1, b, 1, b + 2, num_tokens])
    slots = torch.empty(num_tokens, dtype=torch.int64, device=dev)
    a.new_tokens, a.cu_seqlens, a.kv_lens = new.data_ptr(), cu.data_ptr(), kv_lens.data_ptr()
    a.slots, a.positions, a.ok, a.scratch = slots.data_ptr(), positions.data_ptr(), ok.data_ptr(), scratch.data_ptr()
    a.B, a.T, a.max_len = b, num_tokens, min(p * page_size if max_len is None else max_len, 0x7fffffff)
    a.prompts = int(bool(prompts))
    with torch.cuda.device(dev):
        L.check(L.lib().mv_plan_step(C.byref(a), L.stream_ptr(dev)), "plan_step")
    return Step(cu, kv_lens, table, slots, positions, ok, max_q, prompts)


def release_pages(seqs, lens, pages, free, n_free, *, page_size, lens_out=None, n_free_out=None):
    """Gives back the pages of sequences seqs [B] int32, whose lengths become 0; returns ok [1] int32: 0 where a sequence is
    unknown or there twice, or the stack has no room, and nothing was changed."""
    a, dev = _state(lens, pages, free, n_free, lens_out, n_free_out, page_size)
    L.require_cuda(seqs)
    if seqs.dim() != 1:
        raise ValueError(f"seqs must be [B], got {list(seqs.shape)}")
    _ints(seqs, "seqs", dev)
    ok = torch.empty(1, dtype=torch.int32, device=dev)
    a.seqs, a.ok, a.B = seqs.data_ptr(), ok.data_ptr(), seqs.shape[0]
    with torch.cuda.device(dev):
        L.check(L.lib().mv_release_pages(C.byref(a), L.stream_ptr(dev)), "release_pages")
    return ok


class DeviceSequences:
    """Pages and lengths of up to max_seqs sequences, shared by the caches of all layers, as layer.Sequences, with the state on
    the device."""

    def __init__(self, num_pages, page_size, max_seqs, max_len, device="cuda"):
        self.num_pages, self.page_size, self.device = num_pages, page_size, torch.device(device)
        self.max_len, self.max_pages = max_len, -(-max_len // page_size)
        i32 = dict(dtype=torch.int32, device=self.device)
        self.free = torch.arange(num_pages - 1, -1, -1, **i32)
        self.n_free = torch.full((1,), num_pages, **i32)
        self.pages = torch.zeros(max_seqs, self.max_pages, **i32)
        self.lens = torch.zeros(max_seqs, **i32)

    def cache(self, attn):
        """A cache for one layer's keys and values."""
        return PagedKV.empty(self.num_pages, self.page_size, attn.n_kv_heads, attn.head_dim, attn.dtype, self.device)

    def extend(self, new, num_tokens, seqs=None, *, max_q=None, prompts=False):
        """plan_step on this state. num_tokens: rows of the step's packed tokens (max_q: at most so many of one sequence), both
        known to the host. prompts: every sequence that gets tokens begins here, and a step in which one has tokens already is refused."""
        return plan_step(new, self.lens, self.pages, self.free, self.n_free, page_size=self.page_size,
                         num_tokens=num_tokens, seqs=seqs, max_len=self.max_len, max_q=max_q, prompts=prompts)

    def release(self, seqs):
        """release_pages on this state."""
        return release_pages(seqs, self.lens, self.pages, self.free, self.n_free, page_size=self.page_size)
