"""A whole decoder layer on the paged cache: the attention half in front of MoeBlock.

    h = x + W_o attention(rotate(W_qkv rms_norm(x)))        AttentionBlock
    y = h + MoE(rms_norm(h))                                MoeBlock

The projections are the small-linear kernel (norm prologue, residual epilogue) up to 16 tokens and plain GEMMs above;
the attention is kv_append + paged_attention for new tokens of running sequences, and kv_append + prompt_attention for
whole prompts, which need not be read back from the cache. Inference only: nothing here has a backward pass.

    seqs = Sequences(num_pages=4096, page_size=64, max_seqs=32, max_len=8192)
    layers = [DecoderLayer(attn, moe, seqs.cache(attn)) for attn, moe in ...]
    batch = seqs.extend({0: 700, 3: 41}, prompts=True)      # sequences 0 and 3 begin with prompts of 700 and 41 tokens
    for layer in layers: x = layer(x, batch)
    batch = seqs.extend({0: 1, 3: 1})                       # one new token each
    for layer in layers: x = layer(x, batch)
"""
from __future__ import annotations

import torch

from . import moe
from .attention import PagedKV, kv_append, paged_attention, prompt_attention


class Batch:
    """One step's packed tokens: cu_seqlens, the page table and lengths of its sequences (device), and what the host knows
    of them: the largest number of new tokens, and whether every sequence begins here."""

    __slots__ = ("cu_seqlens", "page_table", "kv_lens", "max_q", "prompts")

    def __init__(self, cu_seqlens, page_table, kv_lens, max_q, prompts):
        self.cu_seqlens, self.page_table, self.kv_lens = cu_seqlens, page_table, kv_lens
        self.max_q, self.prompts = max_q, prompts


class Sequences:
    """Pages and lengths of up to max_seqs sequences, shared by the caches of all layers (a page id means the same page
    in each). Host bookkeeping; extend() copies one step's tables to the device."""

    def __init__(self, num_pages, page_size, max_seqs, max_len, device="cuda"):
        self.num_pages, self.page_size, self.device = num_pages, page_size, torch.device(device)
        self.max_len, self.max_pages = max_len, -(-max_len // page_size)
        self.free = list(range(num_pages - 1, -1, -1))
        self.pages = [[] for _ in range(max_seqs)]
        self.lens = [0] * max_seqs

    def cache(self, attn):
        """A cache for one layer's keys and values."""
        return PagedKV.empty(self.num_pages, self.page_size, attn.n_kv_heads, attn.head_dim, attn.w_qkv.dtype, self.device)

    def extend(self, new, prompts=False):
        """The batch of new[s] tokens for each sequence s of the dict, in its order; their pages are taken now. A step that is
        refused, or fails, changes nothing."""
        pages, taken = {}, 0  # the sequences' pages after the step, and how many of them are new
        for s, n in new.items():
            if n < 0:
                raise ValueError(f"{n} new tokens of sequence {s}")
            if prompts and self.lens[s]:
                raise ValueError(f"sequence {s} has {self.lens[s]} tokens already")
            need = -(-(self.lens[s] + n) // self.page_size)
            more = max(need - len(self.pages[s]), 0)
            if self.lens[s] + n > self.max_len or taken + more > len(self.free):
                raise RuntimeError(f"no room for {n} more tokens of sequence {s}")
            pages[s] = self.pages[s] + [self.free[-1 - i] for i in range(taken, taken + more)]
            taken += more
        cu = [0]
        for n in new.values():
            cu.append(cu[-1] + n)
        i32 = dict(dtype=torch.int32, device=self.device)
        rows = torch.tensor([p + [0] * (self.max_pages - len(p)) for p in pages.values()], **i32)
        batch = Batch(torch.tensor(cu, **i32), rows.reshape(len(pages), self.max_pages),
                      torch.tensor([self.lens[s] + n for s, n in new.items()], **i32), max(new.values(), default=0), prompts)
        del self.free[len(self.free) - taken:]
        for s, n in new.items():
            self.pages[s] = pages[s]
            self.lens[s] += n
        return batch

    def release(self, s):
        """Gives back the pages of sequence s."""
        self.free += self.pages[s]
        self.pages[s], self.lens[s] = [], 0


class AttentionBlock:
    """x + W_o attention(rotate(W_qkv rms_norm(x))): w_qkv [(Hq + 2 Hkv) D, H], w_o [H, Hq D], norm_w [H], bf16;
    cos_sin as in kv_append (attention.rotation_table)."""

    def __init__(self, w_qkv, w_o, norm_w, n_heads, n_kv_heads, head_dim, cos_sin, *, eps=1e-6, interleaved=False):
        if w_qkv.shape[0] != (n_heads + 2 * n_kv_heads) * head_dim or w_o.shape[1] != n_heads * head_dim:
            raise ValueError(f"w_qkv {tuple(w_qkv.shape)} / w_o {tuple(w_o.shape)} do not fit {n_heads} / {n_kv_heads} "
                             f"heads of {head_dim}")
        self.w_qkv, self.w_o, self.norm_w, self.eps = w_qkv, w_o, norm_w, float(eps)
        self.n_heads, self.n_kv_heads, self.head_dim = n_heads, n_kv_heads, head_dim
        self.cos_sin, self.interleaved = cos_sin, interleaved

    def project(self, x):
        """W_qkv rms_norm(x) as [T, Hq + 2 Hkv, D]: a token's query, key and value heads side by side."""
        import fastlinear
        import fused_ops  # the drop-in modules (same directory on sys.path)
        if x.shape[0] <= moe.DECODE_MAX_M:
            qkv = fastlinear.small_linear(x, self.w_qkv, norm=(self.norm_w, self.eps))
        else:
            qkv = torch.nn.functional.linear(fused_ops.rms_norm(x, self.norm_w, self.eps), self.w_qkv)
        return qkv.view(x.shape[0], self.n_heads + 2 * self.n_kv_heads, self.head_dim)

    def attend(self, qkv, cache, batch):
        """Appends the batch's keys and values to `cache` and attends over all of its sequences' tokens: [T, Hq, D]."""
        hq, hk = self.n_heads, self.n_heads + self.n_kv_heads
        k, v = qkv[:, hq:hk], qkv[:, hk:]
        where = (batch.page_table, batch.cu_seqlens, batch.kv_lens)
        turn = dict(cos_sin=self.cos_sin, interleaved=self.interleaved)
        if batch.prompts:
            # the rotated keys are wanted beside the cache as well: they go along as heads of q
            qk = kv_append(cache, k, v, *where, q=qkv[:, :hk], **turn)
            return prompt_attention(qk[:, :hq], qk[:, hq:], v, batch.cu_seqlens, max_q=batch.max_q)
        q = kv_append(cache, k, v, *where, q=qkv[:, :hq], **turn)
        return paged_attention(q, cache, *where, max_q=batch.max_q)

    def output(self, o, x):
        """x + W_o o. Up to 16 tokens the residual is added in fp32 and the sum rounded once; above, it is the accumulator of
        the library GEMM, which may round partial sums to bf16 where it splits them (torch.backends.cuda.matmul.
        allow_bf16_reduced_precision_reduction)."""
        import fastlinear
        o = o.reshape(x.shape[0], -1)
        if x.shape[0] <= moe.DECODE_MAX_M:
            return fastlinear.small_linear(o, self.w_o, residual=x)
        return torch.addmm(x, o, self.w_o.t())

    def __call__(self, x, cache, batch):
        """x [T, H] bf16 of the batch's packed tokens -> [T, H]; their keys and values go into `cache`."""
        with torch.cuda.device(x.device):
            return self.output(self.attend(self.project(x), cache, batch), x)


class DecoderLayer:
    """AttentionBlock and MoeBlock with the layer's cache."""

    def __init__(self, attn, moe_block, cache):
        self.attn, self.moe, self.cache = attn, moe_block, cache

    def __call__(self, x, batch):
        with torch.cuda.device(x.device):
            h = self.attn(x, self.cache, batch)
            return self.moe.decode(h) if h.shape[0] <= moe.DECODE_MAX_M else self.moe.prefill(h)
