"""Attention entry points without a GPU: the argument structs match the header, the host-side checks refuse bad calls
before any launch, CPU tensors are refused, and the 64-bit oracle agrees with torch's own attention."""
import ctypes as C
import os
import re

import pytest
import torch

from conftest import ROOT
from mingmoe import _lib as L
from mingmoe import attention as A
from oracle import attention_oracle as O


def header_fields(name):
    src = open(os.path.join(ROOT, "include", "mingmoe.h")).read()
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), src, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    out = []
    for decl in body.split(";"):
        decl = decl.strip()
        if decl:
            names = [re.search(r"(\w+)\s*$", n.strip()).group(1) for n in decl.split(",")]
            out += names
    return out


@pytest.mark.parametrize("name,mirror", [("mv_paged_kv", L.PagedKV), ("mv_kv_append_args", L.KVAppendArgs),
                                         ("mv_attention_args", L.AttentionArgs)])
def test_structs_match_the_header(name, mirror):
    assert header_fields(name) == [f[0] for f in mirror._fields_]


def test_packed_arguments_are_the_structs():
    vals = list(range(1, 11)) + list(range(11, 21)) + list(range(21, 29))
    s = L.KVAppendArgs.from_buffer_copy(A._APPEND.pack(*vals))
    assert [getattr(s, f[0]) for f in L.KVAppendArgs._fields_] == vals
    vals = list(range(1, 11)) + list(range(11, 20)) + list(range(20, 30)) + [0.5, 0]
    s = L.AttentionArgs.from_buffer_copy(A._ATTN.pack(*vals))
    assert [getattr(s, f[0]) for f in L.AttentionArgs._fields_] == vals


def kv(**kw):
    c = L.PagedKV(k=4096, v=4096, dtype=L.MV_BF16, num_pages=2, page_size=16, n_kv_heads=2, head_dim=128, k_sp=4096,
                  k_st=256, k_sh=128, v_sp=4096, v_st=256, v_sh=128)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def attn(c=None, **kw):
    a = L.AttentionArgs(cache=None if c is None else C.addressof(c), q=4096, k=4096, v=4096, out=4096, cu_seqlens=4096,
                        page_table=4096, kv_lens=4096, q_st=1024, q_sh=128, k_st=256, k_sh=128, v_st=256, v_sh=128,
                        o_st=1024, o_sh=128, pt_stride=4, T=3, B=2, Hq=8, max_q=2, causal=1, max_pages=4, Tk=3, Hkv=2,
                        head_dim=128, dtype=L.MV_BF16, scale=0.1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def append(c, **kw):
    a = L.KVAppendArgs(cache=None if c is None else C.addressof(c), k=4096, v=4096, q=4096, q_out=4096, page_table=4096,
                       cu_seqlens=4096, kv_lens=4096, cos_sin=4096, k_st=256, k_sh=128, v_st=256, v_sh=128, q_st=1024,
                       q_sh=128, qo_st=1024, qo_sh=128, pt_stride=4, cs_stride=128, T=3, B=2, Hq=8, max_pages=4,
                       max_pos=9, rot_dim=128)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_host_checks():
    lib = L.lib()
    nws = lib.mv_attention_workspace_bytes()
    INV, ALN, UNS, WSP = L.MV_ERR_INVALID, L.MV_ERR_ALIGN, L.MV_ERR_UNSUPPORTED, L.MV_ERR_WORKSPACE
    bad_caches = [(INV, None), (INV, kv(k=None)), (UNS, kv(dtype=L.MV_F32)), (UNS, kv(head_dim=96)), (UNS, kv(page_size=12)),
                  (UNS, kv(page_size=512)), (INV, kv(num_pages=0)), (INV, kv(n_kv_heads=0)), (ALN, kv(k=4100)),
                  (ALN, kv(k_st=260)), (INV, kv(v_sh=64)), (ALN, kv(v_sp=4100))]
    for rc, c in bad_caches:
        assert lib.mv_kv_append(C.byref(append(c)), 4096, nws, None) == rc
        assert lib.mv_paged_attention(C.byref(attn(c)), 4096, nws, None) == rc
    c = kv()
    for rc, kw in [(INV, dict(T=-1)), (INV, dict(B=-1)), (INV, dict(Hq=-1)), (INV, dict(k=None)), (INV, dict(q_out=None)),
                   (INV, dict(cu_seqlens=None)), (INV, dict(rot_dim=24)), (INV, dict(rot_dim=144)), (INV, dict(rot_dim=-16)),
                   (INV, dict(cos_sin=None)), (INV, dict(max_pos=0)), (INV, dict(cs_stride=64)), (ALN, dict(cs_stride=130)),
                   (ALN, dict(cos_sin=4100)), (INV, dict(pt_stride=3)), (ALN, dict(q=4104)), (INV, dict(k_st=64))]:
        assert lib.mv_kv_append(C.byref(append(c, **kw)), 4096, nws, None) == rc, kw
    assert lib.mv_kv_append(C.byref(append(c)), None, nws, None) == WSP
    assert lib.mv_kv_append(C.byref(append(c)), 4096, 100, None) == WSP
    assert lib.mv_kv_append(None, 4096, nws, None) == INV
    for rc, kw in [(INV, dict(T=-1)), (INV, dict(B=-2)), (INV, dict(max_q=-1)), (INV, dict(q=None)), (INV, dict(out=None)),
                   (INV, dict(Hq=7)), (INV, dict(Hq=0)), (INV, dict(Hq=130)), (INV, dict(scale=0.0)),
                   (INV, dict(scale=float("nan"))), (INV, dict(scale=float("inf"))), (ALN, dict(q_st=1028)),
                   (INV, dict(o_sh=64))]:
        assert lib.mv_paged_attention(C.byref(attn(c, **kw)), 4096, nws, None) == rc, kw
        assert lib.mv_prompt_attention(C.byref(attn(None, **kw)), 4096, nws, None) == rc, kw
    assert lib.mv_paged_attention(C.byref(attn(c, kv_lens=None)), 4096, nws, None) == INV
    for rc, kw in [(UNS, dict(dtype=L.MV_F32)), (UNS, dict(head_dim=80)), (INV, dict(Hkv=0)), (INV, dict(k=None)),
                   (ALN, dict(v=4104))]:
        assert lib.mv_prompt_attention(C.byref(attn(None, **kw)), 4096, nws, None) == rc, kw
    assert lib.mv_prompt_attention(C.byref(attn(c)), 4096, nws, None) == INV
    for f, a in ((lib.mv_paged_attention, attn(c)), (lib.mv_prompt_attention, attn(None))):
        assert f(C.byref(a), 4096, nws - 1, None) == WSP
        assert f(C.byref(a), 4112, nws, None) == WSP
    # nothing to do is not an error
    for kw in (dict(T=0), dict(B=0)):
        assert lib.mv_kv_append(C.byref(append(c, **kw)), 4096, nws, None) == L.MV_OK
        assert lib.mv_paged_attention(C.byref(attn(c, **kw)), 4096, nws, None) == L.MV_OK
        assert lib.mv_prompt_attention(C.byref(attn(None, **kw)), 4096, nws, None) == L.MV_OK


def test_cpu_tensors_refused():
    z = torch.zeros(2, 16, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        A.PagedKV(z, z)
    q = torch.zeros(3, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        A.prompt_attention(q, q, q, torch.tensor([0, 3], dtype=torch.int32))


@pytest.mark.parametrize("nq,n,causal", [(5, 5, True), (3, 9, True), (4, 7, False), (6, 4, True)])
def test_oracle(nq, n, causal):
    g = torch.Generator().manual_seed(nq)
    q, k, v = (torch.randn(m, h, 64, generator=g).to(torch.bfloat16) for m, h in ((nq, 6), (n, 2), (n, 2)))
    out, lse, tol, tol_lse = O.attention(q, k, v, causal)
    see = torch.ones(nq, n, dtype=torch.bool)
    if causal:
        see = torch.arange(n)[None] <= (n - nq + torch.arange(nq))[:, None]
    kk, vv = (x.double().repeat_interleave(3, 1).transpose(0, 1) for x in (k, v))
    s = (q.double().transpose(0, 1) @ kk.transpose(1, 2) / 8).masked_fill(~see, float("-inf"))
    rows = see.any(1)
    want = torch.softmax(s[:, rows], -1) @ vv
    assert torch.allclose(out[rows].transpose(0, 1), want, atol=1e-12)
    assert torch.allclose(lse[rows].T, torch.logsumexp(s[:, rows], -1), atol=1e-12)
    assert (out[~rows] == 0).all() and torch.isinf(lse[~rows]).all() and (tol[rows] > 0).all() and (tol_lse[rows] > 0).all()
    if rows.all():
        fast = O.attention_fast(q, k, v, causal)
        assert torch.allclose(fast[0], out, atol=1e-12) and torch.allclose(fast[1], lse, atol=1e-12)


@pytest.mark.parametrize("inter", [False, True])
def test_oracle_rotation_turns_and_keeps_the_length(inter):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(7, 3, 64, generator=g).to(torch.bfloat16)
    cs = A.rotation_table(20, 32, device="cpu")
    y, tol = O.rotate(x, cs, torch.arange(7) + 5, inter)
    assert torch.allclose(y.norm(dim=-1), x.double().norm(dim=-1), rtol=1e-6)
    assert torch.equal(y[..., 32:], x[..., 32:].double()) and (tol[..., 32:] == 0).all()
    assert torch.equal(O.rotate(x, cs, torch.zeros(7), inter)[0], x.double())
