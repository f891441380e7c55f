"""What the 8-bit products, draws and plans refuse, without a GPU: the entry points' checks come before any launch, and the Python
calls raise for tensors that do not fit."""
import ctypes as C

import pytest
import torch

from mingmoe import _lib as L
from mingmoe import fp8, paging, sampling
from mingmoe.layer import AttentionBlock, Decoder

P16 = 4096  # an address that is never read


def linear(**kw):
    a = L.Fp8LinearArgs(P16, P16, P16, 0, 1 << 24, P16, 256, 256, 2, 0, 300, 1 << 20, 40, 300, 256, L.MV_BF16, L.MV_F32, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(T=-1), L.MV_ERR_INVALID), (dict(N=-1), L.MV_ERR_INVALID), (dict(K=0), L.MV_ERR_INVALID),
    (dict(x_dtype=L.MV_F32), L.MV_ERR_UNSUPPORTED), (dict(x_dtype=9), L.MV_ERR_UNSUPPORTED),
    (dict(out_dtype=L.MV_I8), L.MV_ERR_UNSUPPORTED), (dict(x=0), L.MV_ERR_INVALID), (dict(wq=0), L.MV_ERR_INVALID),
    (dict(ws=0), L.MV_ERR_INVALID), (dict(out=0), L.MV_ERR_INVALID), (dict(x_st=-1), L.MV_ERR_INVALID),
    (dict(o_st=299), L.MV_ERR_INVALID), (dict(w_st=240), L.MV_ERR_INVALID), (dict(ws_st=1), L.MV_ERR_INVALID),
    (dict(out=P16), L.MV_ERR_INVALID), (dict(out=P16 + 256 * 2 * 39), L.MV_ERR_INVALID),  # x and out overlap
    (dict(residual=(1 << 24) + 4, r_st=300), L.MV_ERR_INVALID), (dict(residual=1 << 24, r_st=299), L.MV_ERR_INVALID),
    (dict(wq=P16 + 8), L.MV_ERR_ALIGN), (dict(w_st=264), L.MV_ERR_ALIGN), (dict(scratch=0), L.MV_ERR_WORKSPACE),
    (dict(scratch=P16 + 16), L.MV_ERR_WORKSPACE), (dict(scratch_bytes=100), L.MV_ERR_WORKSPACE)])
def test_linear_refusals(kw, code):
    assert L.lib().mv_fp8_linear(C.byref(linear(**kw)), P16, 256, None) == code, L.lib().mv_last_error()


def test_linear_workspace_and_nothing_to_do():
    lib = L.lib()
    assert lib.mv_fp8_linear(None, P16, 256, None) == L.MV_ERR_INVALID
    assert lib.mv_fp8_linear(C.byref(linear()), None, 256, None) == L.MV_ERR_WORKSPACE
    assert lib.mv_fp8_linear(C.byref(linear()), P16, 255, None) == L.MV_ERR_WORKSPACE
    for kw in (dict(T=0), dict(N=0)):  # before any pointer is looked at
        assert lib.mv_fp8_linear(C.byref(linear(x=0, out=0, **kw)), None, 0, None) == L.MV_OK
    assert lib.mv_fp8_linear_scratch_bytes(0, 10, 10) == 0
    assert lib.mv_fp8_linear_scratch_bytes(100, 10, 200) >= 100 * 256 + 2 * 100


def test_columns_of_one_buffer_do_not_overlap():
    """x in the first 512 bytes of rows of 2048, the result behind it: taken (and refused for its workspace only)."""
    kw = dict(x=P16, x_st=1024, out=P16 + 512, o_st=512, out_dtype=L.MV_F32)
    assert L.lib().mv_fp8_linear(C.byref(linear(**kw)), None, 0, None) == L.MV_ERR_WORKSPACE
    kw["out"] = P16 + 508
    assert L.lib().mv_fp8_linear(C.byref(linear(**kw)), None, 0, None) == L.MV_ERR_INVALID


def test_quantize_refusals():
    lib = L.lib()
    q = lambda x=P16, dt=L.MV_BF16, st=256, T=4, K=200, q=P16, q_st=256, s=P16, s_st=4: lib.mv_quantize_fp8(x, dt, st, T, K, q, q_st,
                                                                                                           s, s_st, None)
    assert q(T=-1) == q(K=-1) == q(x=None) == q(q=None) == q(s=None) == q(q_st=240) == q(s_st=3) == L.MV_ERR_INVALID
    assert q(dt=L.MV_I8) == L.MV_ERR_UNSUPPORTED
    assert q(q=P16 + 8) == q(q_st=264) == q(x=P16 + 1) == L.MV_ERR_ALIGN
    assert q(T=0, x=None) == q(K=0, x=None) == L.MV_OK
    w = lambda w=P16, dt=L.MV_BF16, st=256, N=300, K=200, q=P16, q_st=256, s=P16, s_st=2: lib.mv_quantize_fp8_weight(w, dt, st, N, K, q,
                                                                                                                     q_st, s, s_st, None)
    assert w(N=-1) == w(st=199) == w(q_st=199) == w(s_st=1) == w(w=None) == L.MV_ERR_INVALID
    assert w(dt=L.MV_I32) == L.MV_ERR_UNSUPPORTED and w(N=0, w=None) == L.MV_OK


def draw(**kw):
    a = L.SampleArgs(P16, P16, 0, 0, 0, 0, P16, 0, 0, 1000, 0, 1.0, 1.0, 0.0, 0, 3, 1000, L.MV_F32, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(B=-1), L.MV_ERR_INVALID), (dict(V=-1), L.MV_ERR_INVALID), (dict(V=(1 << 30) + 1), L.MV_ERR_INVALID),
    (dict(B=(1 << 27) + 1), L.MV_ERR_INVALID), (dict(dtype=L.MV_I32), L.MV_ERR_UNSUPPORTED), (dict(logits=0), L.MV_ERR_INVALID),
    (dict(u=0), L.MV_ERR_INVALID), (dict(tokens=0), L.MV_ERR_INVALID), (dict(st=-1), L.MV_ERR_INVALID),
    (dict(B=0, logits=0, u=0, tokens=0), L.MV_OK)])
def test_sample_refusals(kw, code):
    assert L.lib().mv_sample(C.byref(draw(**kw)), None) == code
    assert L.lib().mv_sample(None, None) == L.MV_ERR_INVALID


def plan(**kw):
    a = L.PlanArgs()
    for n in ("new_tokens", "lens", "n_free", "free_pages", "pages", "lens_out", "n_free_out", "cu_seqlens", "kv_lens", "slots",
              "positions", "ok", "scratch"):
        setattr(a, n, P16)
    a.pages_st, a.B, a.max_seqs, a.max_pages, a.page_size, a.max_len, a.num_pages, a.T = 10, 4, 4, 10, 16, 160, 50, 4
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(B=-1), L.MV_ERR_INVALID), (dict(B=5), L.MV_ERR_INVALID), (dict(B=3), L.MV_ERR_INVALID),
    (dict(max_seqs=(1 << 18) + 1, B=1, seqs=P16, table=P16), L.MV_ERR_INVALID), (dict(max_pages=-1), L.MV_ERR_INVALID),
    (dict(num_pages=-1), L.MV_ERR_INVALID), (dict(page_size=4), L.MV_ERR_UNSUPPORTED), (dict(page_size=24), L.MV_ERR_UNSUPPORTED),
    (dict(page_size=512), L.MV_ERR_UNSUPPORTED), (dict(T=-1), L.MV_ERR_INVALID), (dict(max_len=-1), L.MV_ERR_INVALID),
    (dict(pages_st=9), L.MV_ERR_INVALID), (dict(seqs=P16), L.MV_ERR_INVALID), (dict(seqs=P16, table=P16, table_st=9), L.MV_ERR_INVALID),
    *[({n: 0}, L.MV_ERR_INVALID) for n in ("new_tokens", "lens", "n_free", "free_pages", "pages", "lens_out", "n_free_out", "cu_seqlens",
                                           "kv_lens", "slots", "positions", "ok", "scratch")]])
def test_plan_refusals(kw, code):
    assert L.lib().mv_plan_step(C.byref(plan(**kw)), None) == code


def test_release_refusals():
    lib = L.lib()
    assert lib.mv_plan_step(None, None) == lib.mv_release_pages(None, None) == L.MV_ERR_INVALID
    assert lib.mv_release_pages(C.byref(plan()), None) == L.MV_ERR_INVALID  # no sequences named
    assert lib.mv_release_pages(C.byref(plan(seqs=P16, ok=0)), None) == L.MV_ERR_INVALID
    assert lib.mv_release_pages(C.byref(plan(seqs=P16, page_size=3)), None) == L.MV_ERR_UNSUPPORTED


def test_cpu_tensors_are_refused():
    bf = dict(dtype=torch.bfloat16)
    wq, ws = torch.zeros(128, 128, dtype=torch.uint8).view(fp8.E4M3), torch.ones(1, 1)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    for call in (lambda: fp8.fp8_linear(torch.zeros(2, 128, **bf), wq, ws), lambda: fp8.quantize_fp8(torch.zeros(2, 128, **bf)),
                 lambda: fp8.quantize_fp8_weight(torch.zeros(2, 128, **bf)), lambda: sampling.sample(torch.zeros(2, 5), torch.zeros(2)),
                 lambda: paging.plan_step(i32(2), i32(2), i32(2, 4), i32(9), i32(1), page_size=8, num_tokens=2),
                 lambda: paging.release_pages(i32(1), i32(2), i32(2, 4), i32(9), i32(1), page_size=8)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_weights_that_do_not_fit():
    wq = torch.zeros(640, 100, dtype=torch.uint8).view(fp8.E4M3)
    with pytest.raises(ValueError):
        AttentionBlock((wq, None), torch.zeros(100, 512), torch.ones(100), 8, 2, 64, None)
    with pytest.raises(ValueError):
        Decoder(torch.zeros(10, 96), [], torch.ones(96), (wq, None))


def test_a_decoder_needs_a_token():
    decoder = Decoder(torch.zeros(10, 96), [], torch.ones(96), torch.zeros(10, 96))
    for tokens in (torch.zeros(0, dtype=torch.int64), torch.zeros(1, 2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="tokens"):
            decoder(tokens, None)
