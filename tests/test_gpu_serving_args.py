"""What the Python calls of the 8-bit products, draws and plans refuse, and what they copy because only its layout does not fit:
both host paths (C++ and the Python code behind it) give the same."""
import pytest
import torch

from mingmoe import _lib as L
from mingmoe import _serving, fp8, paging, sampling

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


class Behind:
    """The C++ module as if nothing fitted it: every call goes through the Python code."""
    fp8_linear = sample = plan_step = staticmethod(lambda *a: NotImplemented)
    workspace = staticmethod(lambda *a: None)


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    _serving.host()
    if request.param == "python":
        monkeypatch.setattr(_serving, "_module", Behind)
    return request.param


def test_linear(cuda, path):
    g = torch.Generator(device=cuda).manual_seed(0)
    w = torch.randn(300, 256, generator=g, device=cuda)
    wq, ws = fp8.quantize_fp8_weight(w)
    x = torch.randn(6, 256, generator=g, device=cuda).to(BF)
    y = fp8.fp8_linear(x, wq, ws)
    assert torch.equal(fp8.fp8_linear(x.t().contiguous().t(), wq, ws), y)  # columns side by side: copied
    assert torch.equal(fp8.fp8_linear(x.view(2, 3, 256).transpose(0, 1), wq, ws), y.view(2, 3, 300).transpose(0, 1))
    assert torch.equal(fp8.fp8_linear(x[:1].expand(6, 256), wq, ws), y[:1].expand(6, 300))
    r = torch.randn(300, 6, generator=g, device=cuda).to(BF).t()
    assert torch.equal(fp8.fp8_linear(x, wq, ws, residual=r), fp8.fp8_linear(x, wq, ws, residual=r.contiguous()))
    out = torch.empty(6, 300, dtype=F32, device=cuda)
    assert fp8.fp8_linear(x, wq, ws, out=out, out_dtype=F32) is out or torch.equal(out, fp8.fp8_linear(x, wq, ws, out_dtype=F32))
    for exc, call in [(TypeError, lambda: fp8.fp8_linear(x.float(), wq, ws)),
                      (TypeError, lambda: fp8.fp8_linear(x, wq.view(torch.uint8), ws)),
                      (TypeError, lambda: fp8.fp8_linear(x, wq, ws.double())),
                      (TypeError, lambda: fp8.fp8_linear(x, wq, ws, out_dtype=torch.float64)),
                      (ValueError, lambda: fp8.fp8_linear(x[:, :255], wq, ws)),
                      (ValueError, lambda: fp8.fp8_linear(x, wq, ws[:, :1])),
                      (ValueError, lambda: fp8.fp8_linear(x, wq, ws[:2])),
                      (ValueError, lambda: fp8.fp8_linear(x, wq, ws, residual=y[:5])),
                      (ValueError, lambda: fp8.fp8_linear(x, wq, ws, residual=y.float())),
                      (ValueError, lambda: fp8.fp8_linear(x, wq, ws, out=out)),
                      (RuntimeError, lambda: fp8.fp8_linear(x, wq.cpu(), ws)),
                      (RuntimeError, lambda: fp8.fp8_linear(x[:, :200].contiguous(), wq[:, 8:208], ws))]:
        with pytest.raises(exc):
            call()
    assert not L.all_workspace_errors()


def test_sample(cuda, path):
    g = torch.Generator(device=cuda).manual_seed(1)
    x, u = torch.randn(4, 500, generator=g, device=cuda), torch.rand(4, generator=g, device=cuda)
    t = torch.tensor([0.5, 1.0, 0.0, 2.0], device=cuda)
    want = sampling.sample(x, u, temperature=t, top_k=9)
    assert torch.equal(sampling.sample(x.t().contiguous().t(), u, temperature=t, top_k=9), want)
    assert torch.equal(sampling.sample(x, torch.stack([u, u], 1)[:, 0], temperature=torch.stack([t, t], 1)[:, 0], top_k=9), want)
    assert torch.equal(sampling.sample(x, u, temperature=t, top_k=torch.full((4,), 9, dtype=torch.int32, device=cuda)), want)
    assert torch.equal(sampling.sample(x, u, temperature=1, top_k=10 ** 12), sampling.sample(x, u))
    i64 = torch.full((4,), 9, device=cuda)
    for exc, call in [(TypeError, lambda: sampling.sample(x.double(), u)), (ValueError, lambda: sampling.sample(x[0], u)),
                      (ValueError, lambda: sampling.sample(x, u[:3])), (ValueError, lambda: sampling.sample(x, u.double())),
                      (ValueError, lambda: sampling.sample(x, u, top_k=i64)), (ValueError, lambda: sampling.sample(x, u, top_p=t[:2])),
                      (ValueError, lambda: sampling.sample(x, u, out=i64[:3])),
                      (ValueError, lambda: sampling.sample(x, u, out=i64.int())), (RuntimeError, lambda: sampling.sample(x, u.cpu())),
                      (RuntimeError, lambda: sampling.sample(x, u, min_p=t.cpu()))]:
        with pytest.raises(exc):
            call()


def test_plan(cuda, path):
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)
    state = lambda: (i(3, 9), torch.arange(12, dtype=torch.int32, device=cuda).view(2, 6), i(20, 21, 22, 23), i(4))
    kw = dict(page_size=8, num_tokens=9)
    step = paging.plan_step(i(2, 7), *state(), **kw)
    assert step.ok.item() == 1 and step.kv_lens.tolist() == [5, 16] and step.positions.tolist() == [3, 4, 9, 10, 11, 12, 13, 14, 15]
    lens, pages, free, n_free = state()
    for exc, call in [(TypeError, lambda: paging.plan_step(i(2, 7).long(), lens, pages, free, n_free, **kw)),
                      (ValueError, lambda: paging.plan_step(i(2), lens, pages, free, n_free, **kw)),
                      (ValueError, lambda: paging.plan_step(i(2, 7), lens, pages[:1], free, n_free, **kw)),
                      (ValueError, lambda: paging.plan_step(i(2, 7), lens, pages.t().contiguous().t(), free, n_free, **kw)),
                      (ValueError, lambda: paging.plan_step(i(2, 7), lens, pages, free, i(4, 4), **kw)),
                      (ValueError, lambda: paging.plan_step(i(2, 7), lens, pages, free, n_free, seqs=i(0), **kw)),
                      (ValueError, lambda: paging.plan_step(i(2, 7), lens, pages, free, n_free, lens_out=i(1), **kw)),
                      (RuntimeError, lambda: paging.plan_step(i(2, 7), lens, pages, free, n_free, page_size=12, num_tokens=9)),
                      (RuntimeError, lambda: paging.plan_step(i(2, 7), lens, pages, free.cpu(), n_free, **kw)),
                      (RuntimeError, lambda: paging.plan_step(i(2, 7), lens, pages, free, n_free, page_size=8, num_tokens=-1))]:
        with pytest.raises(exc):
            call()
    torch.cuda.synchronize()
    assert lens.tolist() == [3, 9] and n_free.item() == 4
