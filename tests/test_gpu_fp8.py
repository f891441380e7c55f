"""GPU parity: rounding to e4m3 blocks (bit-equal) and products with 8-bit weights against the plain 64-bit implementation, each
element within the bound that oracle.serving_oracle derives from the promised arithmetic."""
import math

import pytest
import torch

from mingmoe import _lib as L
from mingmoe import fp8 as F
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def randn(dev, shape, seed, dtype=F32, scale=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=dev) * scale).to(dtype)


def errors():
    torch.cuda.synchronize()
    return sorted(c for c, _ in L.all_workspace_errors().values())


def weight(dev, n, k, seed):
    return F.quantize_fp8_weight(randn(dev, (n, k), seed, scale=0.02))


def check(y, x, wq, ws, residual=None):
    ref, mag = O.fp8_linear(x, wq, ws, residual)
    tol = O.fp8_bound(ref, mag, wq.shape[1], y.dtype)
    off = (y.double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol.clamp(min=1e-300)).max())
    assert errors() == []


# ------------------------------------------------------------------------------------------------ rounding

@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("t,k", [(1, 1), (1, 128), (3, 127), (5, 129), (17, 200), (2, 1500), (33, 2048), (7, 252)])
def test_quantize(cuda, dtype, t, k):
    x = randn(cuda, (t, k), 1, dtype, 3.0)
    x[0, : k // 2] *= 100
    q, scale = F.quantize_fp8(x)
    rq, rs = O.quantize(x)
    assert torch.equal(scale.double(), rs) and torch.equal(q.double(), rq)


def test_quantize_every_16_bit_value(cuda):
    """All finite bf16 and f16 values, each at the head of its own block and inside blocks with a larger value."""
    for dtype in (BF, FP):
        x = torch.arange(-32768, 32768, dtype=torch.int32, device=cuda).to(torch.int16).view(dtype)
        x = x[torch.isfinite(x)]
        x = torch.cat([x, x.new_zeros(-x.numel() % 128)])
        for rows in (x.view(-1, 1), x.view(-1, 128), x.sort().values.view(-1, 128)):
            q, scale = F.quantize_fp8(rows)
            rq, rs = O.quantize(rows)
            assert torch.equal(scale.double(), rs) and torch.equal(q.double(), rq)


def test_quantize_strides(cuda):
    """Rows at every alignment of 2 bytes give the same bits."""
    flat = randn(cuda, (9 * 400,), 2, BF)
    for off in range(9):
        for st in (300, 301, 304):
            x = torch.as_strided(flat, (8, 256), (st, 1), off)
            q, scale = F.quantize_fp8(x)
            q2, scale2 = F.quantize_fp8(x.contiguous())
            assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(scale, scale2)


def test_quantize_not_finite(cuda):
    x = randn(cuda, (4, 256), 3, BF)
    x[1, 5], x[2, 200], x[3, 0] = math.nan, math.inf, -math.inf
    _, scale = F.quantize_fp8(x)
    assert torch.isnan(scale).tolist() == [[False, False], [True, False], [False, True], [True, False]]


@pytest.mark.parametrize("dtype", [BF, FP, F32])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (129, 127), (300, 400)])
def test_quantize_weight(cuda, dtype, n, k):
    w = randn(cuda, (n, k), 4, dtype, 0.1)
    q, s = F.quantize_fp8_weight(w)
    assert q.data_ptr() % 16 == 0 and (n == 1 or q.stride(0) % 16 == 0)
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            block = w[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128].float()
            # quotients of fp32 numbers, rounded to fp32 (64 bits hold enough of them that rounding twice is rounding once)
            scale = torch.clamp((block.abs().max().double() / 448).float(), min=2.0 ** -100)
            assert s[i, j] == scale
            block = (block.double() / scale.double()).float()
            got = q[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128].double()
            assert torch.equal(got, O.round_e4m3(block.double().clamp(-448, 448)))


# ------------------------------------------------------------------------------------------------ products

@pytest.mark.parametrize("t", [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("n,k", [(1, 16), (16, 128), (127, 100), (128, 256), (129, 384), (200, 1500), (2560, 2048), (383, 4000)])
def test_sizes(cuda, t, n, k):
    x = randn(cuda, (t, k), 5, BF)
    wq, ws = weight(cuda, n, k, 6)
    check(F.fp8_linear(x, wq, ws, out_dtype=F32), x, wq, ws)


@pytest.mark.parametrize("xt", [BF, FP])
@pytest.mark.parametrize("ot", [BF, FP, F32])
@pytest.mark.parametrize("t,n,k", [(1, 300, 520), (5, 1000, 1000), (40, 130, 2048), (150, 513, 700), (1000, 640, 512)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_types(cuda, xt, ot, t, n, k, with_residual):
    x = randn(cuda, (t, k), 7, xt)
    wq, ws = weight(cuda, n, k, 8)
    r = randn(cuda, (t, n), 9, ot) if with_residual else None
    y = F.fp8_linear(x, wq, ws, residual=r, out_dtype=ot)
    assert y.dtype == ot
    check(y, x, wq, ws, r)


@pytest.mark.parametrize("t,n,k", [(2043, 2048, 2048), (700, 5632, 2048), (4099, 1100, 1408)])
def test_large(cuda, t, n, k):
    x = randn(cuda, (t, k), 10, BF)
    x[:, :5] *= 30
    wq, ws = weight(cuda, n, k, 11)
    check(F.fp8_linear(x, wq, ws), x, wq, ws)


@pytest.mark.parametrize("t", [3, 61])
def test_vocabulary(cuda, t):
    x = randn(cuda, (t, 1500), 12, FP)
    wq, ws = weight(cuda, 50257, 1500, 13)
    check(F.fp8_linear(x, wq, ws, out_dtype=F32), x, wq, ws)


def test_uneven_scales(cuda):
    """Scales of a token's and a weight's blocks that differ by powers of 2^10: each block meets its own factor."""
    x = randn(cuda, (140, 640), 14, BF) * torch.exp2(10.0 * torch.randint(-3, 4, (140, 5, 1), device=cuda).float()).expand(
        140, 5, 128).reshape(140, 640).to(BF)
    wq, ws = weight(cuda, 700, 640, 15)
    ws *= torch.exp2(10.0 * torch.randint(-3, 4, ws.shape, device=cuda).float())
    for t in (1, 7, 140):
        check(F.fp8_linear(x[:t], wq, ws, out_dtype=F32), x[:t], wq, ws)


def test_not_finite_tokens_stay_alone(cuda):
    x = randn(cuda, (40, 300), 16, BF)
    wq, ws = weight(cuda, 200, 300, 17)
    for t in (3, 20, 40):
        good = F.fp8_linear(x[:t], wq, ws)
        bad = x[:t].clone()
        bad[1, 290] = math.inf
        y = F.fp8_linear(bad, wq, ws)
        assert torch.isnan(y[1]).all()
        keep = torch.arange(t, device=cuda) != 1
        assert torch.equal(y[keep], good[keep])
    assert errors() == []


def test_zeros_and_leading_axes(cuda):
    wq, ws = weight(cuda, 100, 256, 18)
    assert bool((F.fp8_linear(torch.zeros(3, 256, dtype=BF, device=cuda), wq, ws) == 0).all())
    x = randn(cuda, (2, 3, 256), 19, BF)
    assert torch.equal(F.fp8_linear(x, wq, ws), F.fp8_linear(x.view(6, 256), wq, ws).view(2, 3, 100))
    assert F.fp8_linear(x[:0], wq, ws).shape == (0, 3, 100)
    assert F.fp8_linear(x[0, 0], wq, ws).shape == (100,)


def test_strides(cuda):
    """Rows of x and the residual inside wider tensors, at odd offsets; weights inside a wider stack."""
    big = randn(cuda, (50, 1000), 20, BF)
    stack, ws = weight(cuda, 256, 1024, 21)
    wq = stack[:, 512:]
    r = randn(cuda, (50, 333), 22, BF)[:, 7:]
    for t in (1, 9, 50):
        for off in (0, 1, 4, 8):
            x = big[:t, off:off + 512]
            res = r[:t, :256]
            y = F.fp8_linear(x, wq, ws[:, 4:], residual=res)
            check(y, x, wq, ws[:, 4:], res)
            out = torch.zeros(t, 300, dtype=BF, device=cuda)
            F.fp8_linear(x, wq, ws[:, 4:], residual=res, out=out[:, 3:259])
            assert torch.equal(out[:, 3:259], y) and bool((out[:, :3] == 0).all()) and bool((out[:, 259:] == 0).all())


@pytest.mark.parametrize("ot", [BF, FP, F32])
@pytest.mark.parametrize("t,n", [(3, 131), (40, 1001), (130, 2095), (700, 2095), (700, 5803), (600, 2944), (2100, 1191)])
def test_columns_beside_the_result_stay(cuda, ot, t, n):
    """Results with a ragged end inside rows of whole 16 bytes, at addresses of whole 16 bytes."""
    x, r = randn(cuda, (t, 200), 60, BF), randn(cuda, (t, n), 61, ot)
    wq, ws = weight(cuda, n, 200, 62)
    buf = torch.full((t + 2, (n + 31) // 16 * 16), 7.0, dtype=ot, device=cuda)
    for at in (0, 8, 16):
        for res in (None, r):
            buf.fill_(7)
            out = buf[1:t + 1, at:at + n]
            if out.shape[1] < n:
                continue
            F.fp8_linear(x, wq, ws, residual=res, out=out, out_dtype=ot)
            check(out, x, wq, ws, res)
            out.fill_(7)
            assert bool((buf == 7).all())


@pytest.mark.parametrize("ot", [BF, FP, F32])
def test_a_ragged_result_of_several_tiles_a_pair(cuda, ot):
    """Lines that are written by elements lie where the next tile's residual goes: the same as from rows that have no such copies."""
    t, n = 9001, 1201
    x = randn(cuda, (t, 384), 65, BF)
    wq, ws = weight(cuda, n, 384, 66)
    wide = randn(cuda, (t, 1216), 67, ot)
    want = F.fp8_linear(x, wq, ws, residual=wide[:, :n].contiguous(), out_dtype=ot)
    check(want[:200], x[:200], wq, ws, wide[:200, :n])
    out = torch.empty_like(wide)[:, :n]
    for _ in range(5):
        out.fill_(7)
        F.fp8_linear(x, wq, ws, residual=wide[:, :n], out=out, out_dtype=ot)
        assert torch.equal(out, want)


@pytest.mark.parametrize("k", [1, 7, 100, 130, 1001])
def test_bytes_behind_a_row_of_weights_do_not_count(cuda, k):
    """Weights whose rows lie in wider ones, with NaNs right behind them."""
    wide = torch.full((5000, (k + 47) // 16 * 16), 0x7f, dtype=torch.uint8, device=cuda).view(F.E4M3)
    good, ws = weight(cuda, 5000, k, 63)
    wide[:, :k] = good
    for t in (2, 9, 100, 600):
        x = randn(cuda, (t, k), 64, BF)
        check(F.fp8_linear(x, wide[:, :k], ws, out_dtype=F32), x, good, ws)


def test_in_place_residual(cuda):
    for t in (2, 200):
        x, r = randn(cuda, (t, 384), 23, BF), randn(cuda, (t, 500), 24, BF)
        wq, ws = weight(cuda, 500, 384, 25)
        y = F.fp8_linear(x, wq, ws, residual=r)
        assert F.fp8_linear(x, wq, ws, residual=r, out=r) is r and torch.equal(r, y)


def test_repeatable(cuda):
    for t, n in ((1, 2560), (61, 9000), (2043, 2048)):
        x = randn(cuda, (t, 2048), 26, BF)
        wq, ws = weight(cuda, n, 2048, 27)
        y = F.fp8_linear(x, wq, ws, out_dtype=F32)
        for _ in range(5):
            assert torch.equal(F.fp8_linear(x, wq, ws, out_dtype=F32), y)


def test_graphs_and_streams(cuda):
    """Two graphs captured on one stream, replayed at once on two others, beside eager calls."""
    xs = [randn(cuda, (t, 2048), 28 + t, BF) for t in (3, 700)]
    wq, ws = weight(cuda, 2048, 2048, 29)
    F.fp8_linear(xs[0], wq, ws)
    want = [F.fp8_linear(x, wq, ws) for x in xs]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for x in xs:
            F.fp8_linear(x, wq, ws)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append([F.fp8_linear(x, wq, ws) for _ in range(3)])
            graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = F.fp8_linear(xs[1], wq, ws)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[1])
        for w, o in zip(want, outs):
            assert all(torch.equal(w, y) for y in o)
    assert errors() == []
