"""GPU parity of drawing tokens from unusual rows in every launch shape: up to 26 rows (CTAs of 512 threads), more (256 threads, one to
eight CTAs a row), rows too long for three CTAs on an SM, and rows that shared memory does not hold. A few rows are repeated over the
batch, and each copy is compared with the plain 64-bit draw."""
import math

import pytest
import torch

from mingmoe import sampling as S
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = math.inf, math.nan

SHAPES = [(3, 2000), (26, 9001), (27, 9001), (40, 50257), (150, 9001), (300, 2000), (300, 9001), (30, 131072)]
LONG = [(40, 300007, F32), (30, 600011, BF), (300, 300007, FP)]


def check(x, u, b, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    n = x.shape[0]
    at = torch.arange(b, device=x.device) % n
    tokens, logprob = S.sample(x[at], u[at], temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, return_logprob=True)
    f32 = lambda v: torch.tensor(v, dtype=F32).item()
    want = [O.sample(row, v, f32(temperature), top_k, f32(top_p), f32(min_p)) for row, v in zip(x.cpu(), u.tolist())]
    assert tokens.tolist() == [want[i % n][0] for i in range(b)]
    for i, got in enumerate(logprob.tolist()):
        p = want[i % n][1]
        # weights are rounded to half a unit each, of which a row of v has 2^(61 - log2 v) and 2^51 at most to its largest weight
        v = x.shape[1]
        assert got == p or abs(got - p) <= 2.0 ** -24 * abs(p) + v * 2.0 ** -min(52, 62 - math.ceil(math.log2(v))) + 1e-12, (i, got, p)


def randn(dev, b, v, seed, flat=2.0):
    return torch.randn(b, v, generator=torch.Generator(device=dev).manual_seed(seed), device=dev) * flat


def uniform(dev, b, seed):
    return torch.rand(b, generator=torch.Generator(device=dev).manual_seed(seed), device=dev)


@pytest.mark.parametrize("b,v", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF, FP])
def test_settings(cuda, b, v, dtype):
    x, u = randn(cuda, 5, v, 1).to(dtype), uniform(cuda, 5, 2)
    for s in (dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(top_p=0.3), dict(min_p=0.05),
              dict(min_p=0.0001), dict(temperature=1.5, top_k=300, top_p=0.95, min_p=0.01), dict(temperature=0.0),
              dict(temperature=0.05, top_p=0.5), dict(temperature=4.0, top_p=0.97), dict(top_k=v // 2), dict(top_k=v // 2, top_p=0.8),
              dict(top_p=0.9, min_p=0.3), dict(temperature=100.0, top_k=900), dict(temperature=100.0, min_p=0.9)):
        check(x, u, b, **s)


@pytest.mark.parametrize("b,v", SHAPES)
@pytest.mark.parametrize("dtype", [F32, BF, FP])
def test_masked_rows(cuda, b, v, dtype):
    """-inf, the type's lowest value, NaN, +inf, one token left, none left."""
    x = randn(cuda, 10, v, 12).to(dtype)
    low = torch.finfo(dtype).min
    x[0, 5:] = -INF
    x[1, :] = -INF
    x[2, :] = -INF
    x[2, v - 1] = low
    x[3, 1:] = low
    x[4, 77] = NAN
    x[5, 3], x[5, 9], x[5, v - 2] = INF, INF, INF
    x[6, :] = low
    x[7, :v // 2] = low
    x[8, ::2] = -INF
    x[9, 0] = torch.finfo(dtype).max
    for s in (dict(), dict(top_k=20), dict(top_k=1500), dict(top_p=0.9), dict(top_p=0.999), dict(min_p=0.1), dict(temperature=0.0),
              dict(temperature=0.01), dict(top_k=1999, top_p=0.5)):
        check(x, uniform(cuda, 10, 13), b, **s)


@pytest.mark.parametrize("b,v", SHAPES)
def test_equal_logits(cuda, b, v):
    """Borders inside runs of equal logits, longer than any list. All sums are whole numbers times one weight."""
    x = torch.zeros(6, v, device=cuda)
    x[3:] = torch.randint(0, 3, (3, v), generator=torch.Generator(device=cuda).manual_seed(10), device=cuda).float() * -200
    u = torch.tensor([0.0, 0.25, 0.99, 0.0, 0.5, 0.99], device=cuda)
    for s in (dict(), dict(top_k=3), dict(top_k=v // 2), dict(top_p=0.25), dict(top_p=0.75, top_k=v // 2 + 1), dict(min_p=1.0), dict(min_p=0.5),
              dict(min_p=1.01), dict(temperature=0.0), dict(top_p=0.0)):
        check(x, u, b, **s)
        check(x.to(BF), u, b, **s)


@pytest.mark.parametrize("b,v", SHAPES)
@pytest.mark.parametrize("temperature", [0.001, 1.0, 200.0])
def test_logits_that_lie_far_apart_for_the_temperature(cuda, b, v, temperature):
    for step, size in ((64.0, 1e9), (0.0625, 1e6), (2.0 ** -19, 12.0)):
        t = temperature * step / 64
        g = torch.Generator(device=cuda).manual_seed(50)
        for lowest in (2, 4000):
            x = size - step * torch.randint(0, lowest, (5, v), generator=g, device=cuda).float()
            x[3:] = size - step
            x[3, v // 2] = size
            x[4, 17] = size
            for s in (dict(), dict(top_p=0.9), dict(top_k=1500), dict(top_k=1500, top_p=0.6), dict(top_k=40, top_p=0.8), dict(min_p=0.02)):
                check(x, uniform(cuda, 5, 51), b, temperature=t, **s)


@pytest.mark.parametrize("b,v", SHAPES)
def test_numbers_at_the_ends_of_the_type(cuda, b, v):
    top = torch.finfo(F32).max
    x = randn(cuda, 4, v, 52)
    x[0, ::2], x[0, 1::2] = top, -top
    x[1] *= 1e38
    x[2] = x[2].clamp(-1, 1) * top
    x[3, 5:] *= 1e-42
    for t in (1e-45, 1e-40, 1e-38, 1.0, 1e38, top, INF):
        for s in (dict(), dict(top_p=0.9), dict(top_k=1500), dict(top_k=1500, top_p=0.6), dict(top_k=40, top_p=0.8), dict(min_p=0.02)):
            check(x, uniform(cuda, 4, 53), b, temperature=t, **s)


@pytest.mark.parametrize("b,v,dtype", LONG)
def test_rows_that_shared_memory_does_not_hold(cuda, b, v, dtype):
    x, u = randn(cuda, 3, v, 40).to(dtype), uniform(cuda, 3, 41)
    for s in (dict(), dict(top_k=60, top_p=0.9), dict(top_k=9000), dict(top_p=0.9), dict(top_k=200000, top_p=0.7), dict(min_p=0.01),
              dict(temperature=0.0)):
        check(x, u, b, **s)


@pytest.mark.parametrize("b", [1, 26, 27, 74, 130, 260, 300])
def test_settings_of_each_row(cuda, b):
    g = torch.Generator().manual_seed(7)
    v = 5003

    def pick(values, dtype):
        return torch.tensor([values[i] for i in torch.randint(0, len(values), (b,), generator=g)], dtype=dtype, device=cuda)

    x, u = randn(cuda, b, v, 8).to(FP), uniform(cuda, b, 9)
    t, k = pick([0.0, 0.3, 1.0, 2.0, -1.0, NAN], F32), pick([0, 1, 50, 2000, 10 ** 9, -5], torch.int32)
    p, m = pick([1.0, 0.9, 0.2, 0.0, 1.5, -1.0, NAN], F32), pick([0.0, 0.1, 1.0, 2.0, -1.0, NAN], F32)
    tokens = S.sample(x, u, temperature=t, top_k=k, top_p=p, min_p=m)
    want = [O.sample(x[r].cpu(), u[r].item(), t[r].item(), k[r].item(), p[r].item(), m[r].item())[0] for r in range(b)]
    assert tokens.tolist() == want
