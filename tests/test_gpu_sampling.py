"""GPU parity: tokens drawn from logits against the plain 64-bit implementation. Tokens are equal; the log-probability is off by
its rounding to fp32 (2^-24 of its magnitude) and that of 64-bit sums."""
import math

import pytest
import torch

from mingmoe import sampling as S
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = math.inf, math.nan


def logits_of(dev, b, v, seed, dtype=F32, flat=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(b, v, generator=g, device=dev) * flat).to(dtype)


def uniform(dev, b, seed):
    return torch.rand(b, generator=torch.Generator(device=dev).manual_seed(seed), device=dev)


def check(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    b = logits.shape[0]
    tokens, logprob = S.sample(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p, return_logprob=True)
    assert tokens.dtype == torch.int64 and tokens.shape == logprob.shape == (b,)

    def at(x, r):
        return x[r].item() if torch.is_tensor(x) else torch.tensor(x, dtype=F32).item() if isinstance(x, float) else x

    cpu = logits.cpu()
    for r in range(b):
        want, lp = O.sample(cpu[r], u[r].item(), at(temperature, r), at(top_k, r), at(top_p, r), at(min_p, r))
        assert tokens[r].item() == want, (r, tokens[r].item(), want)
        got = logprob[r].item()
        assert got == lp or abs(got - lp) <= 2.0 ** -24 * abs(lp) + 1e-9, (r, got, lp)
    return tokens


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(top_p=0.3), dict(min_p=0.05),
            dict(temperature=1.5, top_k=300, top_p=0.95, min_p=0.01), dict(temperature=0.0), dict(temperature=0.05, top_p=0.5),
            dict(temperature=4.0, top_p=0.97), dict(top_k=7, top_p=0.5), dict(top_p=0.9, min_p=0.3), dict(temperature=100.0, top_k=900)]


@pytest.mark.parametrize("setting", SETTINGS)
@pytest.mark.parametrize("dtype", [F32, BF, FP])
def test_settings(cuda, setting, dtype):
    for b, v, flat in ((7, 1000, 2.0), (3, 33333, 1.0), (2, 131072, 3.0)):
        check(logits_of(cuda, b, v, 1, dtype, flat), uniform(cuda, b, 2), **setting)


@pytest.mark.parametrize("v", [1, 2, 3, 7, 31, 32, 33, 127, 255, 256, 257, 1023, 1025, 2047, 4099, 8191, 16385, 65537, 200001])
def test_vocabularies(cuda, v):
    for dtype in (F32, BF):
        x, u = logits_of(cuda, 4, v, 3, dtype), uniform(cuda, 4, 4)
        for s in (dict(), dict(top_k=3), dict(top_k=v // 2), dict(top_p=0.8), dict(top_k=40, top_p=0.9, min_p=0.1)):
            check(x, u, **s)


@pytest.mark.parametrize("v,dtype", [(300007, F32), (600011, BF), (800021, F32), (1300021, BF), (2100001, F32)])
def test_rows_that_shared_memory_does_not_hold(cuda, v, dtype):
    x, u = logits_of(cuda, 3, v, 40, dtype), uniform(cuda, 3, 41)
    for s in (dict(), dict(top_k=60, top_p=0.9), dict(top_k=9000), dict(top_p=0.9), dict(top_k=200000, top_p=0.7), dict(min_p=0.01),
              dict(temperature=0.0)):
        check(x, u, **s)


@pytest.mark.parametrize("b", [1, 2, 5, 18, 19, 37, 60, 148, 149, 300])
def test_batches(cuda, b):
    x, u = logits_of(cuda, b, 3001, 5, BF), uniform(cuda, b, 6)
    check(x, u, temperature=0.9, top_k=100, top_p=0.9)
    check(x, u, top_p=0.95)


def test_settings_of_each_row(cuda):
    b = 24
    g = torch.Generator().manual_seed(7)

    def pick(values, dtype):
        return torch.tensor([values[i] for i in torch.randint(0, len(values), (b,), generator=g)], dtype=dtype, device=cuda)

    for v in (999, 50257):
        check(logits_of(cuda, b, v, 8, BF), uniform(cuda, b, 9), temperature=pick([0.0, 0.3, 1.0, 2.0, -1.0, NAN], F32),
              top_k=pick([0, 1, 50, 2000, 10 ** 9, -5], torch.int32), top_p=pick([1.0, 0.9, 0.2, 0.0, 1.5, -1.0, NAN], F32),
              min_p=pick([0.0, 0.1, 1.0, 2.0, -1.0, NAN], F32))


def test_equal_logits(cuda):
    """Borders inside runs of equal logits: the lower indices are kept. All sums are whole numbers times one weight."""
    for v in (5, 1000, 70001):
        x = torch.zeros(6, v, device=cuda)
        x[3:] = torch.randint(0, 3, (3, v), generator=torch.Generator(device=cuda).manual_seed(10), device=cuda).float() * -200
        u = torch.tensor([0.0, 0.25, 0.99, 0.0, 0.5, 0.99], device=cuda)
        for s in (dict(), dict(top_k=3), dict(top_k=max(1, v // 2)), dict(top_p=0.25), dict(top_p=0.75, top_k=max(1, v // 2 + 1)),
                  dict(min_p=1.0), dict(min_p=1.01), dict(temperature=0.0), dict(top_p=0.0)):
            check(x, u, **s)
            check(x.to(BF), u, **s)


def test_equal_logits_over_and_over(cuda):
    """Borders inside runs of equal logits that are searched over all CTAs of a row: the same at each call."""
    x = torch.zeros(3, 70001, device=cuda)
    x[2, ::3] = -200.0
    u = torch.tensor([0.25, 0.99, 0.5], device=cuda)
    for s in (dict(top_p=0.75), dict(top_p=0.75, top_k=35001), dict(top_k=35000)):
        want = [O.sample(x[r].cpu(), u[r].item(), 1.0, s.get("top_k", 0), s.get("top_p", 1.0), 0.0)[0] for r in range(3)]
        got = torch.stack([S.sample(x, u, **s) for _ in range(100)])
        assert got.tolist() == [want] * 100


def test_zeros_of_both_signs_are_equal(cuda):
    x = torch.full((1, 100), -1.0, device=cuda)
    x[0, 10], x[0, 20] = -0.0, 0.0
    for s in (dict(temperature=0.0), dict(top_k=1)):
        assert check(x, uniform(cuda, 1, 11), **s).item() == 10


def test_masked_rows(cuda):
    """-inf, the type's lowest value, NaN, +inf, one token left, none left."""
    for dtype in (F32, BF, FP):
        x = logits_of(cuda, 10, 2000, 12, dtype)
        low = torch.finfo(dtype).min
        x[0, 5:] = -INF
        x[1, :] = -INF
        x[2, :] = -INF
        x[2, 1999] = low
        x[3, 1:] = low
        x[4, 77] = NAN
        x[5, 3], x[5, 9] = INF, INF
        x[6, :] = low
        x[7, :1000] = low
        x[8, ::2] = -INF
        x[9, 0] = torch.finfo(dtype).max
        for s in (dict(), dict(top_k=20), dict(top_k=1500), dict(top_p=0.9), dict(top_p=0.999), dict(min_p=0.1),
                  dict(temperature=0.0), dict(temperature=0.01), dict(top_k=1999, top_p=0.5)):
            check(x, uniform(cuda, 10, 13), **s)


def test_extreme_numbers(cuda):
    x = logits_of(cuda, 6, 5000, 14)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, NAN], device=cuda)
    for s in (dict(), dict(top_k=10), dict(top_p=0.9)):
        check(x, u, **s)
    v = uniform(cuda, 6, 15)
    for scale, s in ((1e30, dict()), (1e-30, dict(top_p=0.5)), (1.0, dict(temperature=1e-30)), (1.0, dict(temperature=1e30, top_k=77)),
                     (1e-3, dict(temperature=1e-3, top_k=200, top_p=0.7))):
        check(x * scale, v, **s)


@pytest.mark.parametrize("temperature", [0.001, 1.0, 50.0, 200.0])
def test_logits_that_lie_far_apart_for_the_temperature(cuda, temperature):
    """Neighbouring numbers of the logits' size are further apart than weights reach: the least logit of weight has none below it."""
    for step, size in ((64.0, 1e9), (0.0625, 1e6), (2.0 ** -19, 12.0)):
        t = temperature * step / 64
        g = torch.Generator(device=cuda).manual_seed(50)
        for lowest in (2, 4000):
            x = size - step * torch.randint(0, lowest, (5, 9001), generator=g, device=cuda).float()
            x[3:] = size - step  # one at the top, all others next to it
            x[3, 4444] = size
            x[4, 17] = size
            for s in (dict(), dict(top_p=0.9), dict(top_k=3000), dict(top_k=3000, top_p=0.6), dict(top_k=40, top_p=0.8), dict(min_p=0.02)):
                check(x, uniform(cuda, 5, 51), temperature=t, **s)


def test_numbers_at_the_ends_of_the_type(cuda):
    """Distances that pass the largest number, temperatures below the least normal one and infinite ones."""
    top = torch.finfo(F32).max
    x = logits_of(cuda, 4, 9001, 52)
    x[0, ::2], x[0, 1::2] = top, -top
    x[1] *= 1e38
    x[2] = x[2].clamp(-1, 1) * top
    x[3, 5:] *= 1e-42
    for t in (1e-45, 1e-40, 1e-38, 1.0, 1e38, top, INF):
        for s in (dict(), dict(top_p=0.9), dict(top_k=3000), dict(top_k=3000, top_p=0.6), dict(top_k=40, top_p=0.8), dict(min_p=0.02)):
            check(x, uniform(cuda, 4, 53), temperature=t, **s)


def test_strides_and_out(cuda):
    big = logits_of(cuda, 9, 4100, 16, BF)
    u = uniform(cuda, 4, 17)
    for off in (0, 1, 3, 8):
        for v in (1000, 1001, 4000):
            check(big[1::2, off:off + v], u, top_k=30)
            check(big[1::2, off:off + v], u, top_p=0.9)
    check(big.t().contiguous().t()[:4, :900], u, top_k=5)
    out = torch.full((4,), 7, dtype=torch.int64, device=cuda)
    assert S.sample(big[:4], u, out=out) is out and torch.equal(out, S.sample(big[:4], u))
    check(big[:0], u[:0])
    assert S.sample(big[:3, :0], u[:3]).tolist() == [-1] * 3


def test_distribution_follows_the_weights(cuda):
    """4096 even steps of u through one row give each kept token its share of them, to within one step at each end."""
    x = logits_of(cuda, 1, 50, 18)
    n = 4096
    u = (torch.arange(n, device=cuda) + 0.5) / n
    tokens = S.sample(x.expand(n, 50), u, top_k=8)
    p = torch.zeros(50, dtype=torch.float64, device=cuda)
    best = x[0].topk(8).indices
    p[best] = torch.softmax(x[0, best].double(), 0)
    count = torch.bincount(tokens, minlength=50)
    assert bool(((count - n * p).abs() <= 1 + 1e-6).all())


def test_replayed_graph_and_streams(cuda):
    xs = [logits_of(cuda, 5, 40001, 19), logits_of(cuda, 100, 5003, 20, BF)]
    us = [uniform(cuda, x.shape[0], 21) for x in xs]
    kw = dict(temperature=0.9, top_k=0, top_p=0.95)
    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for x, u in zip(xs, us):
            S.sample(x, u, **kw)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(S.sample(x, u, **kw))
            graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for i in range(6):
        for x, u in zip(xs, us):
            u.copy_(uniform(cuda, u.shape[0], 30 + i))
        want = [S.sample(x, u, **kw) for x, u in zip(xs, us)]
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_repeatable(cuda):
    x, u = logits_of(cuda, 40, 131072, 22, F32, 1.0), uniform(cuda, 40, 23)
    for s in (dict(), dict(top_p=0.9), dict(top_k=3000)):
        t, p = S.sample(x, u, return_logprob=True, **s)
        for _ in range(5):
            t2, p2 = S.sample(x, u, return_logprob=True, **s)
            assert torch.equal(t, t2) and torch.equal(p, p2)
