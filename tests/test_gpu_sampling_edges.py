"""GPU parity of drawing tokens where rows fill the lists and histograms, in each of the launch's shapes: batches of up to 26 rows (CTAs of
512 threads), of more (256 threads, one to eight CTAs a row), and of rows too long for three of those on an SM."""
import math

import pytest
import torch

from mingmoe import sampling as S
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def expected(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    f32 = lambda v: torch.tensor(v, dtype=F32).item()
    return O.sample(row, u, f32(temperature), top_k, f32(top_p), f32(min_p))


def check_copies(x, u, b, **s):
    """The rows of x over and over, b in all, each against the plain draw."""
    n = x.shape[0]
    at = torch.arange(b, device=x.device) % n
    tokens, logprob = S.sample(x[at], u[at], return_logprob=True, **s)
    want = [expected(row, v, **s) for row, v in zip(x.cpu(), u.tolist())]
    assert tokens.tolist() == [want[i % n][0] for i in range(b)], s
    for r, got in enumerate(logprob.tolist()):
        p = want[r % n][1]
        assert got == p or abs(got - p) <= 2.0 ** -24 * abs(p) + 1e-9, (r, got, p, s)


# rows and vocabularies of the three launch shapes
SHAPES = [(3, 9001, F32), (40, 9001, F32), (300, 9001, F32), (40, 70001, BF), (30, 131072, F32)]


def unit(v):
    """The number whose multiples weights of v tokens are."""
    return 2.0 ** -min(51, 61 - max(1, math.ceil(math.log2(v))))


@pytest.mark.parametrize("b", [1, 26, 27, 60, 300])
@pytest.mark.parametrize("v", [2047, 2048, 2049, 4095, 4096, 4097])
def test_equal_logits_that_fill_a_list(cuda, b, v):
    """All logits equal: the whole row is one bin of the histogram and of each finer one, up to the list's last place."""
    x = torch.zeros(b, v, device=cuda)
    u = (torch.arange(b, device=cuda) * 0.6180339887) % 1.0
    for s in (dict(top_p=0.9), dict(top_p=0.25), dict(top_k=50, top_p=0.9), dict(top_k=v - 1, top_p=0.75), dict(top_k=v // 2),
              dict(min_p=0.5), dict(top_p=0.5, min_p=0.5)):
        want = [expected(x[0].cpu(), n, **s) for n in u.tolist()]
        tokens, logprob = S.sample(x, u, return_logprob=True, **s)
        assert tokens.tolist() == [t for t, _ in want], s
        assert all(abs(got - p) <= 2.0 ** -24 * abs(p) + 1e-9 for got, (_, p) in zip(logprob.tolist(), want)), s


@pytest.mark.parametrize("v", [1500, 2048, 17000, 70001])
def test_the_unit_of_weights_goes_by_the_vocabulary_alone(cuda, v):
    """u = 0 draws the first token with a weight: one of 0.6 units has one and one of 0.4 has none, whatever the batch."""
    f = [0.4, 0.45, 0.55, 0.6, 0.9]
    x = torch.full((len(f), v), -1.0, device=cuda)
    x[:, 0] = torch.tensor([math.log(n * unit(v)) for n in f])
    x[:, 1] = 0.0
    u = torch.zeros(len(f), device=cuda)
    results = []
    for copies in (1, 6, 12, 60):
        tokens, logprob = S.sample(x.repeat(copies, 1), u.repeat(copies), return_logprob=True)
        assert tokens.tolist() == [int(n < 0.5) for n in f] * copies
        results.append(logprob.view(copies, len(f)))
    assert all(torch.equal(r, results[0].expand_as(r)) for r in results)


@pytest.mark.parametrize("b,v,dtype", SHAPES)
@pytest.mark.parametrize("n", [1, 2, 127, 128, 129, 255, 256, 257, 511, 513, 2047, 2048, 2049, 4095, 4096, 4097, 9000])
def test_lists_of_every_length(cuda, b, v, dtype, n):
    """n candidates that min_p leaves, or that top-k and top-p choose from."""
    g = torch.Generator(device=cuda).manual_seed(n)
    x = torch.full((5, v), -30.0, device=cuda)
    for r in range(5):
        x[r, torch.randperm(v, generator=g, device=cuda)[:n]] = torch.randn(n, generator=g, device=cuda).clamp(-3, 3)
    x, u = x.to(dtype), torch.rand(5, generator=g, device=cuda)
    for s in (dict(min_p=0.0005), dict(top_k=n), dict(top_k=n, top_p=0.8), dict(top_k=max(1, n - 1), min_p=0.01), dict(top_p=0.7)):
        check_copies(x, u, b, **s)


@pytest.mark.parametrize("b,v,dtype", [*SHAPES, (3, 131072, F32), (2, 800021, F32)])
def test_log_probabilities_of_unlikely_tokens(cuda, b, v, dtype):
    """u = 0 draws the first kept token, whose weight is only some thousand units: its log-probability is off by its rounding to fp32
    and by what the rounded weights, half a unit each, make of their sum."""
    g = torch.Generator(device=cuda).manual_seed(1)
    for n, settings in ((120, (dict(), dict(top_k=150), dict(min_p=1e-12), dict(top_k=150, temperature=1.25))),
                        (1500, (dict(), dict(top_k=1600), dict(min_p=1e-12), dict(temperature=0.75)))):
        x = torch.full((5, v), -60.0, device=cuda)
        for r in range(5):
            x[r, torch.randperm(v, generator=g, device=cuda)[:n]] = -2.0 - 16.0 * torch.rand(n, generator=g, device=cuda)
            x[r, 0], x[r, 7] = -18.0 - r, 0.0
        x, u = x.to(dtype), torch.zeros(b, device=cuda)
        for s in settings:
            tokens, logprob = S.sample(x[torch.arange(b, device=cuda) % 5], u, return_logprob=True, **s)
            want = [expected(row, 0.0, **s) for row in x.cpu()]
            assert [t for t, _ in want] == [0] * 5 and tokens.tolist() == [0] * b
            for i, got in enumerate(logprob.tolist()):
                p = want[i % 5][1]
                assert abs(got - p) <= 2.0 ** -24 * abs(p) + v * unit(v) / 2, (i, got, p, s)


@pytest.mark.parametrize("v", [1 << 17, 1 << 19, (1 << 22) - 5])
@pytest.mark.parametrize("units", [0.45, 0.55, 1.45])
def test_tails_of_about_a_unit(cuda, v, units):
    """Weights are rounded to whole units, so a running sum is off by half a unit a token: the token drawn is the definition's but for
    that, whatever the tail adds up to."""
    at = v // 3
    x = torch.full((1, v), math.log(units * unit(v)), device=cuda)
    x[0, at] = 0.0
    run = torch.cumsum(torch.exp(x[0].double()), 0)
    total, off = run[-1].item(), v * unit(v) / 2
    for u in (0.0, 1e-7, 2.0 ** -24, 0.5, 1.0 - 2.0 ** -23, 1.0 - 2.0 ** -24):
        t = S.sample(x, torch.tensor([u], device=cuda))[0].item()
        f = torch.tensor(u, dtype=F32).item()
        assert run[t].item() > f * total - off * (1 + f)
        assert t == 0 or run[t - 1].item() <= f * total + off * (1 + f)
        if units < 0.5:
            assert t == at  # the tail has no weight
        if u == 0.0:
            assert t == (at if units < 0.5 else 0)
