"""GPU parity: planning a step's pages on the device against lists on the host. Everything is whole numbers and equal."""
import random

import pytest
import torch

from mingmoe import paging as P
from mingmoe.layer import Sequences
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class State:
    """The same state on the device and in lists."""

    def __init__(self, dev, lens, page, columns, spare, seed=0):
        need = [-(-n // page) for n in lens]
        ids = list(range(sum(need) + spare))
        random.Random(seed).shuffle(ids)
        rows, at = [], 0
        for n in need:
            rows.append(ids[at:at + n])
            at += n
        self.dev, self.page, self.columns, self.room = dev, page, columns, len(ids)
        self.host = O.Pages(lens, rows, ids[at:], page)
        wide = torch.full((len(lens), columns + 3), 12345, dtype=torch.int32, device=dev)
        self.pages = wide[:, 1:columns + 1]
        for s, r in enumerate(rows):
            self.pages[s, :len(r)] = ints(r, dev)
        self.lens = ints(lens, dev)
        self.free = ints(ids[at:] + [-1] * at, dev)
        self.n_free = ints([spare], dev)

    def same(self):
        assert self.lens.tolist() == self.host.lens
        n = self.n_free.item()
        assert n == len(self.host.free) and self.free[:n].tolist() == self.host.free
        for s, r in enumerate(self.host.pages):
            assert self.pages[s, :len(r)].tolist() == r

    def step(self, new, seqs, T, max_len=None, **kw):
        step = P.plan_step(ints(new, self.dev), self.lens, self.pages, self.free, self.n_free, page_size=self.page, num_tokens=T,
                           seqs=None if seqs is None else ints(seqs, self.dev), max_len=max_len, **kw)
        order = list(range(len(new))) if seqs is None else seqs
        cu, lens, table, slots, positions, ok = self.host.step(new, order, T, 1 << 30 if max_len is None else max_len, self.columns)
        assert step.ok.item() == ok
        assert step.cu_seqlens.tolist() == cu and step.kv_lens.tolist() == lens
        assert step.slots.tolist() == slots and step.positions.tolist() == positions
        if seqs is None:
            assert step.page_table is self.pages
        else:
            assert step.page_table.tolist() == [r + [0] * (self.columns - len(r)) for r in table]
        if not kw:
            self.same()
        return ok


@pytest.mark.parametrize("page", [8, 16, 256])
@pytest.mark.parametrize("with_seqs", [False, True])
def test_steps(cuda, page, with_seqs):
    """A server's life: prompts, single tokens, empty steps, sequences that end."""
    rnd = random.Random(1)
    st = State(cuda, [0] * 13, page, 40, 600)
    for i in range(12):
        seqs = None
        if with_seqs:
            seqs = rnd.sample(range(13), rnd.randrange(0, 14))
        n = 13 if seqs is None else len(seqs)
        new = [rnd.choice([0, 1, 1, 1, 5, page, 3 * page + 1]) for _ in range(n)]
        assert st.step(new, seqs, sum(new) + rnd.choice([0, 0, 3])) == 1
        if i % 4 == 3:
            gone = rnd.sample(range(13), 4)
            assert P.release_pages(ints(gone, cuda), st.lens, st.pages, st.free, st.n_free, page_size=page).item() == 1
            assert st.host.release(gone, st.room) == 1
            st.same()


@pytest.mark.parametrize("with_seqs", [False, True])
@pytest.mark.parametrize("b,new,T", [(1, 1, 1), (1, 5000, 5001), (1024, 1, 1024), (1025, 2, 2050), (3000, 1, 4000), (40, 300, 12000)])
def test_sizes(cuda, with_seqs, b, new, T):
    rnd = random.Random(b)
    lens = [rnd.randrange(0, 500) for _ in range(b)]
    st = State(cuda, lens, 16, 400, b * (new // 16 + 2), seed=2)
    st.step([new] * b, rnd.sample(range(b), b) if with_seqs else None, T)


def test_refusals_change_nothing(cuda):
    # 14 tokens lie in the two pages that 9 had, and 40 need five: all that are free
    assert State(cuda, [9, 0, 3, 20], 8, 6, 5).step(new=[5, 40], seqs=[0, 1], T=45) == 1
    cases = [dict(new=[5, 41], seqs=[0, 1], T=46),       # more pages than are free
             dict(new=[1, 1], seqs=[2, 2], T=2),         # a sequence twice
             dict(new=[1, 1], seqs=[0, 4], T=2),         # a sequence that is not there
             dict(new=[1, 1], seqs=[-1, 0], T=2),
             dict(new=[1, -1], seqs=[0, 1], T=2),        # a negative count
             dict(new=[3, 3], seqs=[0, 1], T=5),         # more tokens than rows
             dict(new=[1, 12], seqs=[0, 3], T=13, max_len=31),
             dict(new=[2 ** 31 - 1, 0], seqs=[0, 3], T=13),
             dict(new=[2 ** 31 - 1, 2 ** 31 - 1, 2], seqs=[0, 1, 3], T=13, max_len=2 ** 31 - 1),
             dict(new=[0, 0, 0, 200], seqs=None, T=200)]  # more columns than the table has
    for c in cases:
        st = State(cuda, [9, 0, 3, 20], 8, 6, 5)
        assert st.step(**c) == 0, c
        # the same state takes a step that fits
        assert st.step([1, 8], [2, 1], 9) == 1


def test_long_sequences_without_new_tokens(cuda):
    """A sequence at its limit stays in the batch with no token."""
    st = State(cuda, [48, 47], 8, 6, 3)
    assert st.step([0, 1], None, 4) == 1
    assert st.step([0, 1], None, 4) == 0


def test_counters_beside_the_state(cuda):
    """With lens_out and n_free_out the state stays, so a step can be planned again and gives the same."""
    for seqs in (None, [2, 0]):
        st = State(cuda, [9, 30, 3], 8, 10, 9)
        new = [4, 9, 17] if seqs is None else [17, 4]
        lens_out, n_free_out = torch.full_like(st.lens, -7), torch.full_like(st.n_free, -7)
        kw = dict(page_size=8, num_tokens=sum(new) + 1, seqs=None if seqs is None else ints(seqs, cuda), lens_out=lens_out,
                  n_free_out=n_free_out)
        args = (ints(new, cuda), st.lens, st.pages, st.free, st.n_free)
        a = P.plan_step(*args, **kw)
        b = P.plan_step(*args, **kw)
        assert torch.equal(a.slots, b.slots) and torch.equal(a.page_table, b.page_table)
        assert st.lens.tolist() == [9, 30, 3] and st.n_free.item() == 9
        st.host.step(new, [0, 1, 2] if seqs is None else seqs, sum(new) + 1, 1 << 30, 10)
        assert lens_out.tolist() == st.host.lens and n_free_out.item() == len(st.host.free)
        got = [3, 9, 30]
        refused = P.plan_step(ints([10 ** 6] * len(new), cuda), *args[1:], **kw)
        assert refused.ok.item() == 0 and lens_out.tolist() == [9, 30, 3] and n_free_out.item() == 9, got


def test_release(cuda):
    st = State(cuda, [9, 30, 0, 100], 8, 20, 4)
    for gone in ([1, 1], [4], [-1]):
        assert P.release_pages(ints(gone, cuda), st.lens, st.pages, st.free, st.n_free, page_size=8).item() == 0
        st.same()
    short = st.free[:6]  # a stack without room for the pages
    assert P.release_pages(ints([3], cuda), st.lens, st.pages, short, st.n_free, page_size=8).item() == 0
    st.same()
    lens_out, n_free_out = torch.empty_like(st.lens), torch.empty_like(st.n_free)
    assert P.release_pages(ints([3, 2], cuda), st.lens, st.pages, st.free, st.n_free, page_size=8, lens_out=lens_out,
                           n_free_out=n_free_out).item() == 1
    assert st.lens.tolist() == [9, 30, 0, 100] and lens_out.tolist() == [9, 30, 0, 0] and n_free_out.item() == 4 + 13
    assert P.release_pages(ints([3, 2, 0, 1], cuda), st.lens, st.pages, st.free, st.n_free, page_size=8).item() == 1
    assert st.host.release([3, 2, 0, 1], st.room) == 1
    st.same()
    assert P.release_pages(ints([], cuda), st.lens, st.pages, st.free, st.n_free, page_size=8).item() == 1


def test_same_as_the_host_bookkeeping(cuda):
    """DeviceSequences against Sequences, page for page."""
    dev, host = P.DeviceSequences(64, 8, 6, 100), Sequences(64, 8, 6, 100)
    rnd = random.Random(4)
    for i in range(20):
        new = {s: rnd.choice([0, 1, 3, 17]) for s in rnd.sample(range(6), rnd.randrange(1, 7))}
        T = sum(new.values())
        step = dev.extend(ints(list(new.values()), cuda), T, seqs=ints(list(new), cuda))
        try:
            batch = host.extend(new)
        except RuntimeError:
            assert step.ok.item() == 0
            gone = rnd.sample(range(6), 3)
            assert dev.release(ints(gone, cuda)).item() == 1
            for s in gone:
                host.release(s)
            continue
        assert step.ok.item() == 1
        for n in ("cu_seqlens", "kv_lens", "page_table"):
            assert torch.equal(getattr(step, n), getattr(batch, n)), n
        assert dev.lens.tolist() == host.lens and dev.free[:dev.n_free.item()].tolist() == host.free


def test_replayed_graph(cuda):
    """A captured step goes on from the state that the last replay left."""
    dev, host = P.DeviceSequences(200, 8, 4, 300), Sequences(200, 8, 4, 300)
    new = ints([1, 1, 1, 1], cuda)
    dev.extend(ints([5, 16, 0, 31], cuda), 52)
    host.extend({0: 5, 1: 16, 2: 0, 3: 31})
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step = dev.extend(new, 4)
    for i in range(30):
        g.replay()
        batch = host.extend({s: 1 for s in range(4)})
        assert step.ok.item() == 1 and torch.equal(step.kv_lens, batch.kv_lens)
        slots = [host.pages[s][(host.lens[s] - 1) // 8] * 8 + (host.lens[s] - 1) % 8 for s in range(4)]
        assert step.slots.tolist() == slots
