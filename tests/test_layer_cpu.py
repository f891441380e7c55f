"""Host bookkeeping of the decoder layer's sequences (no GPU): what a refused step leaves behind."""
import copy

import pytest

from mingmoe.layer import Sequences


def state(seqs):
    return copy.deepcopy((seqs.lens, seqs.pages, seqs.free))


@pytest.mark.parametrize("new,prompts,exc", [
    ({0: 1, 1: 65}, False, RuntimeError),         # the second sequence is longer than its row of the page table
    ({0: 20, 2: 64}, False, RuntimeError),        # each fits alone, the pages do not do for both
    ({2: 20, 0: 1}, True, ValueError),            # the second sequence has tokens already
    ({2: 1, 9: 1}, False, IndexError)])           # no such sequence
def test_refused_step_changes_nothing(new, prompts, exc):
    seqs = Sequences(num_pages=6, page_size=16, max_seqs=3, max_len=64, device="cpu")
    seqs.extend({0: 21}, prompts=True)
    before = state(seqs)
    with pytest.raises(exc):
        seqs.extend(new, prompts=prompts)
    assert state(seqs) == before
    # the same step in parts that fit goes on where the sequences were
    batch = seqs.extend({0: 1, 2: 2})
    assert batch.kv_lens.tolist() == [22, 2] and batch.cu_seqlens.tolist() == [0, 1, 3] and seqs.lens == [22, 0, 2]
    assert len(seqs.free) == 6 - 2 - 1


def test_pages_in_order_and_given_back():
    seqs = Sequences(num_pages=5, page_size=8, max_seqs=2, max_len=32, device="cpu")
    batch = seqs.extend({1: 9, 0: 8}, prompts=True)
    assert batch.page_table.tolist() == [[0, 1, 0, 0], [2, 0, 0, 0]] and batch.max_q == 9 and batch.prompts
    seqs.release(1)
    assert seqs.lens == [8, 0] and sorted(seqs.free) == [0, 1, 3, 4]
    empty = seqs.extend({})
    assert empty.page_table.shape == (0, 4) and empty.cu_seqlens.tolist() == [0] and empty.max_q == 0


@pytest.mark.parametrize("new,exc", [({0: 51}, RuntimeError), ({1: 50, 0: 51}, RuntimeError), ({0: -1}, ValueError)])
def test_lengths_stay_within_max_len(new, exc):
    """max_len inside a page: the page's other slots are no room (a rotation table of max_len rows has none for them)."""
    seqs = Sequences(num_pages=9, page_size=16, max_seqs=2, max_len=50, device="cpu")
    before = state(seqs)
    with pytest.raises(exc):
        seqs.extend(new)
    assert state(seqs) == before
    assert seqs.extend({0: 50}).kv_lens.tolist() == [50]
    with pytest.raises(RuntimeError):
        seqs.extend({0: 1})
