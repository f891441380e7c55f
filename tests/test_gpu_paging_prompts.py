"""Plans of prompts: a sequence that has tokens takes no more of them as a prompt, since those would attend to one another alone."""
import pytest
import torch

from mingmoe import _serving
from mingmoe import paging as P

pytestmark = pytest.mark.gpu


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


class Behind:
    """The C++ module as if nothing fitted it: every call goes through the Python code."""
    plan_step = staticmethod(lambda *a: NotImplemented)


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    _serving.host()
    if request.param == "python":
        monkeypatch.setattr(_serving, "_module", Behind)


def test_prompts_of_sequences_that_have_tokens_are_refused(cuda, path):
    seqs = P.DeviceSequences(40, 8, 4, 100, device=cuda)
    assert seqs.extend(ints([9, 5], cuda), 14, seqs=ints([0, 2], cuda), prompts=True).ok.item() == 1
    for new, which in (([3, 4], [1, 0]), ([4, 3], [2, 1]), ([1, 0, 0, 0], None), ([1, 2, 3, 4], None)):
        step = seqs.extend(ints(new, cuda), 10, seqs=None if which is None else ints(which, cuda), prompts=True)
        assert step.ok.item() == 0 and step.cu_seqlens.tolist() == [0] * (len(new) + 1) and step.slots.tolist() == [-1] * 10
        assert seqs.lens.tolist() == [9, 0, 5, 0] and seqs.n_free.item() == 40 - 3
    # sequences that get no token may have some, and the same tokens are no prompts without the flag
    step = seqs.extend(ints([0, 7, 0, 0], cuda), 10, max_q=7, prompts=True)
    assert step.ok.item() == 1 and step.prompts and seqs.lens.tolist() == [9, 7, 5, 0]
    assert seqs.extend(ints([3, 4], cuda), 10, seqs=ints([3, 0], cuda)).ok.item() == 1
    assert seqs.lens.tolist() == [13, 7, 5, 3]
    # a sequence that has given its pages back begins anew
    assert seqs.release(ints([2], cuda)).item() == 1
    assert seqs.extend(ints([20], cuda), 20, seqs=ints([2], cuda), prompts=True).ok.item() == 1


def test_large_steps_of_prompts(cuda):
    """The same where the tokens are written by a kernel of their own."""
    seqs = P.DeviceSequences(600, 16, 5, 4000, device=cuda)
    assert seqs.extend(ints([1, 3000], cuda), 3001, seqs=ints([4, 1], cuda), prompts=True).ok.item() == 1
    assert seqs.extend(ints([2500, 2], cuda), 2502, seqs=ints([0, 4], cuda), prompts=True).ok.item() == 0
    assert seqs.lens.tolist() == [0, 3000, 0, 0, 1]
    assert seqs.extend(ints([2500, 2], cuda), 2502, seqs=ints([0, 3], cuda), prompts=True).ok.item() == 1
