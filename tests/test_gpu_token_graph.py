"""The captured token step where it cannot go on as it was asked to: no room for its pages, a row of logits without a token."""
import pytest
import torch

from mingmoe import _lib as L
from mingmoe import fp8, sampling
from mingmoe.attention import rotation_table
from mingmoe.block import MoeBlock
from mingmoe.graphs import TokenGraph
from mingmoe.layer import AttentionBlock, Decoder, DecoderLayer, Sequences
from mingmoe.paging import DeviceSequences
from oracle import moe_oracle as MO

pytestmark = pytest.mark.gpu

H, HQ, HKV, D, V = 256, 4, 2, 64, 501


def make(dev, seqs, layers=1):
    g = torch.Generator().manual_seed(0)
    w = lambda *s: (torch.randn(*s, generator=g) * 0.05).to(torch.bfloat16).to(dev)
    one = torch.ones(H, dtype=torch.bfloat16, device=dev)
    stack = []
    for i in range(layers):
        attn = AttentionBlock(fp8.quantize_fp8_weight(w((HQ + 2 * HKV) * D, H)), fp8.quantize_fp8_weight(w(H, HQ * D)), one, HQ, HKV, D,
                              rotation_table(256, D, device=dev))
        block = MoeBlock.from_params(MO.make_block_params(seed=i, H=H, I=128, E=16, I_s=256), top_k=4)
        stack.append(DecoderLayer(attn, block, seqs.cache(attn)))
    return Decoder(w(V, H) * 20, stack, one, fp8.quantize_fp8_weight(w(V, H) * 4))


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def test_a_step_without_room_keeps_the_tokens(cuda):
    """Three sequences over pages of 8, two of which need a page at once where one is left: the step changes nothing, and the loop goes on
    once one sequence has given its pages back, with the tokens of a loop that always had room."""
    prompt = torch.randint(0, V, (22,), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda)
    lens = [7, 7, 8]
    loops = []
    for pages in (5, 50):
        seqs = DeviceSequences(pages, 8, 3, 64, device=cuda)
        loop = TokenGraph(make(cuda, seqs), seqs)
        loop.decoder(prompt, seqs.extend(ints(lens, cuda), 22, max_q=8, prompts=True))
        loop.tokens.copy_(torch.tensor([11, 12, 13]))
        loop.new.fill_(1)
        loops.append(loop)
    tight, wide = loops
    host = Sequences(5, 8, 3, 64, device=cuda)
    host.extend(dict(enumerate(lens)))
    refused = []
    for i in range(10):
        u = torch.rand(3, generator=torch.Generator(device=cuda).manual_seed(10 + i), device=cuda)
        for loop in loops:
            loop.u.copy_(u)
        before = tight.tokens.tolist()
        tight()
        try:
            host.extend({s: 1 for s in range(3 - len(refused))})
        except RuntimeError:
            refused.append(i)
            for _ in range(2):
                assert tight.ok.item() == 0 and tight.tokens.tolist() == before
                assert tight.seqs.lens.tolist() == host.lens and tight.seqs.n_free.item() == len(host.free)
                tight()
            host.release(2)
            for loop in loops:
                loop.new[2] = 0
                assert loop.seqs.release(ints([2], cuda)).item() == 1
            continue
        wide()
        assert tight.ok.item() == wide.ok.item() == 1 and tight.tokens.tolist() == wide.tokens.tolist()
        assert tight.seqs.lens.tolist() == wide.seqs.lens.tolist() == host.lens
    assert refused == [1] and tight.tokens.tolist() != [11, 12, 13]
    assert not L.all_workspace_errors()


def test_a_sequence_without_a_token_stops(cuda):
    """A row whose logits hold no token gives -1, which is no token of the next step: the sequence idles until the caller puts one there."""
    seqs = DeviceSequences(20, 8, 3, 64, device=cuda)
    inner = make(cuda, seqs)
    grammar = torch.full((V,), False, device=cuda)
    grammar[7] = True  # nothing may follow token 7

    def decoder(tokens, batch):
        last = tokens[(batch.cu_seqlens[1:] - 1).clamp(min=0)]
        return inner(tokens, batch).masked_fill(grammar[last][:, None], -float("inf"))

    loop = TokenGraph(decoder, seqs)
    inner(torch.arange(9, device=cuda), seqs.extend(ints([3, 2, 4], cuda), 9, max_q=4, prompts=True))
    loop.tokens.copy_(torch.tensor([1, 7, 2]))
    loop.new.fill_(1)
    loop.temperature.zero_()
    loop()
    assert loop.tokens[1].item() == -1 and loop.logprob[1].item() == -float("inf") and seqs.lens.tolist() == [4, 3, 5]
    others = loop.tokens[[0, 2]]
    assert bool((others >= 0).all()) and not bool((others == 7).any())
    loop()
    assert loop.ok.item() == 1 and loop.tokens[1].item() == -1 and seqs.lens.tolist() == [5, 3, 6]
    loop.tokens[1] = 9
    loop()
    assert loop.tokens[1].item() >= 0 and seqs.lens.tolist() == [6, 4, 7]
    assert not L.all_workspace_errors()


def test_results_are_the_last_steps_whether_captured_or_not(cuda):
    """Steps one by one between replays: logits, logprob and ok are those of the step that came last."""
    seqs = DeviceSequences(3, 8, 2, 64, device=cuda)
    loop = TokenGraph(make(cuda, seqs), seqs)
    loop.decoder(torch.arange(10, device=cuda), seqs.extend(ints([6, 4], cuda), 10, max_q=6, prompts=True))
    loop.new.fill_(1)
    for i, step in enumerate([loop, loop.step, loop, loop, loop.step, loop, loop.step, loop]):
        loop.u.copy_(torch.rand(2, generator=torch.Generator(device=cuda).manual_seed(i), device=cuda))
        before = seqs.lens.tolist()
        step()
        fits = sum(-(-(n + 1) // 8) for n in before) <= 3
        assert loop.ok.item() == fits
        if fits:
            drawn, logprob = sampling.sample(loop.logits, loop.u, return_logprob=True)
            assert torch.equal(drawn, loop.tokens) and torch.equal(logprob, loop.logprob)
        else:
            assert seqs.lens.tolist() == before
    assert not fits
