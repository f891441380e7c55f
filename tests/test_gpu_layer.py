"""The decoder layer on the paged cache: prompts, a chunk of new tokens and single tokens through the attention half and
the MoE block, as they would be used; and a captured step.

Each stage is checked from the GPU's own input of that stage: the projections are calls tested elsewhere; the attended
heads lie within the bound that oracle.attention_oracle derives, over keys the test keeps itself; the MoE block within
BASELINE's tolerance of its oracle (max-abs 2e-2, mean-rel 1e-2, mean-rel being sum|got - ref| / sum|ref|)."""
import pytest
import torch

from mingmoe import _lib as L
from mingmoe.attention import kv_append, rotation_table
from mingmoe.block import MoeBlock
from mingmoe.layer import AttentionBlock, DecoderLayer, Sequences
from oracle import attention_oracle as AO
from oracle import moe_oracle as O

pytestmark = pytest.mark.gpu

H, HQ, HKV, D = 512, 8, 2, 64


def close(got, ref, max_abs=2e-2, mean_rel=1e-2):
    d = (got.double().cpu() - ref.double().cpu()).abs()
    assert d.max().item() <= max_abs, d.max().item()
    assert (d.sum() / ref.double().cpu().abs().sum()).item() <= mean_rel


def make(cuda, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = lambda *s: (torch.randn(*s, generator=g) * 0.05).to(torch.bfloat16).to(cuda)
    attn = AttentionBlock(w((HQ + 2 * HKV) * D, H), w(H, HQ * D), torch.ones(H, dtype=torch.bfloat16, device=cuda), HQ, HKV,
                          D, rotation_table(512, D, device=cuda))
    p = O.make_block_params(seed=seed, H=H, I=128, E=16, I_s=256)
    return attn, p, MoeBlock.from_params(p, top_k=4)


def test_prompts_chunks_and_tokens(cuda):
    attn, p, block = make(cuda)
    seqs = Sequences(num_pages=64, page_size=16, max_seqs=4, max_len=400, device=cuda)
    layer = DecoderLayer(attn, block, seqs.cache(attn))
    k, v = {}, {}  # per sequence: the keys, rotated and rounded as they should lie in the cache, and the values
    steps = [({0: 37, 2: 150}, True), ({1: 5}, True), ({0: 1, 2: 1, 1: 1}, False), ({2: 90, 0: 3}, False),
             ({0: 2, 1: 1, 2: 4}, False), ({1: 1}, False)]
    for step, (new, prompts) in enumerate(steps):
        x = O.make_tokens(sum(new.values()), H=H, seed=step).to(cuda)
        batch = seqs.extend(new, prompts=prompts)
        qkv = attn.project(x)
        o = attn.attend(qkv, layer.cache, batch)
        at = 0
        for row, (s, n) in enumerate(new.items()):
            part = qkv[at:at + n]
            total = seqs.lens[s]
            pos = torch.arange(total - n, total, device=cuda)
            got_k = AO.gather(layer.cache.k, batch.page_table[row], total)
            got_v = AO.gather(layer.cache.v, batch.page_table[row], total)
            want, tol = AO.rotate(part[:, HQ:HQ + HKV], attn.cos_sin, pos, False)
            assert bool(((got_k[-n:].double() - want).abs() <= tol).all())
            # what was there stays there, the new values are copies
            if s in k:
                assert torch.equal(got_k[:-n], k[s]) and torch.equal(got_v[:-n], v[s])
            assert torch.equal(got_v[-n:], part[:, HQ + HKV:])
            k[s], v[s] = got_k, got_v
            # the rotated queries of this call: the same operator into a cache that nobody reads
            q = kv_append(seqs.cache(attn), part[:, HQ:HQ + HKV], part[:, HQ + HKV:], batch.page_table[row:row + 1],
                          torch.tensor([0, n], dtype=torch.int32, device=cuda), batch.kv_lens[row:row + 1],
                          q=part[:, :HQ], cos_sin=attn.cos_sin)
            want, tol = AO.rotate(part[:, :HQ], attn.cos_sin, pos, False)
            assert bool(((q.double() - want).abs() <= tol).all())
            want, _, tol, _ = AO.attention_fast(q, k[s], v[s], True)
            assert bool(((o[at:at + n].double() - want).abs() <= tol).all()), (step, s)
            at += n
        h = attn(x, layer.cache, batch)  # appends the same tokens to the same slots again
        assert torch.equal(h, attn.output(o, x))
        close(layer(x, batch), O.moe_block(h.cpu(), p, top_k=4)[0])
    assert seqs.lens[:3] == [43, 8, 245]
    seqs.release(2)
    assert len(seqs.free) == 64 - 3 - 1
    with pytest.raises(RuntimeError):
        seqs.extend({3: 401})
    with pytest.raises(ValueError):
        seqs.extend({0: 4}, prompts=True)
    assert not L.all_workspace_errors()


def test_captured_token_step(cuda):
    """One token of two sequences through two layers in a CUDA graph, replayed as the sequences grow."""
    layers, seqs = [], Sequences(num_pages=32, page_size=16, max_seqs=2, max_len=200, device=cuda)
    for seed in (1, 2):
        attn, _, block = make(cuda, seed)
        layers.append(DecoderLayer(attn, block, seqs.cache(attn)))

    def run(x, batch):
        for layer in layers:
            x = layer(x, batch)
        return x

    run(O.make_tokens(60, H=H, seed=1).to(cuda), seqs.extend({0: 45, 1: 15}, prompts=True))
    batch = seqs.extend({0: 1, 1: 1})
    x = O.make_tokens(2, H=H, seed=2).to(cuda)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            run(x, batch)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            y = run(x, batch)
    torch.cuda.current_stream().wait_stream(s)
    for i in range(5):
        if i:
            nxt = seqs.extend({0: 1, 1: 1})
            batch.page_table.copy_(nxt.page_table)
            batch.kv_lens.copy_(nxt.kv_lens)
        x.copy_(O.make_tokens(2, H=H, seed=10 + i))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, run(x, batch)), i
    assert not L.all_workspace_errors()
