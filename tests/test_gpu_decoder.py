"""From tokens to the next step's cache slots, as they are used together: a decoder with 8-bit projections and head over pages that
are planned on the device, tokens drawn from its logits, and the whole step captured.

Each stage is checked from the GPU's own input of that stage: products within the bound that oracle.serving_oracle derives,
tokens and pages equal."""
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
from oracle import serving_oracle as O

pytestmark = pytest.mark.gpu

H, HQ, HKV, D, V = 512, 8, 2, 64, 1009


def make(cuda, seqs, n_layers=2, eight_bit=True):
    g = torch.Generator().manual_seed(0)
    w = lambda *s: (torch.randn(*s, generator=g) * 0.05).to(torch.bfloat16).to(cuda)
    pack = fp8.quantize_fp8_weight if eight_bit else lambda t: t
    one = torch.ones(H, dtype=torch.bfloat16, device=cuda)
    layers = []
    for i in range(n_layers):
        attn = AttentionBlock(pack(w((HQ + 2 * HKV) * D, H)), pack(w(H, HQ * D)), one, HQ, HKV, D, rotation_table(512, D, device=cuda))
        block = MoeBlock.from_params(MO.make_block_params(seed=i, H=H, I=128, E=16, I_s=256), top_k=4)
        layers.append(DecoderLayer(attn, block, seqs.cache(attn)))
    return Decoder(w(V, H) * 20, layers, one, pack(w(V, H) * 4))


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def test_prompts_and_tokens(cuda):
    import fused_ops
    seqs, host = DeviceSequences(64, 16, 4, 400, device=cuda), Sequences(64, 16, 4, 400, device=cuda)
    decoder = make(cuda, seqs)
    g = torch.Generator(device=cuda).manual_seed(1)
    steps = [({0: 37, 2: 150}, True), ({1: 5}, True), ({0: 1, 2: 1, 1: 1}, False), ({2: 90, 0: 3}, False), ({1: 1, 0: 1}, False)]
    for new, prompts in steps:
        T = sum(new.values())
        tokens = torch.randint(0, V, (T,), generator=g, device=cuda)
        batch = seqs.extend(ints(list(new.values()), cuda), T, seqs=ints(list(new), cuda), max_q=max(new.values()), prompts=prompts)
        want = host.extend(new, prompts=prompts)
        for name in ("cu_seqlens", "kv_lens", "page_table"):
            assert torch.equal(getattr(batch, name), getattr(want, name))
        # the projections from their own inputs
        attn = decoder.layers[0].attn
        x = decoder.embedding[tokens]
        xn = fused_ops.rms_norm(x, attn.norm_w, attn.eps)
        qkv = attn.project(x)
        ref, mag = O.fp8_linear(xn, *attn.w_qkv)
        assert bool(((qkv.reshape(T, -1).double() - ref).abs() <= O.fp8_bound(ref, mag, H, torch.bfloat16)).all())
        o = attn.attend(qkv, decoder.layers[0].cache, batch)
        ref, mag = O.fp8_linear(o.reshape(T, -1), *attn.w_o, residual=x)
        assert bool(((attn.output(o, x).double() - ref).abs() <= O.fp8_bound(ref, mag, HQ * D, torch.bfloat16)).all())
        # device and host bookkeeping give the same layers' results, in the same cache
        logits = decoder(tokens, batch)
        assert logits.shape == (len(new), V) and logits.dtype == torch.float32 and torch.isfinite(logits).all()
        assert torch.equal(logits, decoder(tokens, want))
        u = torch.rand(len(new), generator=g, device=cuda)
        drawn = sampling.sample(logits, u, temperature=0.8, top_k=40, top_p=0.9)
        t, p = torch.tensor(0.8).item(), torch.tensor(0.9).item()
        assert drawn.tolist() == [O.sample(logits[r], u[r].item(), t, 40, p, 0.0)[0] for r in range(len(new))]
    assert not L.all_workspace_errors()


def test_rows_behind_the_tokens(cuda):
    """A step of fewer tokens than rows: the attention half gives the tokens' rows as the step alone does, bit for bit (its sums do
    not depend on the other rows), and the rows behind them their input, to which it adds W_o 0."""
    a, b = DeviceSequences(32, 16, 2, 200, device=cuda), DeviceSequences(32, 16, 2, 200, device=cuda)
    da, db = make(cuda, a), make(cuda, b)
    tokens = torch.randint(0, V, (40,), generator=torch.Generator(device=cuda).manual_seed(2), device=cuda)
    new = ints([20, 13], cuda)
    for prompts in (True, False):
        ba, bb = a.extend(new, 40, max_q=20, prompts=prompts), b.extend(new, 33, max_q=20, prompts=prompts)
        x = da.embedding[tokens]
        ya = da.layers[0].attn(x, da.layers[0].cache, ba)
        yb = db.layers[0].attn(x[:33], db.layers[0].cache, bb)
        assert torch.equal(ya[:33], yb) and torch.equal(ya[33:], x[33:])
        assert torch.isfinite(da(tokens, ba)).all()
    refused = a.extend(ints([500, 1], cuda), 40, max_q=40)
    assert refused.ok.item() == 0 and torch.isfinite(da(tokens, refused)).all()
    assert not L.all_workspace_errors()


@pytest.mark.parametrize("eight_bit", [True, False])
def test_captured_token_loop(cuda, eight_bit):
    """Replays of the captured step against the same steps run one by one, while sequences start, pause and end."""
    runs = []
    for captured in (True, False):
        seqs = DeviceSequences(60, 8, 5, 150, device=cuda)
        decoder = make(cuda, seqs, eight_bit=eight_bit)
        loop = TokenGraph(decoder, seqs)
        assert seqs.lens.tolist() == [0] * 5 and seqs.n_free.item() == 60
        g = torch.Generator(device=cuda).manual_seed(3)
        prompt = torch.randint(0, V, (40,), generator=g, device=cuda)
        batch = seqs.extend(ints([9, 0, 30, 1, 0], cuda), 40, max_q=30, prompts=True)
        decoder(prompt, batch)
        loop.tokens.copy_(torch.tensor([1, 2, 3, 4, 5]))
        loop.temperature.copy_(torch.tensor([0.0, 1.0, 0.7, 1.3, 1.0]))
        loop.top_p.copy_(torch.tensor([1.0, 0.9, 1.0, 0.95, 0.5]))
        loop.top_k.copy_(torch.tensor([0, 50, 0, 7, 0]))
        got = []
        for i in range(24):
            loop.new.copy_(torch.tensor([1, int(i >= 6), 1, int(i % 3 != 1), int(i >= 12)]))
            loop.u.copy_(torch.rand(5, generator=g, device=cuda))
            before = loop.tokens.clone()
            if captured:
                loop()
            else:
                loop.step()
            got.append((loop.tokens.tolist(), seqs.lens.tolist(), seqs.n_free.item(), loop.ok.item()))
            idle = loop.new == 0
            assert torch.equal(loop.tokens[idle], before[idle]) and loop.ok.item() == 1
            row = 0 if not captured else 2  # a token of a running sequence against the plain draw from the step's logits
            want, _ = O.sample(loop.logits[row], loop.u[row].item(), loop.temperature[row].item(), loop.top_k[row].item(),
                               loop.top_p[row].item(), 0.0)
            assert loop.tokens[row].item() == want
            if i == 15:
                assert seqs.release(ints([2], cuda)).item() == 1
        runs.append(got)
        assert not L.all_workspace_errors()
    assert runs[0] == runs[1]
