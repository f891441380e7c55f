"""The attention calls launch on their tensors' device whichever device is current (host side, with stand-ins for the device, the
host module and the library: no GPU)."""
import types

import pytest
import torch

from mingmoe import _lib as L
from mingmoe import attention as A
from mingmoe import layer


@pytest.fixture
def where(monkeypatch):
    """[current device]: torch.cuda.device and the device query act on it."""
    now = [0]

    class device:
        def __init__(self, d):
            self.to = d if isinstance(d, int) else torch.device(d).index

        def __enter__(self):
            self.back, now[0] = now[0], self.to

        def __exit__(self, *exc):
            now[0] = self.back

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: now[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    return now


class Rows:
    """What the Python path reads of a [T, heads, 128] bf16 tensor on cuda:1."""
    dtype, device, ndim = torch.bfloat16, torch.device("cuda", 1), 3

    def __init__(self, heads):
        self.shape = torch.Size((3, heads, 128))

    data_ptr = staticmethod(lambda: 4096)
    get_device = staticmethod(lambda: 1)

    def stride(self):
        return (self.shape[1] * 128, 128, 1)


def ints(*shape):
    return types.SimpleNamespace(dtype=torch.int32, shape=torch.Size(shape), device=Rows.device, get_device=lambda: 1,
                                 stride=lambda: (1,) if len(shape) == 1 else (shape[1], 1), data_ptr=lambda: 4096)


CACHE = types.SimpleNamespace(_key=(4096, Rows.device, 1, torch.bfloat16, 2, 128))
BATCH = dict(page_table=ints(1, 4), cu_seqlens=ints(2), kv_lens=ints(1))
CALLS = [lambda: A.kv_append(CACHE, Rows(2), Rows(2), q=Rows(8), q_out=Rows(8), **BATCH),
         lambda: A.paged_attention(Rows(8), CACHE, out=Rows(8), **BATCH),
         lambda: A.prompt_attention(Rows(8), Rows(2), Rows(2), ints(2), out=Rows(8))]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("native", [True, False])
def test_launch_device(monkeypatch, where, call, native):
    """Through the host module, which leaves calls for another device to the Python code, and through the Python path behind it."""
    seen = []

    def host(*args):
        if native and where[0] == 1:
            seen.append(where[0])
            return None
        return NotImplemented

    def entry(*args):
        seen.append(where[0])
        return L.MV_OK

    monkeypatch.setattr(A, "_module", types.SimpleNamespace(kv_append=host, paged_attention=host, prompt_attention=host))
    monkeypatch.setattr(A, "_ws", {(1, 0): (4096, 1 << 30)})
    monkeypatch.setattr(L, "_lib", types.SimpleNamespace(mv_kv_append=entry, mv_paged_attention=entry,
                                                         mv_prompt_attention=entry))
    call()
    assert seen == [1] and where == [0]
    where[0] = 1
    call()
    assert seen == [1, 1] and where == [1]


def test_layer_device(monkeypatch, where):
    seen = []
    attn = layer.AttentionBlock(torch.zeros(4 * 64, 8), torch.zeros(8, 2 * 64), torch.ones(8), 2, 1, 64, None)
    x = types.SimpleNamespace(device=Rows.device, shape=(3, 8))
    for name in ("project", "attend", "output"):
        monkeypatch.setattr(attn, name, lambda *a, name=name: seen.append((name, where[0])) or x)
    moe = types.SimpleNamespace(decode=lambda h: seen.append(("moe", where[0])))
    layer.DecoderLayer(attn, moe, None)(x, None)
    assert seen == [("project", 1), ("attend", 1), ("output", 1), ("moe", 1)] and where == [0]
