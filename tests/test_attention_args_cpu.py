"""What the attention calls do with operands that the kernels cannot take as they are (host side, no GPU)."""
import pytest
import torch

from mingmoe import attention as A


@pytest.mark.parametrize("offset", range(1, 8))
def test_contiguous_rows_off_a_16_byte_address_are_copied(offset):
    flat = torch.arange(3 * 2 * 64 + 16).to(torch.bfloat16)
    assert flat.data_ptr() % 16 == 0
    t = flat[offset:offset + 3 * 2 * 64].view(3, 2, 64)
    got, T, H, st, sh, p = A._rows(t, "q", 64, torch.bfloat16, t.device, -1)
    assert p % 16 == 0 and p == got.data_ptr() and (T, H, st, sh) == (3, 2, 128, 64)
    assert torch.equal(got, t)


def test_rows_that_fit_are_taken_as_they_are():
    t = torch.zeros(3, 6, 64, dtype=torch.bfloat16)[:, 2:5]
    got, T, H, st, sh, p = A._rows(t, "q", 64, torch.bfloat16, t.device, -1)
    assert got is t and p == t.data_ptr() and (T, H, st, sh) == (3, 3, 384, 64)


def test_null_page_table_needs_no_columns():
    """The entry point without a GPU: a table of no columns may be null, and what is checked behind it is reached."""
    import ctypes as C

    from mingmoe import _lib as L
    from test_attention_cpu import attn, kv
    lib, c = L.lib(), kv()
    nws = lib.mv_attention_workspace_bytes()
    assert lib.mv_paged_attention(C.byref(attn(c, page_table=None, max_pages=0)), 4096, nws - 1, None) == L.MV_ERR_WORKSPACE
    assert lib.mv_paged_attention(C.byref(attn(c, page_table=None)), 4096, nws - 1, None) == L.MV_ERR_INVALID
