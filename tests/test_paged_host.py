"""Host side of the paged cache, on the CPU: what a PagedKVCache lets a caller
change, and how the workspaces grow."""
import ctypes

import pytest
import torch

from tests.test_paged_abi import batch, cache, lib  # noqa: F401


@pytest.mark.parametrize("name", ["k_pages", "v_pages", "k_exp", "v_exp", "bounds", "num_pages", "kv_heads",
                                  "page_tokens", "heads", "device"])
def test_a_cache_is_fixed(name):
    """The calls use the addresses and sizes taken when it was made: another tensor
    or size in its place, or a tensor let go, would go unseen."""
    from qwen36_attn import paged_attention as pa
    c = pa.PagedKVCache.__new__(pa.PagedKVCache)
    with pytest.raises(AttributeError):
        setattr(c, name, None)
    c.__dict__[name] = None
    with pytest.raises(AttributeError):
        delattr(c, name)


def test_a_cache_takes_a_caller_s_own_attributes():
    from qwen36_attn import paged_attention as pa
    c = pa.PagedKVCache.__new__(pa.PagedKVCache)
    c.free_pages = [1, 2]
    del c.free_pages
    assert not hasattr(c, "free_pages")


def test_attention_workspace_of_short_tables(lib):  # noqa: F811
    """A tile has a partial for each 128 keys that its page table can hold, at most:
    17 rows over one page of 128 need one tile's, not the split of a long prompt."""
    def bytes_of(**kw):
        return lib.qwen36_paged_attention_workspace_bytes(
            ctypes.byref(cache(page_tokens=128, k_page_stride=2 * 128 * 256, v_page_stride=2 * 128 * 256)),
            ctypes.byref(batch(**kw)))
    partial = 2 * 8 * (256 + 2) * 4         # of a token: two KV heads of 8 queries, output, maximum and sum
    one = bytes_of(seqs=1, tokens=17, table_width=1, table_stride=1)
    assert 32 * partial <= one <= 2 * 32 * partial + 4096
    # never less than what a split can use: 8 blocks of keys, 64 rows in 2 tiles and one more for the remainder
    eight = bytes_of(seqs=1, tokens=64, table_width=8, table_stride=8)
    assert 2 * 8 * 32 * partial <= eight <= 3 * 8 * 32 * partial + 4096
    # and no more than before for long tables: tiles and twice the workgroups that the GPU holds
    long = bytes_of(seqs=1, tokens=2048, table_width=2048, table_stride=2048)
    assert long <= (64 + 1 + 256) * 32 * partial + 4096


@pytest.mark.parametrize("stride,ok", [(4096, True), ((1 << 32) - 4, True), (4095, False), (1 << 32, False),
                                       ((1 << 32) + 4096, False)])
def test_row_strides_of_the_c_interface(stride, ok):
    """The C calls take row strides of 32 bits: a longer one would lose its upper bits
    on the way and other rows be read.  (Tensors without memory.)"""
    from qwen36_attn import paged_attention as pa
    t = torch.empty_strided((2, 4096), (stride, 1), dtype=torch.bfloat16, device="meta")
    if ok:
        assert pa._rows(t, "q_gate", 2, 4096, t.get_device())[1] == stride
    else:
        with pytest.raises(ValueError):
            pa._rows(t, "q_gate", 2, 4096, t.get_device())
