"""Host side of the paged cache, on the CPU: what a PagedKVCache lets a caller
change."""
import pytest


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
