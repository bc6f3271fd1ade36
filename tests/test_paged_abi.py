"""The paged-cache entry points' refusals, on the CPU: the C ABI with addresses
that are never read, the Python layer with CPU tensors."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    import os
    from qwen36_attn import _lib
    if not os.path.isfile(_lib.library_path()):
        pytest.skip("library not built")
    return _lib.load()


def cache(**kw):
    from qwen36_attn import _lib
    a = dict(k_pages=4096, v_pages=8192, k_exp=16, v_exp=16, bounds=4096, k_page_stride=2 * 64 * 256,
             v_page_stride=2 * 64 * 256, num_pages=10, page_tokens=64, kv_heads=2, cache_type=1)
    a.update(kw)
    return _lib.PagedCacheArgs(**a)


def batch(**kw):
    from qwen36_attn import _lib
    a = dict(page_table=16, cu_tokens=16, seq_lens=16, table_stride=8, table_width=8, seqs=2, tokens=3)
    a.update(kw)
    return _lib.PagedBatchArgs(**a)


BAD_CACHE = [dict(k_pages=None), dict(v_pages=None), dict(k_pages=4100), dict(num_pages=0), dict(page_tokens=8),
             dict(page_tokens=48), dict(page_tokens=256), dict(kv_heads=0), dict(kv_heads=17), dict(cache_type=2),
             dict(k_page_stride=2 * 64 * 256 - 16), dict(v_page_stride=100), dict(k_page_stride=2 * 64 * 256 + 8),
             dict(k_exp=None), dict(v_exp=None), dict(cache_type=0, k_exp=None), dict(bounds=8)]
BAD_BATCH = [dict(page_table=None), dict(cu_tokens=None), dict(seq_lens=None), dict(seqs=0), dict(seqs=65537),
             dict(tokens=0), dict(tokens=262145), dict(table_width=0), dict(table_width=9),
             dict(table_width=4098, table_stride=5000)]


@pytest.mark.parametrize("c,b", [(x, {}) for x in BAD_CACHE] + [({}, x) for x in BAD_BATCH])
def test_bad_cache_or_batch_is_refused(lib, c, b):
    c, b = ctypes.byref(cache(**c)), ctypes.byref(batch(**b))
    big = 1 << 40
    assert lib.qwen36_paged_attention_workspace_bytes(c, b) == 0
    assert lib.qwen36_paged_select_workspace_bytes(c, b) == 0
    assert lib.qwen36_paged_sparse_attention_workspace_bytes(c, b, 4) == 0
    assert lib.qwen36_paged_append(16, 8192, 16, 512, 16, 512, 16, 16, 16, 16, 512, c, b, 16, None) == 1
    assert lib.qwen36_paged_attention(16, c, b, None, 0, 16, 16, big, None) == 1
    assert lib.qwen36_paged_select(16, c, b, 4, 1, 1, 16, 16, big, None) == 1
    assert lib.qwen36_paged_sparse_attention(16, c, b, 16, 4, None, 0, 16, 16, big, None) == 1


def test_null_structures_are_refused(lib):
    c, b = ctypes.byref(cache()), ctypes.byref(batch())
    assert lib.qwen36_paged_append(16, 8192, 16, 512, 16, 512, 16, 16, 16, 16, 512, None, b, 16, None) == 1
    assert lib.qwen36_paged_attention(16, c, None, None, 0, 16, 16, 1 << 40, None) == 1
    assert lib.qwen36_paged_attention_workspace_bytes(None, b) == 0
    assert lib.qwen36_paged_select_workspace_bytes(c, None) == 0


@pytest.mark.parametrize("change", [{0: None}, {1: 8188}, {1: 8190}, {2: None}, {3: 508}, {3: 514}, {4: None}, {5: 508},
                                    {6: None}, {7: None}, {8: None}, {9: None}, {10: 0}, {13: None}, {0: 12},
                                    {2: 12}, {8: 24}, {13: 20}])
def test_append_refuses(lib, change):
    args = [16, 8192, 16, 512, 16, 512, 16, 16, 16, 16, 512, ctypes.byref(cache()), ctypes.byref(batch()), 16, None]
    for i, x in change.items():
        args[i] = x
    assert lib.qwen36_paged_append(*args) == 1


@pytest.mark.parametrize("change", [{0: None}, {0: 24}, {3: 12, 4: 8192}, {3: 16, 4: 4096}, {3: 16, 4: 8194},
                                    {5: None}, {5: 12}, {6: None}, {6: 24}, {7: 1}])
def test_attention_refuses(lib, change):
    args = [16, ctypes.byref(cache()), ctypes.byref(batch()), None, 0, 16, 16, 1 << 40, None]
    for i, x in change.items():
        args[i] = x
    assert lib.qwen36_paged_attention(*args) == 1


@pytest.mark.parametrize("change", [{0: None}, {0: 24}, {3: 0}, {3: 1025}, {4: 4}, {4: 0xffffffff}, {5: 0}, {5: 4},
                                    {5: 0xffffffff}, {6: None}, {7: None}, {7: 20}, {8: 64}])
def test_select_refuses(lib, change):
    args = [16, ctypes.byref(cache()), ctypes.byref(batch()), 4, 1, 1, 16, 16, 1 << 40, None]
    for i, x in change.items():
        args[i] = x
    assert lib.qwen36_paged_select(*args) == 1


def test_select_needs_bounds(lib):
    assert lib.qwen36_paged_select(16, ctypes.byref(cache(bounds=None)), ctypes.byref(batch()), 4, 1, 1, 16, 16,
                                   1 << 40, None) == 1


@pytest.mark.parametrize("change", [{0: None}, {3: None}, {4: 0}, {4: 1025}, {5: 12, 6: 8192}, {7: None}, {8: None},
                                    {9: 1}])
def test_sparse_attention_refuses(lib, change):
    args = [16, ctypes.byref(cache()), ctypes.byref(batch()), 16, 8, None, 0, 16, 16, 1 << 40, None]
    for i, x in change.items():
        args[i] = x
    assert lib.qwen36_paged_sparse_attention(*args) == 1


def test_python_refuses_cpu_tensors_and_other_types():
    from qwen36_attn import paged_attention as pa
    k = torch.zeros(4, 2, 16, 256, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        pa.PagedKVCache.of(k, k)                       # not on a GPU
    with pytest.raises(ValueError):
        pa.PagedKVCache.of(k.half(), k.half())
    for bad in (dict(page_tokens=24), dict(num_pages=0), dict(kv_heads=0), dict(dtype=torch.int8)):
        with pytest.raises(ValueError):
            pa.PagedKVCache(**{**dict(num_pages=4, page_tokens=16, device="cpu"), **bad})
