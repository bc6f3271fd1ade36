"""Refusals of the page-table entry points, on the CPU: the C ABI with addresses that
are never read, the Python layer with CPU tensors."""
import ctypes

import pytest
import torch

from tests.test_paged_abi import cache, lib  # noqa: F401


def tables(**kw):
    from qwen36_attn import _lib
    a = dict(refs=16, page_table=16, seq_lens=16, table_stride=8, num_pages=10, page_tokens=64, table_width=8, rows=4)
    a.update(kw)
    return ctypes.byref(_lib.PageTablesArgs(**a))


def caches(*kinds):
    from qwen36_attn import _lib
    kinds = kinds or ({},)
    return (_lib.PagedCacheArgs * len(kinds))(*(cache(**k) for k in kinds)), len(kinds)


BAD = [dict(refs=None), dict(page_table=None), dict(seq_lens=None), dict(table_stride=7), dict(num_pages=0),
       dict(num_pages=1 << 31), dict(page_tokens=8), dict(page_tokens=63), dict(table_width=0),
       dict(table_width=4098, table_stride=5000), dict(rows=0), dict(rows=65537)]


@pytest.mark.parametrize("bad", BAD)
def test_bad_tables(lib, bad):  # noqa: F811
    t, (c, n), big = tables(**bad), caches(), 1 << 40
    assert lib.qwen36_pages_trim(t, 16, None) == 1
    assert lib.qwen36_pages_fork(t, 16, None) == 1
    assert lib.qwen36_pages_extend(t, 16, 16, c, n, 16, big, None) == 1
    assert lib.qwen36_pages_compact(t, 16, 16, 8, c, n, 16, big, None) == 1
    assert lib.qwen36_pages_extend_workspace_bytes(t) == 0
    assert lib.qwen36_pages_compact_workspace_bytes(t) == 0


@pytest.mark.parametrize("kinds", [(dict(num_pages=9),), (dict(page_tokens=32),), (dict(k_pages=None),),
                                   ({}, dict(kv_heads=17)), ({}, dict(cache_type=7))])
def test_bad_caches(lib, kinds):  # noqa: F811
    t, (c, n), big = tables(), caches(*kinds), 1 << 40
    assert lib.qwen36_pages_extend(t, 16, 16, c, n, 16, big, None) == 1
    assert lib.qwen36_pages_compact(t, 16, 16, 8, c, n, 16, big, None) == 1


def test_other_refusals(lib):  # noqa: F811
    from qwen36_attn import _lib
    t, (c, n), big = tables(), caches(), 1 << 40
    assert lib.qwen36_pages_trim(t, None, None) == 1
    assert lib.qwen36_pages_trim(None, 16, None) == 1
    assert lib.qwen36_pages_fork(t, None, None) == 1
    for args in ((None, 16, c, n, 16, big), (16, None, c, n, 16, big), (16, 16, None, n, 16, big),
                 (16, 16, c, 1025, 16, big), (16, 16, c, n, None, big), (16, 16, c, n, 8, big), (16, 16, c, n, 16, 64)):
        assert lib.qwen36_pages_extend(t, *args, None) == 1
    for args in ((None, 16, 8, c, n, 16, big), (16, None, 8, c, n, 16, big), (16, 16, 7, c, n, 16, big),
                 (16, 16, 8, None, n, 16, big), (16, 16, 8, c, n, None, big), (16, 16, 8, c, n, 16, 64)):
        assert lib.qwen36_pages_compact(t, *args, None) == 1

    def pool(**kw):
        return ctypes.byref(_lib.SlotPoolArgs(**{**dict(data=16, slot_bytes=64, slot_stride_bytes=64), **kw}))
    assert lib.qwen36_slots_fork(None, 1, 4, 16, None) == 1
    assert lib.qwen36_slots_fork(pool(), 0, 4, 16, None) == 1
    assert lib.qwen36_slots_fork(pool(), 1, 0, 16, None) == 1
    assert lib.qwen36_slots_fork(pool(), 1, 65537, 16, None) == 1
    assert lib.qwen36_slots_fork(pool(), 1, 4, None, None) == 1
    for bad in (dict(data=None), dict(data=8), dict(slot_bytes=0), dict(slot_bytes=72, slot_stride_bytes=80),
                dict(slot_stride_bytes=48), dict(slot_stride_bytes=72), dict(slot_bytes=(1 << 30) + 16, slot_stride_bytes=1 << 31)):
        assert lib.qwen36_slots_fork(pool(**bad), 1, 4, 16, None) == 1


def test_python_refuses_cpu_tensors():
    from qwen36_attn import page_tables as pt
    from qwen36_attn import ragged_deltanet as rd
    refs, table, lens = pt.new_refs(4, "cpu"), torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: pt.trim(refs, table, lens, lens, 16), lambda: pt.fork(refs, table, lens, lens, 16),
                 lambda: pt.extend(refs, table, lens, lens, []), lambda: pt.compact(refs, table, lens, [1]),
                 lambda: rd.fork_states([], lens), lambda: rd.fork_states([torch.zeros(2, 4)], lens)):
        with pytest.raises(ValueError):
            call()
