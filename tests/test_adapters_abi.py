"""Refusals of the adapter entry points, on the CPU: the C ABI with addresses that are
never read, the Python layer with CPU tensors."""
import ctypes

import pytest
import torch

from tests.test_paged_abi import lib  # noqa: F401


def adapters(widths=(8192, 512, 512, 0), **kw):
    from qwen36_attn import _lib
    a = dict(a=16, b=16, ranks=None, scales=None, adapters=4, rank=16, k=2048, slices=3)
    a.update(kw)
    return ctypes.byref(_lib.AdaptersArgs(widths=(ctypes.c_uint * 4)(*widths), **a))


def args(adapters, **kw):
    a = dict(x=16, xs=2048, y=16, ys=9216, w=adapters, plan=16, pb=1 << 30, seqs=2, tokens=5, ws=16, wb=1 << 40)
    a.update(kw)
    return (*a.values(), None)


BAD = [dict(a=None), dict(b=None), dict(a=8), dict(b=8), dict(adapters=0), dict(adapters=4097), dict(rank=0), dict(rank=12),
       dict(rank=136), dict(k=0), dict(k=2000), dict(k=16512), dict(slices=0), dict(slices=5), dict(slices=4),
       dict(widths=(8192, 510, 512, 0)), dict(widths=(65536, 8, 8, 0)), dict(widths=(65544, 8, 8, 0))]


@pytest.mark.parametrize("bad", BAD)
def test_bad_adapters(lib, bad):  # noqa: F811
    w = adapters(**bad)
    assert lib.qwen36_adapter_apply(*args(w, xs=16512, ys=1 << 20)) == 1
    assert lib.qwen36_adapter_workspace_bytes(w, 2, 5) == 0


@pytest.mark.parametrize("bad", [dict(x=None), dict(x=8), dict(xs=2040), dict(xs=2052), dict(y=None), dict(y=8), dict(ys=9208),
                                 dict(ys=9220), dict(w=None), dict(plan=None), dict(plan=8), dict(pb=64), dict(seqs=0),
                                 dict(seqs=65537), dict(tokens=0), dict(tokens=262145), dict(ws=None), dict(ws=8), dict(wb=64)])
def test_apply_refuses(lib, bad):  # noqa: F811
    assert lib.qwen36_adapter_apply(*args(adapters(), **bad)) == 1


def test_plan_refuses(lib):  # noqa: F811
    good = [16, 16, 2, 5, 4, 16, 1 << 20, None]
    for i, x in ((0, None), (1, None), (2, 0), (2, 65537), (3, 0), (3, 262145), (4, 0), (4, 4097), (5, None), (5, 8), (6, 16)):
        bad = list(good)
        bad[i] = x
        assert lib.qwen36_adapter_plan(*bad) == 1
        if i in (2, 3, 4):
            assert lib.qwen36_adapter_plan_bytes(*bad[2:5]) == 0


def test_python_refuses_cpu_tensors():
    from qwen36_attn import adapters as ad
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        ad.AdapterBatch(i, i[:1], 3, 1)
    with pytest.raises(ValueError):
        ad.AdapterSet(torch.zeros(1, 1, 8, 128, dtype=torch.bfloat16), torch.zeros(1, 8, 8, dtype=torch.bfloat16), (8,))
