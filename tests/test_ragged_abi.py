"""Refusals of the ragged DeltaNet entry points, on the CPU: the C ABI with addresses
that are never read, the Python layer with CPU tensors."""
import ctypes

import pytest
import torch

from tests.test_paged_abi import lib  # noqa: F401


def batch(**kw):
    from qwen36_attn import _lib
    a = dict(cu_tokens=16, slots=16, has_state=None, seqs=2, tokens=3, num_slots=4)
    a.update(kw)
    return ctypes.byref(_lib.StateBatchArgs(**a))


BAD = [dict(cu_tokens=None), dict(slots=None), dict(seqs=0), dict(seqs=65537), dict(tokens=0), dict(tokens=262145),
       dict(num_slots=0), dict(num_slots=1 << 31)]


def conv_args(b):
    return [16, 8192, 16, 16, 24576, b, 16, None]


def delta_args(b):
    return [16, 16, 16, 16, 2048, 4096, 16, 16, 16, 32 * 128 * 128, b, 0, 16, 16, 1 << 40, None]


@pytest.mark.parametrize("bad", BAD)
def test_bad_batches(lib, bad):  # noqa: F811
    assert lib.qwen36_gdn_ragged_conv1d(*conv_args(batch(**bad))) == 1
    assert lib.qwen36_gdn_ragged_delta(*delta_args(batch(**bad))) == 1
    assert lib.qwen36_gdn_ragged_delta_workspace_bytes(batch(**bad), 0) == 0


def test_delta_workspace(lib):  # noqa: F811
    """None where no sequence can be long, or is said to be."""
    of = lib.qwen36_gdn_ragged_delta_workspace_bytes
    assert of(batch(seqs=64, tokens=12), 0) == 0 and of(batch(seqs=64, tokens=500), 1) == 0
    assert of(batch(seqs=64, tokens=500), 0) == of(batch(seqs=64, tokens=500), 200) > 0


@pytest.mark.parametrize("change", [{0: None}, {0: 24}, {1: 8184}, {1: 8196}, {2: None}, {2: 8}, {3: None}, {3: 8},
                                    {4: 24568}, {4: 24580}, {5: None}, {6: None}, {6: 8}])
def test_conv_refuses(lib, change):  # noqa: F811
    args = conv_args(batch())
    for i, x in change.items():
        args[i] = x
    assert lib.qwen36_gdn_ragged_conv1d(*args) == 1


@pytest.mark.parametrize("change", [{0: None}, {1: None}, {2: None}, {0: 8}, {1: 8}, {2: 8}, {3: 8}, {3: 17}, {3: 32},
                                    {4: 2040}, {4: 2052}, {4: (1 << 24) + 8}, {5: 4088}, {5: 4100}, {5: (1 << 24) + 8}, {6: None}, {7: None}, {8: None}, {8: 8},
                                    {9: 32 * 128 * 128 - 4}, {9: 32 * 128 * 128 + 2}, {10: None}, {12: None}, {12: 8},
                                    {13: None}, {13: 8}, {14: 1000}])
def test_delta_refuses(lib, change):  # noqa: F811
    args = delta_args(batch(tokens=90))
    for i, x in change.items():
        args[i] = x
    assert lib.qwen36_gdn_ragged_delta(*args) == 1


def test_python_refuses_cpu_tensors():
    from qwen36_attn import ragged_deltanet as rd
    x = torch.zeros(3, 8192, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError):
        rd.ragged_conv1d(x, x.new_zeros(8192, 4), x.new_zeros(2, 8192, 3), i, i[:1])
    with pytest.raises(ValueError):
        rd.ragged_delta_rule(x, x, x, x, x, torch.zeros(2, 32, 128, 128), i, i[:1])


@pytest.mark.parametrize("flags,status", [(4, 1), (8, 1), (1 << 31, 1)])
def test_delta_flags(lib, flags, status):  # noqa: F811
    args = delta_args(batch(tokens=90))
    assert lib.qwen36_gdn_ragged_delta_ex(*args[:12], flags, *args[12:]) == status
