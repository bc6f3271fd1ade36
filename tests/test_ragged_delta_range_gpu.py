"""The ends of what the delta rule over ragged batches is made for, against 64 bits: gates
that forget everything."""
import math

import pytest
import torch

from qwen36_attn import ragged_deltanet as rd
from tests import ragged_reference as R
from tests.test_ragged_deltanet_gpu import BF16, batch, check_delta, core

pytestmark = pytest.mark.gpu

# rows of a sequence of 200: the first, an inner and the last of a chunk, the ends of a tile of
# 16, two in a row, two in one tile, the sequence's first and last
RESETS = [[64], [70], [63], [79, 80], [20, 21], [3, 9, 100], [0], [199], [0, 63, 64, 127, 128, 199], list(range(200))]


@pytest.mark.parametrize("rows", RESETS)
@pytest.mark.parametrize("value", [-math.inf, -3e38, -1e30, -1e10, -500.0, -128.0, -100.0])
def test_gates_that_forget(gpu, rows, value):
    """e^g is zero or next to it: what came before is gone, what comes after is as precise
    as ever, in the sequence of many rows and in those of few, and in one head of four."""
    lens, slots, has = [200, 5, 12], [1, 0, 2], [True] * 3
    q, k, v, g, beta, gen = core(gpu, sum(lens), 59, 0.5)
    g[rows, ::4] = value
    g[[201, 205, 210, 216], 1::4] = value
    states = torch.randn(3, 32, 128, 128, generator=gen, device=gpu)
    before = states.clone()
    out = torch.full((sum(lens), 32, 128), 7.0, dtype=BF16, device=gpu)
    rd.ragged_delta_rule(q, k, v, g, beta, states, *batch(lens, slots, has, gpu), out=out)
    want, after = R.delta(q, k, v, g, beta, before, R.cu_of(lens), slots, has)
    check_delta(out, states, want, after, [])


@pytest.mark.parametrize("n", [7, 8, 90])
def test_a_gate_that_is_no_number(gpu, n):
    """It reaches its head's state and the rows from it on, by either form; other heads and
    sequences are as without it."""
    lens, slots, has = [n, 30], [1, 0], [True] * 2
    q, k, v, g, beta, gen = core(gpu, sum(lens), 61, 0.5)
    states = torch.randn(2, 32, 128, 128, generator=gen, device=gpu)
    other = states.clone()
    where = batch(lens, slots, has, gpu)
    want = rd.ragged_delta_rule(q, k, v, g, beta, other, *where)
    g[4, 5] = math.nan
    got = rd.ragged_delta_rule(q, k, v, g, beta, states, *where)
    heads = [h for h in range(32) if h != 5]
    assert got[4:n, 5].isnan().all() and states[1, 5].isnan().all()
    assert torch.equal(got[:, heads], want[:, heads]) and torch.equal(got[n:], want[n:])
    assert torch.equal(states[:, heads], other[:, heads]) and torch.equal(states[0], other[0])
