"""The delta rule's chunks over rows whose values are of very different sizes."""
import pytest
import torch

from qwen36_attn import ragged_deltanet as rd
from tests import ragged_reference as R
from tests.test_ragged_deltanet_gpu import BF16, batch, check_delta, core

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [-10, -20, -28, -40])
@pytest.mark.parametrize("lens", [[64, 20], [200, 64, 9, 130, 70, 90]])
def test_small_rows_before_large_ones(gpu, lens, power):
    """The first 16 rows of a sequence without a state hold values of 2^power beside the
    next rows' in one chunk.  A row beta v enters its product as two fp16 values of a column
    whose largest is at 2^13 at least: they lose 2^-22 of a value, or half of fp16's least
    step, 2^-25 there, which is 2^-38 of the column's largest.  Those of up to 16 rows change
    a state's column by 16 of them at most (each update, and what follows, takes a column's
    norm no further for beta to 2), and a row's output by their norm over sqrt(128): beside
    what check_delta allows, 2^-38 16 / sqrt(128) of the largest |beta v| of the column."""
    n = len(lens)
    q, k, v, g, beta, gen = core(gpu, sum(lens), 67, 0.5)
    v = v.contiguous()
    cu = R.cu_of(lens)
    for a in cu[:-1]:
        v[a:a + min(16, lens[cu.index(a)])] *= 2.0 ** power
    states = torch.randn(n, 32, 128, 128, generator=gen, device=gpu)
    before, has = states.clone(), [False] * n
    out = torch.full((sum(lens), 32, 128), 7.0, dtype=BF16, device=gpu)
    rd.ragged_delta_rule(q, k, v, g, beta, states, *batch(lens, range(n), has, gpu), out=out)
    want, after = R.delta(q, k, v, g, beta, before, cu, range(n), has)
    for i, a in enumerate(cu[:-1]):
        m = min(16, lens[i])
        w, o = want[a:a + m], out[a:a + m].double()
        largest = (beta[a:a + min(64, lens[i])].double()[..., None] * v[a:a + min(64, lens[i])].double()).abs().amax(0)
        tol = 2.0 ** -8 * w.abs() + 2.0 ** -12 * w.abs().amax(-1, keepdim=True) + 2.0 ** -38 * 16 * 128 ** -0.5 * largest
        err = (o - w).abs()
        assert (err <= tol).all(), (i, (err / tol).max().item())
    rest = torch.ones(sum(lens), dtype=torch.bool, device=gpu)
    for i, a in enumerate(cu[:-1]):
        rest[a:a + min(16, lens[i])] = False
    out[~rest] = 7.0
    want[~rest] = float("nan")
    check_delta(out, states, want, after, [])
