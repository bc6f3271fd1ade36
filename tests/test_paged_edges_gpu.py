"""The paged-cache operators where a row's answer hangs on something rare: gates
that are NaN over an attention of exactly zero."""
import pytest
import torch

from qwen36_attn import paged_attention as pa
from qwen36_attn import synthetic as syn
from tests import paged_reference as R
from tests.test_paged_gpu import filled_cache, upload

pytestmark = pytest.mark.gpu
FP8, BF16 = torch.float8_e4m3fn, torch.bfloat16


@pytest.mark.parametrize("new", [1, 2, 5, 12, 40])
@pytest.mark.parametrize("dtype", [FP8, BF16])
def test_nan_gate_over_an_attention_of_zero(gpu, dtype, new):
    """Values of zero: 0 * sigmoid(NaN) is a NaN whatever tile a row falls into and
    however its keys are split; a row that sees nothing stays zeros."""
    lens = [new + 50, 900, new // 2]            # one chunk, several, and rows of negative position
    b = R.Batch(lens, [new] * 3, 16, seed=new)
    c, state = filled_cache(gpu, b, 2, dtype, seed=new, junk=False)
    state.v.zero_()
    upload(c, state)
    q = syn.randn((b.tokens, 16, 256), syn.gen(new)).to(gpu)
    gate = torch.zeros(b.tokens, 16, 512, dtype=BF16, device=gpu)
    bad = torch.zeros(b.tokens, 16, 256, dtype=torch.bool)
    bad[:, 3::5, 7::64] = True
    gate[:, :, 256:][bad.to(gpu)] = float("nan")
    got = pa.paged_attention(q, c, *b.where(gpu), q_gate=gate.flatten(1)).view(b.tokens, 16, 256).cpu()
    for row, _, pos in b.rows():
        want = bad[row] if pos >= 0 else torch.zeros_like(bad[row])
        assert torch.equal(torch.isnan(got[row]), want), (row, pos)
        assert (got[row][~want] == 0).all(), (row, pos)
