"""vLLM's chunk rule over packed sequences as a serving program calls it."""
import pytest
import torch

from qwen36_attn import gated_deltanet as gd
from tests import ragged_reference as R
from tests.test_ragged_deltanet_gpu import core

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_under_another_default_type(gpu, dtype):
    """A program whose default type is its weights' gets the same, states in fp32."""
    lens = [70, 1, 9]
    q, k, v, g, beta, _ = core(gpu, sum(lens), 71)
    cu = torch.tensor(R.cu_of(lens), device=gpu)

    def call():
        return gd.vllm_chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], output_final_state=True,
                                              cu_seqlens=cu, use_qk_l2norm_in_kernel=True)
    want, before = call(), torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        got = call()
    finally:
        torch.set_default_dtype(before)
    assert got[1].dtype is torch.float32 and all(torch.equal(x, y) for x, y in zip(got, want))
