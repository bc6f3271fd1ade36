"""When a batch of adapters reads its offsets and ids: once, when it is made."""
import torch

import pytest

from qwen36_attn import adapters as ad
from tests.test_adapters_gpu import BF16, MIXED, make, vector

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("within", [True, False])
def test_a_graph_goes_by_the_batch_that_it_holds(gpu, within):
    """Captured over a batch made before, a call keeps that batch's assignment; over one made
    within the capture, it follows the numbers."""
    a, b, scales, adapters, g = make(gpu, MIXED, 4, 16, [16, 8, 12, 3], 6)
    x, y = (torch.randn(20, n, generator=g, device=gpu).to(BF16) for n in (2048, sum(MIXED[1])))
    before, first = y.clone(), ([0, 5, 6, 20], [0, 1, 2])
    cu, ids = (vector(v, gpu) for v in first)
    made = ad.AdapterBatch(cu, ids, 20, 4)

    def step():
        return ad.apply_adapters(y, x, adapters, ad.AdapterBatch(cu, ids, 20, 4) if within else made)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for c, i in (first, ([0, 0, 19, 20], [3, -1, 0]), ([0, 1, 2, 3], [7, 2, 2])):
        cu.copy_(vector(c, gpu))
        ids.copy_(vector(i, gpu))
        y.copy_(before)
        graph.replay()
        torch.cuda.synchronize()
        c, i = (c, i) if within else first
        want = ad.apply_adapters(before.clone(), x, adapters, ad.AdapterBatch(vector(c, gpu), vector(i, gpu), 20, 4))
        assert torch.equal(y, want), c
