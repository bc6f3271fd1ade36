"""The paged-cache operators where a row's answer hangs on something rare: gates
that are NaN over an attention of exactly zero, sequences that outgrow the
rotation tables of a layer, more rows than one launch holds."""
import pytest
import torch

from qwen36_attn import full_attention as fa
from qwen36_attn import paged_attention as pa
from qwen36_attn import synthetic as syn
from tests import paged_reference as R
from tests.test_paged_gpu import filled_cache, upload
from tests.test_paged_use_gpu import layer_weights

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


@pytest.mark.parametrize("budget", [None, 2])
def test_layer_over_a_sequence_longer_than_its_rotation_tables(gpu, budget):
    """Tables of 70 positions under a page table of 96: nothing of the sequence of 71
    tokens is appended, so nothing of it is attended; the others are as ever."""
    page, w = 32, layer_weights(gpu, 5)
    b = R.Batch([70, 71, 40], [3, 2, 1], page, seed=5)
    outs, caches = [], []
    for lens in ([70, 71, 40], [70, 0, 40]):
        b.lens = lens
        cache, _ = filled_cache(gpu, R.Batch([70, 71, 40], [3, 2, 1], page, seed=5), 2, FP8, True, seed=6)
        layer = pa.PagedFullAttentionLayer(w, cache, fa.rotary_table(70, 0, gpu), budget)
        inp = syn.randn((6, 2048), syn.gen(7)).to(gpu)
        outs.append(layer.forward(inp, *b.where(gpu)))
        caches.append(R.CacheState(cache))
    assert (outs[0][3:5] == 0).all()
    assert torch.equal(outs[0], outs[1]) and (outs[0][:3] != 0).any() and (outs[0][5] != 0).any()
    for name in ("k", "v", "ke", "ve", "bounds"):
        assert torch.equal(getattr(caches[0], name), getattr(caches[1], name)), name


def test_selection_of_more_rows_than_one_launch_holds(gpu):
    """262,144 rows of 16 KV heads over a table of 4,353 pages: 2^32 threads.  The
    last 80 rows see something."""
    heads, page, width, rows, budget = 16, 16, 4353, 262144, 2
    need = rows * heads * (8 * 256 * 2 + width * 4 + budget * 4)
    if torch.cuda.mem_get_info()[0] < need + (4 << 30):
        pytest.skip("needs 90 GB of free GPU memory")
    g = syn.gen(1)
    c = pa.PagedKVCache(5, page, gpu, FP8, heads, True)
    c.bounds.copy_(torch.randint(-100, 101, c.bounds.shape, generator=g, dtype=torch.int8).sort(2, descending=True)[0])
    c.k_exp.copy_(torch.randint(118, 121, c.k_exp.shape, generator=g, dtype=torch.uint8))
    state = R.CacheState(c)
    b = R.Batch([80], [80], page, spare=0)
    q = torch.empty(rows, heads * 8, 256, dtype=BF16, device=gpu)
    mine = syn.randn((80, heads * 8, 256), g)
    q[-80:] = mine.to(gpu)
    table = torch.zeros(1, width, dtype=torch.int32, device=gpu)
    table[:, :5] = b.table.to(gpu)
    got = pa.select_pages(q, c, table, torch.tensor([0, rows], dtype=torch.int32, device=gpu),
                          torch.tensor([80], dtype=torch.int32, device=gpu), budget)
    assert bool((got[:-80] == -1).all())
    got = got[-80:].cpu()
    for (row, h), want in R.select(state, b, mine, budget, 1, 1).items():
        assert got[row, h].tolist() == want + [-1] * (budget - len(want)), (row, h)
    del q, got, table
    torch.cuda.empty_cache()
