"""The paged-cache operators at the lengths their loops are made for: several
stages, windows of pages and steps a wave, one chunk and many, whole rows joined
by one wave, selections over thousands of pages.  Sequences share the pages of a
small pool (read, pages may be shared), and sampled rows are compared with the
64-bit form.  Each case states the form that it is there for by the split that
the call wrote down, or by the rule it follows."""
import numpy as np
import pytest
import torch

from qwen36_attn import _lib
from qwen36_attn import paged_attention as pa
from qwen36_attn import synthetic as syn
from tests import paged_reference as R
from tests.test_paged_gpu import filled_cache

pytestmark = pytest.mark.gpu
FP8, BF16 = torch.float8_e4m3fn, torch.bfloat16


def shared(gpu, lens, new, page, heads, dtype, pool, bounds=False, absent=0, seed=0):
    """Sequences over random pages of a pool, some of their ids outside of it."""
    whole = R.Batch([pool * page], [1], page, seed=seed, spare=0)
    c, state = filled_cache(gpu, whole, heads, dtype, bounds, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    b = R.Batch([1], [1], page)
    b.lens, b.new, b.width, b.pool = list(lens), list(new), max(-(-n // page) for n in lens), pool
    b.table = torch.randint(0, pool, (len(lens), b.width), generator=g, dtype=torch.int32)
    for _ in range(absent):
        i, p = (int(torch.randint(0, n, (1,), generator=g)) for n in b.table.shape)
        b.table[i, p] = (-1, pool, 2 ** 31 - 1)[p % 3]
    b.cu = torch.tensor([0] + b.new).cumsum(0).to(torch.int32)
    b.tokens = int(b.cu[-1])
    return b, c, state


def queries(b, heads, seed, scale=1.5):
    g = syn.gen(seed)
    q = (scale * torch.randn(b.tokens, heads * 8, 256, generator=g)).to(BF16)
    return q, torch.randn(b.tokens, heads * 8 * 512, generator=g).to(BF16)


def attention(gpu, c, b, q, gate):
    """The call over a workspace of the test's own: (output, the first word of the
    workspace: 128-key blocks of a chunk, or of a share where tiles have two tokens)."""
    where = b.where(gpu)
    batch, lib = pa._batch(c, b.tokens, *where), _lib.load()
    n = lib.qwen36_paged_attention_workspace_bytes(c._args, batch)
    ws = torch.full((n,), 0xFF, dtype=torch.uint8, device=gpu)
    out = torch.empty(b.tokens, c.heads * 256, dtype=BF16, device=gpu)
    q, gate = q.to(gpu), gate.to(gpu)
    assert lib.qwen36_paged_attention(q.data_ptr(), c._args, batch, gate.data_ptr(), gate.stride(0), out.data_ptr(),
                                      ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream) == 0
    return out.double().cpu(), int(ws[:4].view(torch.int32))


def check_rows(got, state, b, q, gate, rows, heads, pages=None):
    """Rows (and KV heads) of a call against R.attend's form of them."""
    at = {row: (i, pos) for row, i, pos in b.rows()}
    got = got.view(b.tokens, -1, 256)
    for row in rows:
        i, pos = at[row]
        for h in heads:
            mine = range(pos // b.page + 1) if pages is None else [int(x) for x in pages[row, h] if 0 <= int(x) <= pos // b.page]
            s = slice(8 * h, 8 * h + 8)
            o, tol = R.attend_row(state, b, q[row, s], i, h, pos, mine)
            g = torch.sigmoid(gate[row].double().view(-1, 2, 256)[s, 1])
            o, tol = o * g, tol * g + 2.0 ** -20 * (o * g).abs()
            assert torch.isfinite(got[row, s]).all(), (row, h)
            assert ((got[row, s] - o).abs() <= tol).all(), (row, h, ((got[row, s] - o).abs() - tol).max().item())


# ------------------------------------------------------- prompts and drafts

@pytest.mark.parametrize("dtype", [FP8, BF16])
@pytest.mark.parametrize("page", [16, 64, 128])
def test_prompt_in_long_chunks(gpu, dtype, page):
    """2,048 rows over 6,200 keys: two chunks of some 4,096 keys, so four windows of
    1,024 keys and every stage of a window, tiles that end in either chunk, and 4,096
    (row, KV head) pairs to join, a wave for 8 heads."""
    b, c, state = shared(gpu, [8248], [2048], page, 2, dtype, 3000 // page, absent=6, seed=page)
    q, gate = queries(b, 2, page)
    got, blocks = attention(gpu, c, b, q, gate)
    assert 16 < blocks < 64 and b.tokens * 2 >= 2048
    check_rows(got, state, b, q, gate, [0, 1, 31, 32, 777, 1030, 1900, 2015, 2016, 2047], (0, 1))


@pytest.mark.parametrize("dtype", [FP8, BF16])
def test_prompt_in_one_chunk(gpu, dtype):
    """Four KV heads, so that 2,000 rows fill the GPU without a split: up to 3,100 keys
    straight to the output."""
    b, c, state = shared(gpu, [3100], [2000], 32, 4, dtype, 80, absent=3, seed=3)
    q, gate = queries(b, 4, 4)
    got, blocks = attention(gpu, c, b, q, gate)
    assert blocks * 128 >= 3100
    check_rows(got, state, b, q, gate, [0, 31, 32, 500, 1111, 1983, 1984, 1999], (0, 3))


@pytest.mark.parametrize("dtype", [FP8, BF16])
@pytest.mark.parametrize("new", [5, 8, 12, 16])
def test_short_turns_in_long_chunks(gpu, dtype, new):
    """5 to 16 rows of as many sequences as fill the GPU: tiles of 8 and of 16 tokens
    over more than one window of keys, in one chunk, and 2,048 and more pairs of rows
    and KV heads for the join to find already written."""
    heads = 4
    lens = [1090 + 13 * (i % 11) for i in range(128)]
    b, c, state = shared(gpu, lens, [new] * 128, 64, heads, dtype, 40, absent=40, seed=new)
    q, gate = queries(b, heads, new)
    got, blocks = attention(gpu, c, b, q, gate)
    assert blocks * 128 >= max(lens) and b.tokens * heads >= 2048
    check_rows(got, state, b, q, gate, [0, new - 1, new, 10 * new + 3, 64 * new + 1, 127 * new, b.tokens - 1], (0, 3))


@pytest.mark.parametrize("dtype", [FP8, BF16])
@pytest.mark.parametrize("new", [5, 12])
def test_short_turns_split(gpu, dtype, new):
    """Chunks of more than one window where few sequences are long: 3 of 24,000 keys
    over 16 KV heads."""
    b, c, state = shared(gpu, [24000, 23001, 20500], [new] * 3, 128, 16, dtype, 12, absent=5, seed=new)
    q, gate = queries(b, 16, new)
    got, blocks = attention(gpu, c, b, q, gate)
    assert 8 < blocks < 188
    check_rows(got, state, b, q, gate, [0, new - 1, new, 3 * new - 1], (0, 9, 15))


# ------------------------------------------------------------- single tokens

@pytest.mark.parametrize("dtype", [FP8, BF16])
@pytest.mark.parametrize("lens,new", [([80000], [2]), ([80000], [1]), ([47000, 3, 33300], [1, 2, 1])])
def test_decode_in_long_shares(gpu, dtype, lens, new):
    """16 KV heads, so that a head has 16 workgroups: shares of more than 4,096 keys,
    a wave's second window of steps."""
    b, c, state = shared(gpu, lens, new, 128, 16, dtype, 12, absent=9, seed=sum(new))
    q, gate = queries(b, 16, 5)
    got, blocks = attention(gpu, c, b, q, gate)
    assert blocks > 32
    check_rows(got, state, b, q, gate, range(b.tokens), (0, 7, 15))


# -------------------------------------------------------------------- lists

@pytest.mark.parametrize("dtype", [FP8, BF16])
@pytest.mark.parametrize("rows,listed", [(130, 45), (64, 100), (3, 1024)])
def test_long_lists(gpu, dtype, rows, listed):
    """Lists of 5,760 to 131,072 keys in chunks of more than 4,096, or of several steps
    a wave: 130 rows a chunk each, 64 rows two in one grid of 256, 3 rows in many."""
    b, c, state = shared(gpu, [40000], [rows], 128, 2, dtype, 30, absent=20, seed=rows)
    q, gate = queries(b, 2, rows)
    g = torch.Generator().manual_seed(rows)
    pages = torch.randint(-3, 320, (rows, 2, listed), generator=g, dtype=torch.int32)
    where, lib = b.where(gpu), _lib.load()
    got = pa.sparse_paged_attention(q.to(gpu), c, *where, pages.to(gpu), q_gate=gate.to(gpu)).double().cpu()
    slot = (rows and 2 * 8 * (256 + 2) * 4)     # a chunk's partial of a row: two KV heads of 8 queries
    chunks = lib.qwen36_paged_sparse_attention_workspace_bytes(c._args, pa._batch(c, rows, *where), listed) // (rows * slot)
    keys = -(-listed * 128 // chunks)
    assert keys > (4096 if rows > 3 else 256)
    check_rows(got, state, b, q, gate, sorted({0, 1, rows // 2, rows - 1}), (0, 1), pages)


# ---------------------------------------------------------------- selection

def picked(state, b, q, i, h, pos, budget, sinks, recents):
    """R.select for one row and KV head over many pages at once: whole numbers times
    exact powers of two, sorted without moving equals."""
    n = pos // b.page + 1
    if n <= budget:
        return list(range(n))
    x = q.double()
    step = 2.0 ** (np.frexp(x.abs().max().item())[1] - 7)
    qi = torch.round(x / step).clamp(-127, 127)
    ids = b.table[i, :n].long()
    ok = (ids >= 0) & (ids < state.k.shape[0])
    at = torch.where(ok, ids, torch.zeros_like(ids))
    bd = state.bounds[at, h].double()
    s = torch.maximum(qi[:, None] * bd[None, :, 0], qi[:, None] * bd[None, :, 1]).sum(-1).amax(0)
    score = np.ldexp(s.numpy(), state.ke[at, h].numpy().astype(np.int64) - 127)
    score[~ok.numpy()] = -np.inf
    forced = np.arange(n)
    forced = (forced < sinks) | (forced >= n - recents)
    order = np.argsort(-score, kind="stable")
    rest = [int(p) for p in order if not forced[p]][:budget - int(forced.sum())]
    return sorted([int(p) for p in np.nonzero(forced)[0]] + rest)


@pytest.mark.parametrize("width,seqs,new", [(3000, 40, 1), (3000, 1, 101), (4352, 1, 1), (2049, 3, 7), (4353, 2, 1),
                                            (9000, 16, 1), (9000, 1, 24)])
@pytest.mark.parametrize("heads", [1, 2])
def test_selection_over_thousands_of_pages(gpu, width, seqs, new, heads):
    """2,049 to 9,000 pages a sequence, ties among them (a pool of 700): every width of
    the choice, and rows (single and by twos) whose waves score several groups of 16."""
    page = 16
    lens = [width * page - 37 * i for i in range(seqs)]
    g = syn.gen(width + new)
    c = pa.PagedKVCache(700, page, gpu, FP8, heads, True)
    c.bounds.copy_(torch.randint(-100, 101, c.bounds.shape, generator=g, dtype=torch.int8).sort(2, descending=True)[0])
    c.k_exp.copy_(torch.randint(118, 121, c.k_exp.shape, generator=g, dtype=torch.uint8))
    state = R.CacheState(c)
    b = R.Batch([1], [1], page)
    b.lens, b.new, b.width = lens, [new] * seqs, width
    b.table = torch.randint(0, 700, (seqs, width), generator=torch.Generator().manual_seed(width), dtype=torch.int32)
    b.table[0, 5], b.table[-1, 1999] = 700, -1
    b.cu = torch.tensor([0] + b.new).cumsum(0).to(torch.int32)
    b.tokens = seqs * new
    q = syn.randn((b.tokens, heads * 8, 256), g)
    rows = list(b.rows())
    for budget, sinks, recents in ((2, 1, 1), (97, 3, 2), (1024, 0, 1)):
        got = pa.select_pages(q.to(gpu), c, *b.where(gpu), budget, sinks, recents).cpu()
        for row, i, pos in rows[:3] + rows[len(rows) // 2:][:2] + rows[-3:]:
            for h in range(heads):
                want = picked(state, b, q[row, 8 * h:8 * h + 8], i, h, pos, budget, sinks, recents)
                assert got[row, h].tolist() == want, (row, h, budget)


# ------------------------------------------------------------------- memory

@pytest.mark.parametrize("dtype", [FP8, BF16])
@pytest.mark.parametrize("lens,new", [([1500, 70, 3], [1, 1, 1]), ([900, 300], [2, 2]), ([2000, 70, 4], [5, 8, 6]),
                                      ([1000, 41, 9], [16, 12, 12]), ([1600, 70, 20], [90, 40, 33]), ([7000], [1])])
def test_results_do_not_depend_on_what_workspaces_and_outputs_held(gpu, dtype, lens, new):
    """Workspaces and outputs of the test's own, filled with bytes of one pattern right
    before each call: the same results whatever they held, and rows behind the last
    sequence as they were.  Every size of tile, split rows, lists in several chunks."""
    b = R.Batch(lens, new, 16, seed=sum(new), rows_behind=2)
    c, _ = filled_cache(gpu, b, 2, dtype, True, seed=sum(lens))
    q, gate = (x.to(gpu) for x in queries(b, 2, 9))
    where, lib, t = b.where(gpu), _lib.load(), b.tokens
    batch, stream = pa._batch(c, t, *where), torch.cuda.current_stream().cuda_stream
    listed, live = 12, t - 2
    sizes = (lib.qwen36_paged_attention_workspace_bytes(c._args, batch), lib.qwen36_paged_select_workspace_bytes(c._args, batch),
             lib.qwen36_paged_sparse_attention_workspace_bytes(c._args, batch, listed))
    want = None
    for fill in (0x00, 0xFF, 0x7F, 0x5A):
        def own(n, fill=fill):
            return torch.full((n,), fill, dtype=torch.uint8, device=gpu)
        ws, out, pages, sparse = [own(n) for n in sizes], own(t * 8192), own(t * 2 * listed * 4), own(t * 8192)
        assert lib.qwen36_paged_attention(q.data_ptr(), c._args, batch, gate.data_ptr(), gate.stride(0), out.data_ptr(),
                                          ws[0].data_ptr(), sizes[0], stream) == 0
        assert lib.qwen36_paged_select(q.data_ptr(), c._args, batch, listed, 1, 1, pages.data_ptr(), ws[1].data_ptr(),
                                       sizes[1], stream) == 0
        assert lib.qwen36_paged_sparse_attention(q.data_ptr(), c._args, batch, pages.data_ptr(), listed, gate.data_ptr(),
                                                 gate.stride(0), sparse.data_ptr(), ws[2].data_ptr(), sizes[2], stream) == 0
        got = [x.view(t, -1) for x in (out, pages, sparse)]
        for x in got:
            assert (x[live:] == fill).all()
        got = [x[:live] for x in got]
        if want is None:
            want = got
        for x, y in zip(got, want):
            assert torch.equal(x, y), fill
    ref = pa.select_pages(q, c, *where, listed)[:live]
    assert torch.equal(want[1].reshape(-1).view(torch.int32), ref.reshape(-1))
    assert torch.equal(want[0].reshape(-1).view(BF16), pa.paged_attention(q, c, *where, q_gate=gate)[:live].reshape(-1))
