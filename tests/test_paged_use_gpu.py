"""The paged-cache operators as a serving program uses them: a layer over
prompts and decode steps, captured and replayed steps, other streams, pages in
one allocation, many sequences, memory that held something before."""
import pytest
import torch

from qwen36_attn import full_attention as fa
from qwen36_attn import paged_attention as pa
from qwen36_attn import synthetic as syn
from tests import paged_reference as R
from tests.test_paged_gpu import check, filled_cache, layer_rows

pytestmark = pytest.mark.gpu
FP8, BF16 = torch.float8_e4m3fn, torch.bfloat16


def layer_weights(gpu, seed):
    g = syn.gen(seed)
    w = {"q_proj": syn.randn((8192, 2048), g) * 0.03, "k_proj": syn.randn((512, 2048), g) * 0.03,
         "v_proj": syn.randn((512, 2048), g) * 0.03, "o_proj": syn.randn((2048, 4096), g) * 0.02,
         "q_norm": 0.2 * syn.randn((256,), g), "k_norm": 0.2 * syn.randn((256,), g)}
    return {k: v.to(BF16).to(gpu) for k, v in w.items()}


@pytest.mark.parametrize("dtype,budget", [(BF16, None), (FP8, None), (FP8, 4), (BF16, 3)])
def test_layer_over_prompts_and_decode_steps(gpu, dtype, budget):
    """Three sequences: prompts together, a second turn of one beside single tokens
    of the others, then a single token of one.  Each output against the reference
    attention over the cache as it then is, through o_proj."""
    w = layer_weights(gpu, 1)
    page, steps = 32, [[70, 33, 150], [1, 40, 1], [1, 1, 5], [1, 0, 0]]
    rope = fa.rotary_table(512, 0, gpu)
    cache = pa.PagedKVCache(24, page, gpu, dtype, 2, budget is not None)
    layer = pa.PagedFullAttentionLayer(w, cache, rope, budget, 1, 1)
    lens = [0, 0, 0]
    for n, new in enumerate(steps):
        lens = [a + b for a, b in zip(lens, new)]
        b = R.Batch([256] * 3, new, page, seed=7, spare=0)     # the same pages at every step
        b.lens = lens
        inp = syn.randn((b.tokens, 2048), syn.gen(20 + n)).to(gpu)
        got = layer.forward(inp, *b.where(gpu)).double().cpu()
        from qwen36_attn.prefill_gemm import linear
        from qwen36_attn.projections import gemv
        if b.tokens == 1:
            q_gate, k, v = layer._qkv(inp)
        else:
            q_gate, k, v = layer._qkv.split_rows(linear(inp, layer._qkv.w))
        # appending again writes what is there, so that this changes nothing
        before = R.CacheState(cache)
        q = pa.paged_append(q_gate, k, v, w["q_norm"], w["k_norm"], rope, cache, *b.where(gpu))
        before.same(cache)
        pages = None if budget is None else pa.select_pages(q, cache, *b.where(gpu), budget).cpu()
        a, tol, rows = R.attend(before, b, q.cpu(), q_gate.cpu(), pages)
        wo = w["o_proj"].double().cpu()
        want = a @ wo.t()
        # fp32 sums of 4,096 products, one rounding to bf16
        bound = tol @ wo.abs().t() + 2.0 ** -8 * want.abs() + 4100 * 2.0 ** -24 * (a.abs() @ wo.abs().t())
        bound = bound * (1 + 2.0 ** -7)
        assert rows == list(range(b.tokens))
        check(got, want, bound, rows, n)


def test_layer_equals_the_dense_layer(gpu):
    """One sequence, bf16 pages: the dense layer's cache rows bit for bit, and its
    outputs but for the roundings that both make."""
    w = layer_weights(gpu, 3)
    dense = fa.FullAttentionLayer(w, 256, gpu)
    b = R.Batch([256], [100], 32, seed=1)
    cache = pa.PagedKVCache(b.pool, 32, gpu, BF16)
    paged = pa.PagedFullAttentionLayer(w, cache, fa.rotary_table(256, 0, gpu))
    for start, n in ((0, 100), (100, 1), (101, 30), (131, 1)):
        b.lens, b.cu = [start + n], torch.tensor([0, n], dtype=torch.int32)
        inp = syn.randn((n, 2048), syn.gen(40 + start)).to(gpu)
        x = dense.forward(inp, start, "decode" if n == 1 else "prefill").double()
        y = paged.forward(inp, *b.where(gpu)).double()
        at = b.table[0].long().to(gpu)
        k = cache.k_pages[at].transpose(1, 2).reshape(-1, 2, 256)[:start + n]
        v = cache.v_pages[at].transpose(1, 2).reshape(-1, 2, 256)[:start + n]
        assert torch.equal(k, dense.k_cache[:start + n]) and torch.equal(v, dense.v_cache[:start + n])
        # dense: P, attention, sigmoid, gated product, output; paged: P, gated product,
        # output: eight roundings of at most 2^-8, evenly spread, so each 2^-8 / sqrt(3)
        # in the norm, and independent
        assert ((x - y).norm() / x.norm()).item() < (8 / 3) ** 0.5 * 2.0 ** -8


def _step_inputs(gpu, b, seed, heads=2):
    q_gate, k, v, qn, kn = layer_rows(gpu, b.tokens, heads, seed)
    return [q_gate.contiguous(), k.contiguous(), v.contiguous(), qn, kn]


@pytest.mark.parametrize("lens,new", [([300, 41, 129], [1, 1, 1]), ([300, 80], [40, 30]), ([500], [1])])
def test_captured_step_follows_its_tensors(gpu, lens, new):
    """append, attention, selection and sparse attention in one graph, replayed
    with other rows, lengths and pages, with eager work between the replays."""
    b = R.Batch(lens, new, 16, seed=1, room=32)
    cache, state = filled_cache(gpu, b, 2, FP8, True, seed=2)
    eager, _ = filled_cache(gpu, b, 2, FP8, True, seed=2)
    rope = fa.rotary_table(1024, 0, gpu)
    x = _step_inputs(gpu, b, 3)
    where = [t.clone() for t in b.where(gpu)]

    def step(c, inputs, at):
        q = pa.paged_append(*inputs, rope, c, *at)
        a = pa.paged_attention(q, c, *at, q_gate=inputs[0])
        pages = pa.select_pages(q, c, *at, 6)
        return q, a, pages, pa.sparse_paged_attention(q, c, *at, pages, q_gate=inputs[0])
    step(cache, x, where)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(cache, x, where)
    step(eager, x, where)    # the eager cache has seen what the first's warm-up and capture wrote
    for n in range(4):
        y = _step_inputs(gpu, b, 10 + n)
        for mine, theirs in zip(x, y):
            mine.copy_(theirs)
        if n:
            where[2].add_(1)     # every sequence one token longer
        if n == 2:               # two pages change places, contents too
            t = where[0][0, :2].clone()
            where[0][0, :2] = t.flip(0)
            for c in (cache, eager):
                for p in (c.k_pages.view(torch.uint8), c.v_pages.view(torch.uint8), c.k_exp, c.v_exp, c.bounds):
                    p[t.long()] = p[t.flip(0).long()].clone()
        graph.replay()
        want = step(eager, x, where)
        torch.cuda.synchronize()
        junk = torch.full((1 << 22,), float("nan"), device=gpu)
        for got, ref in zip(outs, want):
            assert torch.equal(got, ref), n
        R.CacheState(eager).same(cache)
        del junk


def test_two_graphs_on_two_streams_share_nothing(gpu):
    sets = []
    for i in range(2):
        b = R.Batch([700 + 50 * i, 333], [1, 1], 16, seed=i)
        cache, _ = filled_cache(gpu, b, 2, FP8, True, seed=i)
        q = syn.randn((2, 16, 256), syn.gen(i)).to(gpu)
        where = b.where(gpu)
        run = lambda q=q, c=cache, w=where: (pa.paged_attention(q, c, *w), pa.select_pages(q, c, *w, 9))  # noqa: E731
        want = [t.clone() for t in run()]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = run()
        sets.append((g, outs, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for g, _, _, s in sets:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, outs, want, _ in sets:
        for a, b in zip(outs, want):
            assert torch.equal(a, b)


def test_calls_on_two_streams_at_once(gpu):
    b = R.Batch([2000, 900], [1, 1], 16, seed=4)
    cache, _ = filled_cache(gpu, b, 2, FP8, seed=4)
    where = b.where(gpu)
    qs = [syn.randn((2, 16, 256), syn.gen(i)).to(gpu) for i in range(4)]
    want = [pa.paged_attention(q, cache, *where) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    got = []
    for _ in range(5):
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append(pa.paged_attention(q, cache, *where))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 4])


def test_pages_in_one_allocation_and_a_wide_table(gpu):
    """K and V pages as slices of one [pages, 2, ...] tensor, the table a slice of a
    wider one: bit for bit what separate tensors give."""
    b = R.Batch([200, 45], [1, 3], 32, seed=5)
    one, state = filled_cache(gpu, b, 2, FP8, True, seed=5)
    both = torch.stack((one.k_pages.view(torch.uint8), one.v_pages.view(torch.uint8)), 1).contiguous().view(FP8)
    two = pa.PagedKVCache.of(both[:, 0], both[:, 1], one.k_exp.clone(), one.v_exp.clone(), one.bounds.clone())
    wide = torch.full((2, b.width + 5), 10 ** 6, dtype=torch.int32, device=gpu)
    wide[:, 2:2 + b.width] = b.table.to(gpu)
    x = _step_inputs(gpu, b, 6)
    rope = fa.rotary_table(256, 0, gpu)
    outs = []
    for c, t in ((one, b.table.to(gpu)), (two, wide[:, 2:2 + b.width])):
        where = (t, *b.where(gpu)[1:])
        q = pa.paged_append(*x, rope, c, *where)
        outs.append((q, pa.paged_attention(q, c, *where), pa.select_pages(q, c, *where, 3)))
    for a, b_ in zip(*outs):
        assert torch.equal(a, b_)
    R.CacheState(one).same(two)


@pytest.mark.parametrize("seqs,new", [(300, 1), (300, 4), (700, 1), (130, 20), (1100, 2)])
def test_many_sequences(gpu, seqs, new):
    """More sequences than a workgroup has threads, some empty: append and attend."""
    g = syn.gen(seqs)
    news = [(0 if i % 7 == 3 else 1 + (i * 5) % new) for i in range(seqs)]
    lens = [n and n + int(x) for n, x in zip(news, torch.randint(0, 60, (seqs,), generator=g))]
    b = R.Batch(lens, news, 16, seed=seqs, rows_behind=1)
    c, state = filled_cache(gpu, b, 1, FP8, seed=seqs)
    x = _step_inputs(gpu, b, 8, 1)
    q = torch.zeros(b.tokens, 8, 256, dtype=BF16, device=gpu)
    pa.paged_append(*x, fa.rotary_table(128, 0, gpu), c, *b.where(gpu), q_out=q)
    state = R.CacheState(c)
    got = pa.paged_attention(q, c, *b.where(gpu))
    want, tol, rows = R.attend(state, b, q.cpu())
    check(got, want, tol, rows)


@pytest.mark.parametrize("cu,tokens", [([0, 100] * 6 + [0], 100), ([0, 2] * 20 + [0], 30), ([50, 0, 99, 7, 200, 3, 3, -5, 60], 60),
                                       ([0, 2 ** 31 - 1, -2 ** 31, 90], 90), ([0, 17] * 5 + [0], 40)])
def test_offsets_of_no_batch_stay_in_bounds(gpu, cu, tokens):
    """Offsets that overlap, fall or leave the call: whatever the rows then hold,
    nothing is written outside the outputs, the workspaces and the table's pages."""
    import ctypes
    from qwen36_attn import _lib
    seqs, page, width = len(cu) - 1, 16, 60
    b = R.Batch([900], [1], page, seed=3)
    c, _ = filled_cache(gpu, b, 2, FP8, True, seed=3)
    table = b.table.repeat(seqs, 1)[:, :width].contiguous().to(gpu)
    where = (table, torch.tensor(cu, dtype=torch.int64).clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32).to(gpu),
             torch.tensor([900 - i for i in range(seqs)], dtype=torch.int32, device=gpu))
    batch = pa._batch(c, tokens, *where)
    q = syn.randn((tokens, 16, 256), syn.gen(1)).to(gpu)
    lib, edge = _lib.load(), 1 << 20

    def guarded(n):
        return torch.full((n + edge,), 0x5A, dtype=torch.uint8, device=gpu)
    n = lib.qwen36_paged_attention_workspace_bytes(c._args, batch)
    ws, out = guarded(n), guarded(tokens * 4096 * 2)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.qwen36_paged_attention(q.data_ptr(), c._args, batch, None, 0, out.data_ptr(), ws.data_ptr(), n, stream) == 0
    m = lib.qwen36_paged_select_workspace_bytes(c._args, batch)
    ws2, pages = guarded(m), guarded(tokens * 2 * 8 * 4)
    assert lib.qwen36_paged_select(q.data_ptr(), c._args, batch, 8, 1, 1, pages.data_ptr(), ws2.data_ptr(), m, stream) == 0
    k = lib.qwen36_paged_sparse_attention_workspace_bytes(c._args, batch, 8)
    ws3, out3 = guarded(k), guarded(tokens * 4096 * 2)
    assert lib.qwen36_paged_sparse_attention(q.data_ptr(), c._args, batch, pages.data_ptr(), 8, None, 0, out3.data_ptr(),
                                             ws3.data_ptr(), k, stream) == 0
    x = layer_rows(gpu, tokens, 2, 2)
    before = R.CacheState(c)
    pa.paged_append(*x, fa.rotary_table(1024, 0, gpu), c, *where)
    torch.cuda.synchronize()
    for t in (ws, out, ws2, pages, ws3, out3):
        assert (t[-edge:] == 0x5A).all()
    after = R.CacheState(c)
    spare = [p for p in range(b.pool) if p not in b.table[0].tolist()]
    assert torch.equal(after.k[spare], before.k[spare]) and torch.equal(after.v[spare], before.v[spare])


def test_results_do_not_depend_on_what_memory_held(gpu):
    b = R.Batch([600, 70], [2, 40], 16, seed=11)
    c, _ = filled_cache(gpu, b, 2, BF16, True, seed=11)
    q = syn.randn((42, 16, 256), syn.gen(12)).to(gpu)
    where = b.where(gpu)
    outs = []
    for fill in (0x00, 0xFF, 0x7F):
        junk = [torch.full((1 << 26,), fill, dtype=torch.uint8, device=gpu) for _ in range(3)]
        torch.cuda.synchronize()
        del junk
        pages = pa.select_pages(q, c, *where, 4)
        outs.append((pa.paged_attention(q, c, *where), pages, pa.sparse_paged_attention(q, c, *where, pages)))
    for o in outs[1:]:
        for a, b_ in zip(outs[0], o):
            assert torch.equal(a, b_)


def test_python_refusals(gpu):
    b = R.Batch([64], [2], 16, seed=1)
    c, _ = filled_cache(gpu, b, 2, FP8, seed=1)
    table, cu, lens = b.where(gpu)
    q = torch.zeros(2, 16, 256, dtype=BF16, device=gpu)
    bad = [(q, table.long(), cu, lens), (q, table, cu.long(), lens), (q, table, cu, lens.cpu()), (q[:, :8], table, cu, lens),
           (q.float(), table, cu, lens), (q.transpose(0, 1), table, cu, lens), (q, table[0], cu, lens),
           (q, table, cu[:1], lens), (q, table.t(), cu, lens), (q[:0], table, cu, lens), (q, table[:0], cu, lens),
           (q, torch.zeros(1, 16393, dtype=torch.int32, device=gpu), cu, lens), (q.cpu(), table, cu, lens)]
    for x, t, u, n in bad:
        with pytest.raises(ValueError):
            pa.paged_attention(x, c, t, u, n)
    with pytest.raises(ValueError):
        pa.paged_attention(q, c, table, cu, lens, q_gate=torch.zeros(2, 4096, dtype=BF16, device=gpu))
    with pytest.raises(ValueError):
        pa.paged_attention(q, c, table, cu, lens, out=torch.zeros(2, 4096, device=gpu))
    with pytest.raises(ValueError):
        pa.select_pages(q, c, table, cu, lens, 4)                       # no bounds
    d, _ = filled_cache(gpu, b, 2, FP8, True, seed=1)
    for budget, sinks, recents in ((0, 0, 1), (2, 2, 1), (4, 0, 0), (1025, 1, 1), (4, -1, 1)):
        with pytest.raises(ValueError):
            pa.select_pages(q, d, table, cu, lens, budget, sinks, recents)
    for shape, dtype in (((2, 2, 1025), torch.int32), ((2, 2, 0), torch.int32), ((2, 1, 4), torch.int32),
                         ((2, 2, 4), torch.int64)):
        with pytest.raises(ValueError):
            pa.sparse_paged_attention(q, c, table, cu, lens, torch.zeros(shape, dtype=dtype, device=gpu))
    x = _step_inputs(gpu, b, 2)
    rope = fa.rotary_table(64, 0, gpu)
    for i, y in ((0, x[0][:, :8190]), (0, x[0].float()), (1, x[1][:, ::2]), (2, x[2][:1]), (3, x[3][:128]), (4, x[4].cpu())):
        z = list(x)
        z[i] = y
        with pytest.raises(ValueError):
            pa.paged_append(*z, rope, c, table, cu, lens)
    for r in ((rope[0], rope[1][:10]), (rope[0][:, :16], rope[1][:, :16]), (rope[0].double(), rope[1].double())):
        with pytest.raises(ValueError):
            pa.paged_append(*x, r, c, table, cu, lens)
    k = torch.zeros(4, 2, 16, 256, dtype=BF16, device=gpu)
    e = torch.zeros(4, 2, dtype=torch.uint8, device=gpu)
    for args in ((k, k[:3]), (k, k.float()), (k[..., ::2], k[..., ::2]), (k.to(FP8), k.to(FP8)), (k.to(FP8), k.to(FP8), e, e[:2]),
                 (k, k, None, None, torch.zeros(4, 2, 2, 256, dtype=torch.int8, device=gpu)), (k[:, :, :8], k[:, :, :8])):
        with pytest.raises(ValueError):
            pa.PagedKVCache.of(*args)
