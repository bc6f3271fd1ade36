"""The paged KV cache's operators against their plain forms in 64 bits and whole
numbers: ragged batches, page edges, both page types, head layouts, rows and
pages that hold nothing, non-finite values where a row must not look."""
import pytest
import torch

from qwen36_attn import full_attention as fa
from qwen36_attn import paged_attention as pa
from qwen36_attn import synthetic as syn
from tests import paged_reference as R

pytestmark = pytest.mark.gpu
FP8, BF16 = torch.float8_e4m3fn, torch.bfloat16


def filled_cache(gpu, b, heads, dtype, bounds=False, seed=0, junk=True):
    """A cache whose pages hold keys and values of every sequence; behind each
    sequence's end, and in pages of none, NaN bytes."""
    g = syn.gen(seed)
    c = pa.PagedKVCache(b.pool, b.page, gpu, dtype, heads, bounds)
    k = torch.randn(b.pool, heads, b.page, 256, generator=g) * torch.exp(0.4 * torch.randn(heads, 1, 256, generator=g))
    v = torch.randn(b.pool, heads, b.page, 256, generator=g)
    k, v = k.to(BF16), v.to(BF16)
    live = torch.zeros(b.pool, b.page, dtype=torch.bool)
    for i, n in enumerate(b.lens):
        for p in range(-(-n // b.page)):
            live[int(b.table[i, p]), :min(b.page, n - p * b.page)] = True
    state = R.CacheState(c)
    for pid in range(b.pool):
        for h in range(heads):
            if state.ke is not None:
                state.ke[pid, h] = R.least_byte(k[pid, h].abs().max().item())
                if bounds:
                    step = 4.0 * 2.0 ** (int(state.ke[pid, h]) - 127)
                    state.bounds[pid, h, 0] = torch.ceil(k[pid, h].double().amax(0) / step).to(torch.int8)
                    state.bounds[pid, h, 1] = torch.floor(k[pid, h].double().amin(0) / step).to(torch.int8)
            if state.ve is not None:
                state.ve[pid, h] = R.least_byte(v[pid, h].abs().max().item())
            if dtype == FP8:
                state.k[pid, h] = R.to_e4m3(k[pid, h].double() * 2.0 ** (127 - int(state.ke[pid, h])))
                state.v[pid, h] = R.to_e4m3(v[pid, h].double() * 2.0 ** (127 - int(state.ve[pid, h])))
            else:
                state.k[pid, h], state.v[pid, h] = k[pid, h], v[pid, h]
            if junk:
                state.k[pid, h][~live[pid]] = 0x7F if dtype == FP8 else float("nan")
                state.v[pid, h][~live[pid]] = 0x7F if dtype == FP8 else float("nan")
    upload(c, state)
    return c, state


def upload(c, state):
    if state.fp8:
        c.k_pages.view(torch.uint8).copy_(state.k)
        c.v_pages.view(torch.uint8).copy_(state.v)
    else:
        c.k_pages.copy_(state.k)
        c.v_pages.copy_(state.v)
    for mine, theirs in ((c.k_exp, state.ke), (c.v_exp, state.ve), (c.bounds, state.bounds)):
        if mine is not None:
            mine.copy_(theirs)


def check(got, want, tol, rows, at=""):
    got = got.double().cpu()
    for r in rows:
        assert torch.isfinite(got[r]).all(), (at, r)
        over = (got[r] - want[r]).abs() - tol[r]
        assert (over <= 0).all(), (at, r, over.max().item(), tol[r].max().item())


# ---------------------------------------------------------------- append

APPENDS = [  # lens, new: prompts from nothing, over a part of a page, single tokens, an empty sequence
    ([1], [1]), ([130], [130]), ([64, 17, 1], [64, 1, 1]), ([200, 70, 0, 33], [5, 70, 0, 16]),
    ([129, 128, 127, 300], [1, 128, 2, 171]), (list(range(1, 71)), [1] * 70)]


def layer_rows(gpu, t, heads, seed, scale=1.0):
    g = syn.gen(seed)
    hq = heads * 8
    wide = (torch.randn(t, (2 * hq + 2 * heads) * 256, generator=g) * scale).to(BF16).to(gpu)
    return (wide[:, :2 * hq * 256], wide[:, 2 * hq * 256:(2 * hq + heads) * 256], wide[:, (2 * hq + heads) * 256:],
            (0.3 * torch.randn(256, generator=g)).to(BF16).to(gpu), (0.3 * torch.randn(256, generator=g)).to(BF16).to(gpu))


def dense_norm(gpu, q_gate, k, v, qn, kn, heads, positions):
    """q and k of the dense path's head norm, row by row at the rows' positions
    (two KV heads a call)."""
    t = len(positions)
    q = torch.zeros(t, heads * 8, 256, dtype=BF16, device=gpu)
    ko = torch.zeros(t, heads, 256, dtype=BF16, device=gpu)
    kc = torch.zeros(max(positions + [0]) + 1, 2, 256, dtype=BF16, device=gpu)
    vc = torch.zeros_like(kc)
    for r, pos in enumerate(positions):
        if pos < 0:
            continue
        for h in range(0, heads, 2):
            n = min(2, heads - h)
            qg, kk, vv = (torch.zeros(1, w, dtype=BF16, device=gpu) for w in (8192, 512, 512))
            qg[:, :n * 4096] = q_gate[r, h * 4096:(h + n) * 4096]
            kk[:, :n * 256] = k[r, h * 256:(h + n) * 256]
            vv[:, :n * 256] = v[r, h * 256:(h + n) * 256]
            out = fa.head_norm_rope_kv_write(qg, kk, vv, qn, kn, kc, vc, pos)
            q[r, h * 8:(h + n) * 8] = out[0, :n * 8]
            ko[r, h:h + n] = kc[pos, :n]
    return q, ko


@pytest.mark.parametrize("dtype,bounds", [(FP8, False), (FP8, True), (BF16, False), (BF16, True)])
@pytest.mark.parametrize("page,heads", [(16, 2), (64, 1), (128, 3), (32, 2)])
@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_equals_the_plain_form(gpu, dtype, bounds, page, heads, case):
    lens, new = APPENDS[case]
    b = R.Batch(lens, new, page, seed=case, rows_behind=2)
    c, state = filled_cache(gpu, b, heads, dtype, bounds, seed=case + 10)
    rope = fa.rotary_table(512, 0, gpu)
    # larger rows than the cache's, so that scales grow under kept rows
    q_gate, k, v, qn, kn = layer_rows(gpu, b.tokens, heads, case + 20, 3.0)
    positions = [-1] * b.tokens
    for row, _, pos in b.rows():
        positions[row] = pos
    want_q, want_k = dense_norm(gpu, q_gate, k, v, qn, kn, heads, positions)
    state.append(b, want_k.cpu(), v.cpu().view(b.tokens, heads, 256))
    q = torch.full((b.tokens, heads * 8, 256), 7.0, dtype=BF16, device=gpu)
    got = pa.paged_append(q_gate, k, v, qn, kn, rope, c, *b.where(gpu), q_out=q)
    assert got is q
    for row, pos in enumerate(positions):
        want = want_q[row] if pos >= 0 else torch.full_like(want_q[row], 7.0)   # rows behind the last: untouched
        assert torch.equal(got[row], want), row
    state.same(c)


def test_append_token_by_token_keeps_bounds_of_the_whole(gpu):
    """A page filled one token a time has the bounds and scale of one filled at
    once, whatever the order of magnitudes, and each kept value is within half a
    step of the scale it was last rounded to, and half of the one before."""
    n, page = 64, 64
    rope = fa.rotary_table(n, 0, gpu)
    q_gate, k, v, qn, kn = layer_rows(gpu, n, 2, 5)
    v = (v.float() * torch.logspace(-6, 3, n, device=gpu)[torch.randperm(n, generator=syn.gen(1)).to(gpu), None]).to(BF16)
    one = pa.PagedKVCache(1, page, gpu, FP8, 2, True)
    many = pa.PagedKVCache(1, page, gpu, FP8, 2, True)
    table = torch.zeros(1, 1, dtype=torch.int32, device=gpu)

    def where(lo, hi):
        return table, torch.tensor([0, hi - lo], dtype=torch.int32, device=gpu), torch.tensor([hi], dtype=torch.int32, device=gpu)
    pa.paged_append(q_gate, k, v, qn, kn, rope, one, *where(0, n))
    state = R.CacheState(many)
    for i in range(n):
        r = slice(i, i + 1)
        pa.paged_append(q_gate[r], k[r], v[r], qn, kn, rope, many, *where(i, i + 1))
        _, kk = dense_norm(gpu, q_gate[r], k[r], v[r], qn, kn, 2, [i])
        b = R.Batch([i + 1], [1], page)
        b.table[:] = 0
        b.width = 1
        state.append(b, kk.cpu(), v[r].cpu().view(1, 2, 256))
        state.same(many)
    assert torch.equal(one.k_exp, many.k_exp) and torch.equal(one.v_exp, many.v_exp)
    assert torch.equal(one.bounds, many.bounds)
    _, va = one.values()
    _, vb = many.values()
    step = torch.exp2(many.v_exp.float() - 127.0)[:, :, None, None]
    # two roundings: 2^-4 of the value each, or half the smallest subnormal step 2^-9 of the scale
    tol = va.abs().float() * 2.0 ** -3 + step * 2.0 ** -9
    assert ((va.float() - vb.float()).abs() <= tol).all()


def test_append_nonfinite_values(gpu):
    b = R.Batch([40, 9], [7, 9], 16, seed=3)
    c, state = filled_cache(gpu, b, 2, FP8, True, seed=4)
    q_gate, k, v, qn, kn = layer_rows(gpu, b.tokens, 2, 6)
    v, k = v.clone(), k.clone()
    v[2, 5], v[3, 300], v[8, 1] = float("inf"), float("nan"), float("-inf")
    k[4, 10] = float("nan")       # the whole head of that row: a norm of NaN
    k[12, 300] = float("inf")
    positions = [-1] * b.tokens
    for row, _, pos in b.rows():
        positions[row] = pos
    want_q, want_k = dense_norm(gpu, q_gate, k, v, qn, kn, 2, positions)
    state.append(b, want_k.cpu(), v.cpu().view(-1, 2, 256))
    got = pa.paged_append(q_gate, k, v, qn, kn, fa.rotary_table(64, 0, gpu), c, *b.where(gpu))
    assert torch.equal(got, want_q)
    state.same(c)


def test_append_leaves_bad_batches_alone(gpu):
    """Page ids outside the pool, a sequence longer than its table or than the
    rotation tables, more rows than tokens: what has no place is not written."""
    b = R.Batch([40, 40, 40, 40], [20, 20, 20, 20], 16, seed=5)
    c, state = filled_cache(gpu, b, 2, FP8, True, seed=5)
    q_gate, k, v, qn, kn = layer_rows(gpu, b.tokens, 2, 7)
    b.table[0, 1], b.table[0, 2] = 10 ** 9, -5
    b.lens[1], b.lens[2], b.lens[3] = 49, 47, 9        # 49: over 3 pages of 16; 47: over 46 positions; 9: of 20 rows
    positions = [-1] * b.tokens
    for row, i, pos in b.rows():
        positions[row] = pos if i in (0, 3) else -1
    want_q, want_k = dense_norm(gpu, q_gate, k, v, qn, kn, 2, positions)
    lens = b.lens
    b.lens = [40, 0, 0, 9]
    state.append(b, want_k.cpu(), v.cpu().view(-1, 2, 256))
    b.lens = lens
    q = torch.full((b.tokens, 16, 256), 7.0, dtype=BF16, device=gpu)
    pa.paged_append(q_gate, k, v, qn, kn, fa.rotary_table(46, 0, gpu), c, *b.where(gpu), q_out=q)
    for row, pos in enumerate(positions):
        assert torch.equal(q[row], want_q[row] if pos >= 0 else torch.full_like(q[row], 7.0)), row
    state.same(c)


# ------------------------------------------------------------- attention

ATTENDS = [  # lens, new
    ([1], [1]), ([33], [1]), ([127, 128, 129, 16, 15], [1] * 5), ([700], [1]), ([40, 0, 300, 1], [2, 0, 5, 1]),
    ([90], [90]), ([513, 64, 65], [33, 64, 2]), (list(range(1, 300, 4)), [1] * 75), ([260, 31], [100, 31]),
    ([3, 200], [7, 1]), ([900, 40, 40, 40], [257, 1, 1, 1])]


@pytest.mark.parametrize("dtype", [FP8, BF16])
@pytest.mark.parametrize("page,heads", [(16, 2), (32, 1), (64, 2), (128, 3)])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention_equals_the_plain_form(gpu, dtype, page, heads, case):
    lens, new = ATTENDS[case]
    b = R.Batch(lens, new, page, seed=case, rows_behind=1)
    c, state = filled_cache(gpu, b, heads, dtype, seed=case + 30)
    g = syn.gen(case + 40)
    q = (1.5 * torch.randn(b.tokens, heads * 8, 256, generator=g)).to(BF16)
    gate = torch.randn(b.tokens, heads * 8 * 512, generator=g).to(BF16) if case % 2 else None
    out = torch.full((b.tokens, heads * 2048), 7.0, dtype=BF16, device=gpu)
    got = pa.paged_attention(q.to(gpu), c, *b.where(gpu), q_gate=None if gate is None else gate.to(gpu), out=out)
    assert got is out
    want, tol, rows = R.attend(state, b, q, gate)
    check(got, want, tol, rows)
    assert (got[b.tokens - 1] == 7.0).all()     # behind the last sequence
    again = pa.paged_attention(q.to(gpu), c, *b.where(gpu), q_gate=None if gate is None else gate.to(gpu))
    assert torch.equal(again[:b.tokens - 1], got[:b.tokens - 1])


@pytest.mark.parametrize("dtype", [FP8, BF16])
@pytest.mark.parametrize("lens,new", [([70, 40], [2, 5]), ([97], [97]), ([200, 64], [40, 33])])
def test_later_rows_of_nan_do_not_reach_earlier_ones(gpu, dtype, lens, new):
    """K and V of each sequence's last position are NaN: only its last row, which
    sees that position, may turn NaN."""
    b = R.Batch(lens, new, 16, seed=9)
    c, state = filled_cache(gpu, b, 2, dtype, seed=9)
    q = syn.randn((b.tokens, 16, 256), syn.gen(10))
    want, tol, rows = R.attend(state, b, q)
    last = [int(b.cu[i + 1]) - 1 for i in range(len(lens))]
    for kv in ("k", "v"):
        for i, n in enumerate(lens):
            page = getattr(state, kv)[int(b.table[i, (n - 1) // 16])]
            page[:, (n - 1) % 16] = 0x7F if dtype == FP8 else float("nan")
        upload(c, state)
        got = pa.paged_attention(q.to(gpu), c, *b.where(gpu))
        check(got, want, tol, [r for r in rows if r not in last], kv)
        assert torch.isnan(got[last]).all()


@pytest.mark.parametrize("new", [1, 2, 5, 12, 40])
@pytest.mark.parametrize("dtype", [FP8, BF16])
def test_queries_of_unequal_sizes_and_not_finite_ones(gpu, dtype, new):
    """Channels from 2^-30 to 2^3 in one query; a query with a NaN, one with an
    infinity: their rows are not finite, their neighbours as ever."""
    b = R.Batch([190, 77], [new, new], 32, seed=new)
    c, state = filled_cache(gpu, b, 2, dtype, seed=new)
    g = syn.gen(new)
    q = torch.randn(b.tokens, 16, 256, generator=g) * torch.exp2(torch.randint(-30, 4, (1, 1, 256), generator=g).float())
    q = q.to(BF16)
    q[new - 1, 3, 17], q[b.tokens - 1, 9, 200] = float("nan"), float("inf")
    q2 = q.clone()
    q2[new - 1, 3], q2[b.tokens - 1, 9] = 0, 0
    want, tol, rows = R.attend(state, b, q2)
    got = pa.paged_attention(q.to(gpu), c, *b.where(gpu)).view(b.tokens, 16, 256)
    assert not torch.isfinite(got[new - 1, 3]).any() and not torch.isfinite(got[b.tokens - 1, 9]).any()
    got[new - 1, 3] = want.view(b.tokens, 16, 256)[new - 1, 3].to(got)
    got[b.tokens - 1, 9] = want.view(b.tokens, 16, 256)[b.tokens - 1, 9].to(got)
    tol = tol + 2.0 ** -8 * want.abs()      # of the two rows put in above
    check(got.flatten(1), want, tol, rows)


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** -20, 2.0 ** 6])
def test_queries_of_all_sizes(gpu, scale):
    b = R.Batch([130], [50], 16, seed=1)
    c, state = filled_cache(gpu, b, 1, FP8, seed=1)
    q = (syn.randn((50, 8, 256), syn.gen(3)).float() * scale).to(BF16)
    want, tol, rows = R.attend(state, b, q)
    check(pa.paged_attention(q.to(gpu), c, *b.where(gpu)), want, tol, rows)


@pytest.mark.parametrize("scale", [1.5, 2.0 ** 6])
@pytest.mark.parametrize("dtype", [FP8, BF16])
@pytest.mark.parametrize("lens,new", [([3, 8, 32, 33], [3, 8, 8, 3]), ([64, 65, 96, 97, 128, 129], [4, 5, 8, 8, 1, 8]),
                                      ([1100, 2081, 40], [5, 8, 7]), ([5000], [8]), ([31, 0, 0, 2050], [6, 0, 0, 6])])
def test_drafts_over_parts_of_a_stage(gpu, lens, new, dtype, scale):
    """Three to eight rows a sequence, whose keys end in either half of 64, or leave the
    second half empty; large queries put the two halves' maxima far apart."""
    b = R.Batch(lens, new, 16, seed=sum(lens), rows_behind=1)
    c, state = filled_cache(gpu, b, 2, dtype, seed=sum(new))
    g = syn.gen(len(lens))
    q = (syn.randn((b.tokens, 16, 256), g).float() * scale).to(BF16)
    gate = torch.randn(b.tokens, 16 * 512, generator=g).to(BF16)
    want, tol, rows = R.attend(state, b, q, gate)
    check(pa.paged_attention(q.to(gpu), c, *b.where(gpu), q_gate=gate.to(gpu)), want, tol, rows)


def test_attention_with_pages_that_hold_nothing(gpu):
    """Page ids outside the pool hold no tokens; a row whose pages are all such,
    a sequence longer than its table and rows of negative position are zeros."""
    b = R.Batch([100, 60, 50, 5], [3, 1, 2, 9], 16, seed=2)
    c, state = filled_cache(gpu, b, 2, FP8, seed=2)
    b.table[0, 2], b.table[0, 5] = b.pool, -1
    b.table[1, :] = 2 ** 31 - 1
    b.lens[2] = b.width * 16 + 1
    q = syn.randn((b.tokens, 16, 256), syn.gen(3))
    want, tol, rows = R.attend(state, b, q)
    got = pa.paged_attention(q.to(gpu), c, *b.where(gpu))
    check(got, want, tol, rows)
    assert (got[3:6] == 0).all() and (got[6:10] == 0).all() and (got[10:] != 0).any()


@pytest.mark.parametrize("dtype", [FP8, BF16])
def test_long_decode_splits_agree(gpu, dtype):
    """20,000 keys, far more chunks than a short call, and a large pool whose last
    pages lie past 2^32 bytes."""
    page, n = 128, 20000
    need = -(-n // page)
    pool = (1 << 32) // (2 * page * 256 * (1 if dtype == FP8 else 2)) + need + 5
    k = torch.zeros(pool, 2, page, 256, dtype=torch.uint8, device=gpu).view(FP8) if dtype == FP8 else torch.zeros(
        pool, 2, page, 256, dtype=BF16, device=gpu)
    v = torch.zeros_like(k.view(torch.uint8)).view(FP8) if dtype == FP8 else torch.zeros_like(k)
    exps = [torch.full((pool, 2), 127, dtype=torch.uint8, device=gpu) for _ in range(2)] if dtype == FP8 else [None] * 2
    g = syn.gen(4)
    kk, vv = (torch.randn(need, 2, page, 256, generator=g).to(BF16).to(dtype) for _ in range(2))
    at = torch.arange(pool - need, pool)
    for pages, x in ((k, kk), (v, vv)):
        pages.view(torch.uint8)[pool - need:] = x.to(gpu).view(torch.uint8)
    c = pa.PagedKVCache.of(k, v, *exps)
    q = syn.randn((1, 16, 256), g)
    got = pa.paged_attention(q.to(gpu), c, at.to(torch.int32).view(1, -1).to(gpu), torch.tensor([0, 1], dtype=torch.int32, device=gpu),
                             torch.tensor([n], dtype=torch.int32, device=gpu)).double().cpu()
    for h in range(2):
        ks, vs = (x.double()[:, h].reshape(-1, 256)[:n] for x in (kk, vv))
        qq = q[0, 8 * h:8 * h + 8].double()
        p = torch.softmax(qq @ ks.t() / 16, -1)
        score = (qq.abs() @ ks.abs().t()).amax(-1, keepdim=True) / 16 * 258 * 2.0 ** -24
        o = p @ vs
        tol = (2.0 ** -8 + 2 * score + (2 * n + 64) * 2.0 ** -24) * (p @ vs.abs()) + 2.0 ** -8 * o.abs()
        assert ((got[0].view(16, 256)[8 * h:8 * h + 8] - o).abs() <= tol).all()


# ---------------------------------------------------------------- sparse

@pytest.mark.parametrize("dtype", [FP8, BF16])
@pytest.mark.parametrize("page,heads,lens,new,budget,sinks,recents", [
    (16, 2, [900, 30, 0, 333], [1, 1, 0, 1], 8, 1, 1), (32, 1, [700, 64], [9, 3], 5, 0, 1), (64, 3, [1500], [1], 24, 2, 3),
    (128, 2, [1300, 1290], [2, 20], 3, 1, 2), (16, 2, [250], [250], 7, 3, 4), (16, 1, [17], [1], 1, 0, 1)])
def test_selection_and_sparse_attention(gpu, dtype, page, heads, lens, new, budget, sinks, recents):
    b = R.Batch(lens, new, page, seed=budget, rows_behind=1)
    c, state = filled_cache(gpu, b, heads, dtype, True, seed=budget + 1)
    g = syn.gen(budget + 2)
    q = (2.0 * torch.randn(b.tokens, heads * 8, 256, generator=g)).to(BF16)
    gate = torch.randn(b.tokens, heads * 8 * 512, generator=g).to(BF16)
    pages = torch.full((b.tokens, heads, budget), 77, dtype=torch.int32, device=gpu)
    pa.select_pages(q.to(gpu), c, *b.where(gpu), budget, sinks, recents, out=pages)
    want = R.select(state, b, q, budget, sinks, recents)
    got = pages.cpu()
    for (row, h), mine in want.items():
        assert got[row, h].tolist() == mine + [-1] * (budget - len(mine)), (row, h)
    assert (got[-1] == 77).all()
    out = pa.sparse_paged_attention(q.to(gpu), c, *b.where(gpu), pages, q_gate=gate.to(gpu))
    ref, tol, rows = R.attend(state, b, q, gate, got)
    check(out, ref, tol, rows)


def test_selection_ties_and_odd_queries(gpu):
    """Equal pages: the lowest are taken.  Queries with NaN, infinities, zeros, and
    of the least and largest magnitudes, and pages outside the pool."""
    b = R.Batch([16 * 40], [6], 16, seed=1)
    c, state = filled_cache(gpu, b, 2, FP8, True, seed=1)
    for p in range(3, 30):
        state.bounds[int(b.table[0, p])] = state.bounds[int(b.table[0, 2])]
        state.ke[int(b.table[0, p])] = state.ke[int(b.table[0, 2])]
    upload(c, state)
    b.table[0, 33], b.table[0, 4] = -1, b.pool + 9
    q = syn.randn((6, 16, 256), syn.gen(2))
    q[0, 3, 9], q[0, 4, 10], q[0, 12, 7] = float("nan"), float("inf"), float("-inf")
    q[1] = 0
    q[2] *= 2.0 ** -120
    q[3] = (q[3].float() * 2.0 ** 124).to(BF16)
    q[4, :8] = float("nan")
    got = pa.select_pages(q.to(gpu), c, *b.where(gpu), 9, 1, 1).cpu()
    for (row, h), mine in R.select(state, b, q, 9, 1, 1).items():
        assert got[row, h].tolist() == mine, (row, h)


@pytest.mark.parametrize("lens,new,page", [
    ([330, 290, 50, 401], [3, 5, 0, 7], 16), ([257, 258, 259], [2, 2, 3], 16), ([1, 600, 0, 1, 700], [1, 1, 0, 1, 33], 32),
    ([2100], [131], 64), ([3, 640], [9, 6], 16)])
def test_selection_for_rows_by_twos(gpu, lens, new, page):
    """Sequences of odd numbers of rows, rows on both sides of a page's end, rows of
    negative position, and neighbours whose queries are of quite different sizes."""
    b = R.Batch(lens, new, page, seed=len(lens))
    c, state = filled_cache(gpu, b, 2, FP8, True, seed=sum(new))
    g = syn.gen(sum(lens))
    q = torch.randn(b.tokens, 16, 256, generator=g) * torch.exp2(torch.randint(-9, 9, (b.tokens, 1, 1), generator=g).float())
    q = q.to(BF16)
    got = pa.select_pages(q.to(gpu), c, *b.where(gpu), 6, 1, 2).cpu()
    for (row, h), mine in R.select(state, b, q, 6, 1, 2).items():
        assert got[row, h].tolist() == mine + [-1] * (6 - len(mine)), (row, h)


def test_selection_over_many_pages(gpu):
    """More pages than one register block: 5,000 pages of 16 tokens."""
    n = 80000
    b = R.Batch([n], [1], 16, seed=6)
    c = pa.PagedKVCache(b.pool, 16, gpu, FP8, 1, True)
    g = syn.gen(8)
    c.bounds.copy_(torch.randint(-100, 101, c.bounds.shape, generator=g, dtype=torch.int8).sort(2, descending=True)[0])
    c.k_exp.copy_(torch.randint(118, 121, c.k_exp.shape, generator=g, dtype=torch.uint8))
    state = R.CacheState(c)
    q = syn.randn((1, 8, 256), g)
    for budget in (2, 100, 1024):
        got = pa.select_pages(q.to(gpu), c, *b.where(gpu), budget).cpu()
        assert got[0, 0].tolist() == R.select(state, b, q, budget, 1, 1)[0, 0]


def test_sparse_lists_of_any_order(gpu):
    """Unsorted lists, repeats (counted twice), indices of no page."""
    b = R.Batch([300, 45], [2, 1], 16, seed=7)
    c, state = filled_cache(gpu, b, 2, FP8, seed=7)
    pages = torch.tensor([[[18, 3, 3, -1, 99], [0, 17, 1, 2 ** 31 - 1, -7]], [[18, 18, 18, 0, 5], [-1] * 5],
                          [[1, 0, 2, 3, 1], [2, -1, -1, -1, -1]]], dtype=torch.int32)
    q = syn.randn((3, 16, 256), syn.gen(8))
    want, tol, rows = R.attend(state, b, q, None, pages)
    got = pa.sparse_paged_attention(q.to(gpu), c, *b.where(gpu), pages.to(gpu))
    check(got, want, tol, rows)
    assert (got[1].view(2, -1)[1] == 0).all()


def test_sparse_of_all_pages_is_the_dense_attention(gpu):
    b = R.Batch([1000], [1], 16, seed=7)
    c, state = filled_cache(gpu, b, 2, FP8, True, seed=7)
    q = syn.randn((1, 16, 256), syn.gen(8))
    pages = pa.select_pages(q.to(gpu), c, *b.where(gpu), 100)
    assert pages[0, 0].tolist() == list(range(63)) + [-1] * 37
    got = pa.sparse_paged_attention(q.to(gpu), c, *b.where(gpu), pages)
    want, tol, rows = R.attend(state, b, q)
    check(got, want, tol, rows)
