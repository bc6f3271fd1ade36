"""The Gated-DeltaNet convolution and delta rule over ragged batches against plain
forms in 64 bits: lengths from one token to many chunks, slots in any order,
sequences without a state, padding, strides, captured calls, the layer."""
import pytest
import torch

from qwen36_attn import gated_deltanet as gd
from qwen36_attn import ragged_deltanet as rd
from qwen36_attn import synthetic as syn
from tests import ragged_reference as R

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def batch(lens, slots, has, gpu):
    return (torch.tensor(R.cu_of(lens), dtype=torch.int32, device=gpu),
            torch.tensor(slots, dtype=torch.int32, device=gpu), torch.tensor(has, device=gpu))


CONV = [([1], [2], [True], 0), ([1], [0], [False], 1), ([2, 1, 3], [3, 0, 1], [True, False, True], 0),
        ([4, 5, 0, 17, 1, 66], [5, 2, 3, 0, 6, 1], [True, False, True, True, False, True], 3),
        ([3, 2, 7], [-1, 4, 9], [True, True, True], 2), ([1] * 70, list(range(69, -1, -1)), [i % 3 > 0 for i in range(70)], 0),
        ([9, 200, 1], [1, 0, 2], [False, False, True], 5)]


@pytest.mark.parametrize("lens,slots,has,behind", CONV)
def test_conv(gpu, lens, slots, has, behind):
    """Against 64 bits, and bit for bit against the operator of one sequence.  The sum is
    rounded to bf16 (off by a step of 2^-8 of it where 32 and 64 bits fall on two sides:
    SiLU's slope is below 1.1), the result once more."""
    g = torch.Generator(device=gpu).manual_seed(len(lens))
    t, n = sum(lens) + behind, max(7, len(lens))
    x = torch.randn(t, 8192 + 24, generator=g, device=gpu).to(BF16)[:, :8192]
    w = torch.randn(8192, 4, generator=g, device=gpu).to(BF16)
    pool = torch.randn(n, 2, 8192, 3, generator=g, device=gpu).to(BF16)
    states, before = pool[:, 0], pool.clone()
    out = torch.full((t, 8192), 7.0, dtype=BF16, device=gpu)
    cu, sl, h = batch(lens, slots, has, gpu)
    rd.ragged_conv1d(x, w, states, cu, sl, h, out=out)
    want, after = R.conv(x, w, before[:, 0], R.cu_of(lens), slots, has)
    there = ~want.isnan()
    assert torch.equal(out[~there], torch.full_like(out[~there], 7.0))
    y = out[there].double()
    assert ((y - want[there]).abs() <= 2.0 ** -8 * want[there].abs() + 1.1 * 2.0 ** -7 * want[there].abs() + 1e-4).all()
    assert ((y - want[there]).norm() / want[there].norm()).item() <= 2.0 ** -8
    assert torch.equal(states.double(), after)
    assert torch.equal(pool[:, 1], before[:, 1])
    a = 0
    for m, slot, hs in zip(lens, slots, has):
        if m and 0 <= slot < n:
            old = before[slot, 0].contiguous() if hs else torch.zeros(8192, 3, dtype=BF16, device=gpu)
            one, last = gd.causal_conv1d(x[a:a + m], old, w)
            assert torch.equal(out[a:a + m], one) and torch.equal(states[slot], last)
        a += m


def core(gpu, t, seed, a_max=2.0, qk_heads=16, pad=0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    x = torch.nn.functional.silu(torch.randn(t, 2 * qk_heads * 128 + 4096 + pad, generator=g, device=gpu)).to(BF16)
    q = x[:, :qk_heads * 128].view(t, qk_heads, 128)
    k = x[:, qk_heads * 128:2 * qk_heads * 128].view(t, qk_heads, 128)
    v = x[:, 2 * qk_heads * 128:2 * qk_heads * 128 + 4096].view(t, 32, 128)
    gg = -torch.nn.functional.softplus(torch.randn(t, 32, generator=g, device=gpu)) \
        * torch.rand(32, generator=g, device=gpu) * a_max
    return q, k, v, gg, torch.sigmoid(torch.randn(t, 32, generator=g, device=gpu)), g


def check_delta(out, states, want, after, untouched):
    """fp32 dot products of 128 keys or 64 tokens, a few roundings each: 256 units of 2^-24
    of the 2-norm (earlier errors decay with the state that holds them), which is at most
    2^-12 of a row's largest value for an element; the output is rounded to bf16."""
    there = ~want.isnan()
    assert torch.equal(out[~there], torch.full_like(out[~there], 7.0))
    err = (out.double() - want).abs()
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -12 * want.abs().amax(-1, keepdim=True)
    bad = there & ~(err <= tol)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), (err / tol)[there].max().item())
    rel = (states.double() - after).flatten(1).norm(dim=1) / after.flatten(1).norm(dim=1).clamp(min=1e-30)
    print("state errors", rel.max().item(), flush=True)
    assert rel.max().item() <= 256 * 2.0 ** -24
    assert torch.equal(states[untouched].double(), after[untouched])


DELTA = [([1], [2], [True], 0, None), ([1], [0], [False], 2, 1), ([2, 1, 8], [3, 0, 1], [True, False, True], 0, 8),
         ([9, 16, 17, 1], [3, 0, 1, 4], [True, False, True, True], 1, None),
         ([64, 63, 65, 0, 1, 128], [5, 2, 3, 0, 6, 1], [True, False, True, True, False, True], 3, 128),
         ([64, 63, 65, 0, 1, 128], [5, 2, 3, 0, 6, 1], [False, True, True, True, False, False], 0, None),
         ([70, 30, 3], [-1, 4, 9], [True, True, True], 2, 70), ([1] * 70, list(range(69, -1, -1)), [i % 3 > 0 for i in range(70)], 0, 1),
         ([1] * 66 + [130] + [1] * 3 + [77], list(range(71)), [i % 5 > 0 for i in range(71)], 0, None),
         ([1, 513, 2, 40], [3, 2, 1, 0], [True, True, False, False], 0, 1),       # more rows than `longest` says
         ([1000], [1], [True], 0, 1000)]


@pytest.mark.parametrize("lens,slots,has,behind,longest", DELTA)
def test_delta(gpu, lens, slots, has, behind, longest):
    t, n = sum(lens) + behind, max(7, len(lens))
    q, k, v, g, beta, gen = core(gpu, t, 3 * len(lens) + max(lens))
    states = torch.randn(n, 32, 128, 128, generator=gen, device=gpu) * 0.2
    before = states.clone()
    out = torch.full((t, 32, 128), 7.0, dtype=BF16, device=gpu)
    cu, sl, h = batch(lens, slots, has, gpu)
    print("delta", lens[:8], longest, flush=True)
    rd.ragged_delta_rule(q, k, v, g, beta, states, cu, sl, h, out=out, longest=longest)
    want, after = R.delta(q, k, v, g, beta, before, R.cu_of(lens), slots, has)
    used = {s for s, m in zip(slots, lens) if m}
    check_delta(out, states, want, after, [i for i in range(n) if i not in used])


@pytest.mark.parametrize("a_max", [16.0, 0.02])
@pytest.mark.parametrize("qk_heads,pad", [(16, 40), (32, 8)])
def test_delta_decays_heads_and_strides(gpu, a_max, qk_heads, pad):
    """Fast and slow decays, 32 repeated key heads, padded rows, slots apart."""
    lens, slots, has = [150, 1, 12, 300], [2, 0, 3, 1], [True, True, False, True]
    q, k, v, g, beta, gen = core(gpu, sum(lens), 11, a_max, qk_heads, pad)
    pool = torch.randn(5, 2, 32, 128, 128, generator=gen, device=gpu) * 0.2
    before = pool.clone()
    out = torch.full((sum(lens), 32, 128), 7.0, dtype=BF16, device=gpu)
    cu, sl, h = batch(lens, slots, has, gpu)
    rd.ragged_delta_rule(q, k, v, g, beta, pool[:, 1], cu, sl, h, out=out)
    want, after = R.delta(q, k, v, g, beta, before[:, 1], R.cu_of(lens), slots, has)
    check_delta(out, pool[:, 1], want, after, [4])
    assert torch.equal(pool[:, 0], before[:, 0])


def test_delta_of_rows_without_keys(gpu):
    """Rows of zeros (a norm of nothing), gates of zero and decays to nothing."""
    lens, slots, has = [100, 3], [0, 1], [True, True]
    q, k, v, g, beta, gen = core(gpu, 103, 5)
    q, k, beta, g = q.clone(), k.clone(), beta.clone(), g.clone()
    k[10:20] = 0
    q[30:40] = 0
    beta[50:60] = 0
    g[70] = -200.0
    g[101] = -1000.0
    states = torch.randn(3, 32, 128, 128, generator=gen, device=gpu)
    before = states.clone()
    out = torch.full((103, 32, 128), 7.0, dtype=BF16, device=gpu)
    rd.ragged_delta_rule(q, k, v, g, beta, states, *batch(lens, slots, has, gpu), out=out)
    want, after = R.delta(q, k, v, g, beta, before, R.cu_of(lens), slots, has)
    check_delta(out, states, want, after, [2])


def test_captured_calls_follow_the_batch(gpu):
    """One capture, replayed over other lengths, slots and states, with eager work
    between; each replay against the eager call."""
    t, n = 160, 6
    q, k, v, g, beta, gen = core(gpu, t, 9)
    w = torch.randn(8192, 4, generator=gen, device=gpu).to(BF16)
    x = torch.randn(t, 8192, generator=gen, device=gpu).to(BF16)
    conv = torch.randn(n, 8192, 3, generator=gen, device=gpu).to(BF16)
    ssm = torch.randn(n, 32, 128, 128, generator=gen, device=gpu) * 0.2
    cu, sl, h = batch([100, 1, 59], [0, 1, 2], [True] * 3, gpu)
    first = conv.clone(), ssm.clone()

    def step():
        return rd.ragged_conv1d(x, w, conv, cu, sl, h), rd.ragged_delta_rule(q, k, v, g, beta, ssm, cu, sl, h)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for lens, slots, has in (([100, 1, 59], [0, 1, 2], [True] * 3), ([1, 1, 1], [5, 3, 4], [True, False, True]),
                             ([0, 130, 30], [1, 0, 5], [False, True, True]), ([1, 2, 157], [2, -1, 3], [True] * 3)):
        for p, q0 in zip((conv, ssm), first):
            p.copy_(q0)
        for p, q0 in zip((cu, sl, h), batch(lens, slots, has, gpu)):
            p.copy_(q0)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs] + [conv.clone(), ssm.clone()]
        for p, q0 in zip((conv, ssm), first):
            p.copy_(q0)
        rows = torch.zeros(t, dtype=torch.bool, device=gpu)
        for a, z, s in zip(R.cu_of(lens), R.cu_of(lens)[1:], slots):
            rows[a:z] = s >= 0
        want = list(step()) + [conv, ssm]
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a[rows] if i < 2 else a, b[rows] if i < 2 else b), (lens, i)


def test_layer_over_prompts_and_decode_steps(gpu):
    """The layer over a batch against the layer of one sequence, turn by turn."""
    w = {k: v.to(gpu) for k, v in syn.linear_attention_weights(syn.gen(4), a_max=2.0).items()}
    n, slots = 3, [4, 0, 2]
    conv = torch.full((5, 8192, 3), 3.0, dtype=BF16, device=gpu)
    ssm = torch.full((5, 32, 128, 128), 3.0, device=gpu)
    layer = rd.RaggedLinearAttentionLayer(w, conv, ssm)
    singles = [gd.LinearAttentionLayer(w, gpu) for _ in range(n)]
    for step, lens in enumerate(([70, 5, 130], [1, 33, 1], [1, 1, 1], [0, 1, 0])):
        inp = syn.randn((sum(lens), 2048), syn.gen(50 + step)).to(gpu)
        cu, sl, h = batch(lens, slots, [step > 0] * n, gpu)
        got = layer.forward(inp, cu, sl, h, longest=max(lens))
        for i, (a, m) in enumerate(zip(R.cu_of(lens), lens)):
            if m:
                one = singles[i].forward(inp[a:a + m], "prefill" if m > 1 else "decode")
                # bf16 roundings of the projections (each of another product order), the conv,
                # the norm's two and the output, carried through the delta rule: 8 of 2^-8 at most
                rel = ((got[a:a + m].double() - one.double()).norm() / one.double().norm()).item()
                assert rel <= 8 * 2.0 ** -8, (step, i, rel)
                s = (ssm[slots[i]].double() - singles[i].ssm_state.double()).norm() / singles[i].ssm_state.double().norm()
                assert s.item() <= 8 * 2.0 ** -8
    assert (ssm[1] == 3.0).all() and (conv[3] == 3.0).all()


def test_on_another_stream(gpu):
    lens, slots, has = [5, 90], [1, 0], [True, True]
    q, k, v, g, beta, gen = core(gpu, 95, 21)
    states = torch.randn(2, 32, 128, 128, generator=gen, device=gpu)
    other = states.clone()
    want = rd.ragged_delta_rule(q, k, v, g, beta, states, *batch(lens, slots, has, gpu))
    where = batch(lens, slots, has, gpu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = rd.ragged_delta_rule(q, k, v, g, beta, other, *where)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(other, states)


@pytest.mark.parametrize("lens,qk_heads", [([200, 330, 257, 70, 500, 12, 13], 16), ([449, 13, 64, 320, 1, 193], 32)])
def test_delta_of_many_chunks(gpu, lens, qk_heads):
    n = len(lens)
    slots, has = [(3 * i + 1) % n if n % 3 else (5 * i + 1) % n for i in range(n)], [i % 3 != 1 for i in range(n)]
    q, k, v, g, beta, gen = core(gpu, sum(lens), 31, 0.5, qk_heads)
    states = torch.randn(n, 32, 128, 128, generator=gen, device=gpu)
    before = states.clone()
    out = torch.full((sum(lens), 32, 128), 7.0, dtype=BF16, device=gpu)
    rd.ragged_delta_rule(q, k, v, g, beta, states, *batch(lens, slots, has, gpu), out=out, longest=max(lens))
    want, after = R.delta(q, k, v, g, beta, before, R.cu_of(lens), slots, has)
    check_delta(out, states, want, after, [])


def test_delta_without_decay_and_with_reflections(gpu):
    """g = 0 and beta = 2, the ends of what the gates give: every token reflects the state."""
    lens, slots, has = [300, 70, 5], [2, 0, 1], [True, False, True]
    q, k, v, g, beta, gen = core(gpu, sum(lens), 17)
    states = torch.randn(3, 32, 128, 128, generator=gen, device=gpu)
    before = states.clone()
    out = torch.full((sum(lens), 32, 128), 7.0, dtype=BF16, device=gpu)
    rd.ragged_delta_rule(q, k, v, torch.zeros_like(g), torch.full_like(beta, 2.0), states, *batch(lens, slots, has, gpu), out=out)
    want, after = R.delta(q, k, v, torch.zeros_like(g), torch.full_like(beta, 2.0), before, R.cu_of(lens), slots, has)
    check_delta(out, states, want, after, [])


def test_states_far_apart(gpu):
    """Slots behind 2^31 elements and 2^32 bytes of their pools."""
    lens, slots, has = [3, 80], [2, 1], [True, True]
    q, k, v, g, beta, gen = core(gpu, sum(lens), 23)
    at, size = 2 ** 30 + 128, 32 * 128 * 128
    states = torch.empty(2 * at + size, device=gpu).as_strided((3, 32, 128, 128), (at, 128 * 128, 128, 1))
    near = torch.randn(3, 32, 128, 128, generator=gen, device=gpu)
    states[1:] = near[1:]
    where = batch(lens, slots, has, gpu)
    got = rd.ragged_delta_rule(q, k, v, g, beta, states, *where)
    assert torch.equal(got, rd.ragged_delta_rule(q, k, v, g, beta, near, *where)) and torch.equal(states[1:], near[1:])
    rd.fork_states([states], torch.tensor([2, -1, -1], dtype=torch.int32, device=gpu))
    assert torch.equal(states[0], near[2])
    del states
    x = torch.randn(sum(lens), 8192, generator=gen, device=gpu).to(BF16)
    w = torch.randn(8192, 4, generator=gen, device=gpu).to(BF16)
    conv = torch.empty(2 * at + 8192 * 3, dtype=BF16, device=gpu).as_strided((3, 8192, 3), (at, 3, 1))
    close = torch.randn(3, 8192, 3, generator=gen, device=gpu).to(BF16)
    conv[1:] = close[1:]
    got = rd.ragged_conv1d(x, w, conv, *where)
    assert torch.equal(got, rd.ragged_conv1d(x, w, close, *where)) and torch.equal(conv[1:], close[1:])


def test_two_calls_at_once(gpu):
    """Calls on two streams, their workspaces their own."""
    lens, slots, has = [700, 90, 400, 13, 64], [1, 0, 3, 2, 4], [True] * 5
    q, k, v, g, beta, gen = core(gpu, sum(lens), 29)
    first = torch.randn(5, 32, 128, 128, generator=gen, device=gpu)
    where = batch(lens, slots, has, gpu)
    ins = [(q, k, v, g, beta), (k, q, v, 0.5 * g, 1 - beta)]
    want = []
    for x in ins:
        states = first.clone()
        want += [rd.ragged_delta_rule(*x, states, *where), states]
    pools = [first.clone() for _ in range(6)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for n in range(6):
        with torch.cuda.stream(streams[n % 2]):
            got.append(rd.ragged_delta_rule(*ins[n % 2], pools[n], *where))
    torch.cuda.synchronize()
    for n in range(6):
        assert torch.equal(got[n], want[2 * (n % 2)]) and torch.equal(pools[n], want[2 * (n % 2) + 1])


def test_delta_of_hundreds_of_sequences(gpu):
    """More sequences than a wave has lanes, of all kinds, some of them padding."""
    n = 150
    lens = [(7 * i) % 23 if i % 31 else 70 + i for i in range(n)]
    slots, has = [(11 * i + 3) % n if i % 9 != 4 else -1 for i in range(n)], [i % 4 > 0 for i in range(n)]
    q, k, v, g, beta, gen = core(gpu, sum(lens), 37)
    states = torch.randn(n, 32, 128, 128, generator=gen, device=gpu) * 0.3
    before = states.clone()
    out = torch.full((sum(lens), 32, 128), 7.0, dtype=BF16, device=gpu)
    rd.ragged_delta_rule(q, k, v, g, beta, states, *batch(lens, slots, has, gpu), out=out)
    want, after = R.delta(q, k, v, g, beta, before, R.cu_of(lens), slots, has)
    used = {s for s, m in zip(slots, lens) if m}
    check_delta(out, states, want, after, [i for i in range(n) if i not in used])


def test_as_many_sequences_as_a_call_has(gpu):
    """65,536 rows of a sequence each, all but a few of them padding."""
    n, real = 65536, {0: 2, 63: 0, 64: 5, 40000: 1, 65535: 3}
    q, k, v, g, beta, gen = core(gpu, n, 41)
    x = torch.randn(n, 8192, generator=gen, device=gpu).to(BF16)
    w = torch.randn(8192, 4, generator=gen, device=gpu).to(BF16)
    slots = torch.full((n,), -1, dtype=torch.int32, device=gpu)
    for i, s in real.items():
        slots[i] = s
    cu = torch.arange(n + 1, dtype=torch.int32, device=gpu)
    states, conv = torch.randn(6, 32, 128, 128, generator=gen, device=gpu), torch.randn(6, 8192, 3, generator=gen, device=gpu).to(BF16)
    few, few_conv, at = states.clone(), conv.clone(), torch.tensor(list(real), device=gpu)
    where = batch([1] * len(real), list(real.values()), [True] * len(real), gpu)
    got = rd.ragged_delta_rule(q, k, v, g, beta, states, cu, slots, longest=1)
    want = rd.ragged_delta_rule(q[at], k[at], v[at], g[at], beta[at], few, *where, longest=1)
    assert torch.equal(got[at], want) and torch.equal(states, few)
    got, want = rd.ragged_conv1d(x, w, conv, cu, slots), rd.ragged_conv1d(x[at], w, few_conv, *where)
    assert torch.equal(got[at], want) and torch.equal(conv, few_conv)


@pytest.mark.parametrize("cu,slots", [([5, -3, 1 << 30, 7, 40], [0, 1, 7, -5]), ([0, 90, 30, 90, 200], [2, 3, 0, 1 << 30]),
                                      ([-(1 << 31), (1 << 31) - 1, 0, 64, 1], [1, -(1 << 31), 2, 0])])
def test_offsets_that_make_no_sense(gpu, cu, slots):
    """They are cut to the call's rows: nothing around its tensors changes."""
    t, n = 90, 4
    q, k, v, g, beta, gen = core(gpu, t, 43)
    out, pool = torch.full((t + 64, 32, 128), 7.0, dtype=BF16, device=gpu), torch.full((n + 2, 32, 128, 128), 0.5, device=gpu)
    rows, conv = torch.full((t + 64, 8192), 7.0, dtype=BF16, device=gpu), torch.full((n + 2, 8192, 3), 0.5, dtype=BF16, device=gpu)
    x = torch.randn(t, 8192, generator=gen, device=gpu).to(BF16)
    w = torch.randn(8192, 4, generator=gen, device=gpu).to(BF16)
    cu, sl = torch.tensor(cu, device=gpu).to(torch.int32), torch.tensor(slots, device=gpu).to(torch.int32)
    named = [s for s in slots if 0 <= s < n]
    for longest in (None, 1):
        rd.ragged_delta_rule(q, k, v, g, beta, pool[1:n + 1], cu, sl, out=out[32:t + 32], longest=longest)
        rd.ragged_conv1d(x, w, conv[1:n + 1], cu, sl, out=rows[32:t + 32])
        for y in (out, rows):
            assert (y[:32] == 7.0).all() and (y[t + 32:] == 7.0).all()
        for p in (pool, conv):
            for s in set(range(-1, n + 1)) - set(named):
                assert (p[s + 1] == 0.5).all(), s


@pytest.mark.parametrize("flags", [gd.QK_NORMALIZED, gd.STATE_VK, gd.QK_NORMALIZED | gd.STATE_VK])
@pytest.mark.parametrize("lens", [[5, 1, 0, 7, 2], [130, 1, 64, 9, 7], [300]])
def test_delta_flags(gpu, lens, flags):
    """q and k as given (of norm 1, rounded to bf16), states by columns."""
    n = len(lens)
    slots, has = [(2 * i + 1) % n for i in range(n)], [i % 2 == 0 for i in range(n)]
    q, k, v, g, beta, gen = core(gpu, sum(lens), 47)
    as_given, by_columns = bool(flags & gd.QK_NORMALIZED), bool(flags & gd.STATE_VK)
    if as_given:
        q, k = R.normed(q).to(BF16), R.normed(k).to(BF16)
    states = torch.randn(n, 32, 128, 128, generator=gen, device=gpu)
    before = states.mT if by_columns else states.clone()
    before = before.contiguous()
    out = torch.full((sum(lens), 32, 128), 7.0, dtype=BF16, device=gpu)
    rd.ragged_delta_rule(q, k, v, g, beta, states, *batch(lens, slots, has, gpu), out=out, flags=flags)
    want, after = R.delta(q, k, v, g, beta, before, R.cu_of(lens), slots, has, *([torch.Tensor.double] if as_given else []))
    check_delta(out, (states.mT if by_columns else states).contiguous(), want, after, [s for s, m in zip(slots, lens) if not m])


@pytest.mark.parametrize("norm_in_kernel", [True, False])
@pytest.mark.parametrize("initial", [True, False])
def test_vllm_chunk_rule_over_packed_sequences(gpu, norm_in_kernel, initial):
    lens = [70, 1, 200, 9]
    q, k, v, g, beta, gen = core(gpu, sum(lens), 53)
    if not norm_in_kernel:
        q, k = R.normed(q).to(BF16), R.normed(k).to(BF16)
    first = torch.randn(4, 32, 128, 128, generator=gen, device=gpu) if initial else None
    kept = None if first is None else first.clone()
    cu = torch.tensor(R.cu_of(lens), device=gpu)
    out, last = gd.vllm_chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], initial_state=first,
                                               output_final_state=True, cu_seqlens=cu, use_qk_l2norm_in_kernel=norm_in_kernel)
    before = torch.zeros(4, 32, 128, 128, device=gpu) if first is None else first.mT.contiguous()
    want, after = R.delta(q, k, v, g, beta, before, R.cu_of(lens), range(4), [initial] * 4,
                          *([] if norm_in_kernel else [torch.Tensor.double]))
    assert out.shape == (1, sum(lens), 32, 128) and (first is None or torch.equal(first, kept))
    check_delta(out[0], last.mT.contiguous(), want, after, [])
    none = gd.vllm_chunk_gated_delta_rule(q[None], k[None], v[None], g[None], beta[None], initial_state=first,
                                          cu_seqlens=cu, use_qk_l2norm_in_kernel=norm_in_kernel)
    assert none[1] is None and torch.equal(none[0], out)
