"""Turns of a server over both kinds of layers: growing page tables, forks of prompts with
their pages and states, requests with adapters of their own, rows given up and taken again,
compaction, a captured turn; against each request alone, its adapter merged into the weights."""
import copy

import pytest
import torch

from qwen36_attn import adapters as ad
from qwen36_attn import full_attention as fa
from qwen36_attn import gated_deltanet as gd
from qwen36_attn import page_tables as pt
from qwen36_attn import paged_attention as pa
from qwen36_attn import ragged_deltanet as rd
from qwen36_attn import synthetic as syn
from tests.test_paged_use_gpu import layer_weights

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
PAGE, PAGES, WIDTH, ROWS, ADAPTERS, RANK = 16, 24, 8, 4, 3, 16
QKV, MIXED = ("q_proj", "k_proj", "v_proj"), ("in_proj_qkv", "in_proj_z", "in_proj_b", "in_proj_a")


def vector(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def adapters_of(w, names, out, seed, gpu):
    """Adapters of a layer and, for each of them, the weights with it merged in."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    ranks, scales = [16, 5, 9], torch.tensor([0.5, -1.0, 0.8], device=gpu)
    sets, merged = [], [dict(w) for _ in range(ADAPTERS)]
    for group in (names, (out,)):
        widths, k = [w[n].shape[0] for n in group], w[group[0]].shape[1]
        a = (torch.randn(ADAPTERS, len(group), RANK, k, generator=g, device=gpu) * k ** -0.5).to(BF16)
        b = (torch.randn(ADAPTERS, sum(widths), RANK, generator=g, device=gpu) * 0.1).to(BF16)
        sets.append(ad.AdapterSet(a, b, widths, vector(ranks, gpu), scales))
        for i, r in enumerate(ranks):
            for s, (n, m) in enumerate(zip(group, b[i, :, :r].double().split(widths))):
                merged[i][n] = (w[n].double() + scales[i].double() * m @ a[i, s, :r].double()).to(BF16)
    return ad.LayerAdapters(*sets), merged


class Server:
    def __init__(self, gpu):
        self.gpu = gpu
        wf, wl = layer_weights(gpu, 5), {k: v.to(gpu) for k, v in syn.linear_attention_weights(syn.gen(6), a_max=2.0).items()}
        af, self.full = adapters_of(wf, QKV, "o_proj", 7, gpu)
        al, self.linear = adapters_of(wl, MIXED, "out_proj", 8, gpu)
        self.full.append(wf)                                   # adapter -1: none
        self.linear.append(wl)
        conv = torch.full((ROWS, 8192, 3), 3.0, dtype=BF16, device=gpu)
        ssm = torch.full((ROWS, 32, 128, 128), 3.0, device=gpu)
        self.states = [conv, ssm]
        cache = pa.PagedKVCache(PAGES, PAGE, gpu, BF16)
        self.attn = pa.PagedFullAttentionLayer(wf, cache, fa.rotary_table(256, 0, gpu), adapters=af)
        self.delta = rd.RaggedLinearAttentionLayer(wl, conv, ssm, adapters=al)
        self.refs = pt.new_refs(PAGES, gpu)
        self.table = torch.full((ROWS, WIDTH), -1, dtype=torch.int32, device=gpu)
        self.lens = vector([0] * ROWS, gpu)
        self.slots = vector(list(range(ROWS)), gpu)
        self.alone = [None] * ROWS                              # each request by itself

    def turn(self, inp, add, cu, ids, has, longest):
        """What a server runs for a turn: pages, the rows by adapter, both layers."""
        granted = pt.extend(self.refs, self.table, self.lens, add, [self.attn.cache])
        batch = ad.AdapterBatch(cu, ids, inp.shape[0], ADAPTERS)
        return (granted, self.delta.forward(inp, cu, self.slots, has, longest, batch),
                self.attn.forward(inp, self.table, cu, self.lens, batch))

    def begin(self, row, adapter):
        self.alone[row] = [adapter, 0, gd.LinearAttentionLayer(self.linear[adapter], self.gpu),
                           fa.FullAttentionLayer(self.full[adapter], 256, self.gpu)]

    def fork(self, parents):
        p = vector(parents, self.gpu)
        pt.fork(self.refs, self.table, self.lens, p, PAGE)
        rd.fork_states(self.states, p)
        for i, x in enumerate(parents):
            if x >= 0:
                self.alone[i] = self.alone[x][:2] + [copy.copy(layer) for layer in self.alone[x][2:]]
                for layer in self.alone[i][2:]:
                    for name, v in vars(layer).items():
                        if isinstance(v, torch.Tensor):
                            setattr(layer, name, v.clone())

    def check(self, inp, add, got):
        """The layers' chains round to bf16 in the same places but for the adapters: one
        rounding of the merged weights here, one of the sum with what the adapter gives
        there, of at most 2^-8 each, for both projections: 4 beside the 8 that the delta
        layer leaves over a batch.  The attention layer leaves 8 evenly spread ones (2^-8 /
        sqrt 3 each in the norm); the 4, and 4 more where they reach the softmax through q
        and k, whose scores of 256 products over 16 are off by what one product is: 16, and
        twice their independent sum, as a row's share their keys."""
        granted, delta, attn = got
        assert granted.tolist() == [1] * ROWS
        at = 0
        for i, n in enumerate(add):
            if n:
                one = self.alone[i]
                mode, x = "decode" if n == 1 else "prefill", inp[at:at + n].contiguous()
                for y, want, bound in ((delta, one[2].forward(x, mode), 12), (attn, one[3].forward(x, one[1], mode), 2 * (16 / 3) ** 0.5)):
                    rel = ((y[at:at + n].double() - want.double()).norm() / want.double().norm()).item()
                    assert rel <= bound * 2.0 ** -8, (i, n, rel)
                one[1] += n
            at += n

    def rows(self, new, seed):
        return syn.randn((sum(new), 2048), syn.gen(seed)).to(self.gpu)

    def step(self, new, ids, has, seed):
        inp, cu = self.rows(new, seed), [sum(new[:i]) for i in range(ROWS + 1)]
        got = self.turn(inp, vector(new, self.gpu), vector(cu, self.gpu), vector(ids, self.gpu),
                        torch.tensor(has, dtype=torch.bool, device=self.gpu), max(new))
        self.check(inp, new, got)


def served(gpu):
    """A prompt with an adapter, forked twice, and one without; a fork given up, its pages
    and slot for another request."""
    s = Server(gpu)
    s.begin(0, 1)
    s.begin(2, -1)
    s.step([37, 0, 21, 0], [1, 0, -1, 2], [0] * 4, 50)
    s.fork([-1, 0, -1, 0])
    ids = [1, 1, -1, 1]
    for n in range(2):
        s.step([1, 1, 1, 1], ids, [1] * 4, 51 + n)
    pt.trim(s.refs, s.table, s.lens, vector([256, 0, 256, 256], gpu), PAGE)
    pt.compact(s.refs, s.table, s.lens, [s.attn.cache], s.refs, s.table)
    held = int((s.refs > 0).sum())
    assert (s.refs[:held] > 0).all() and held == 2 + 1 + 1 + 2      # two of the prompt, both last ones, row 2's
    s.begin(1, 0)
    s.step([1, 18, 1, 5], [1, 0, -1, 1], [1, 0, 1, 1], 60)
    return s, [1, 0, -1, 1]


def test_turns_of_forked_requests_with_adapters(gpu):
    s, ids = served(gpu)
    for n in range(2):
        s.step([1, 0, 1, 1], ids, [1] * 4, 70 + n)
    s.step([0, 1, 0, 0], ids, [1] * 4, 75)                     # one row in all


def test_captured_turns_of_forked_requests(gpu):
    """The same, then decode turns by a graph, beside eager work and on another stream."""
    s, ids = served(gpu)
    inp = s.rows([1] * 4, 80)
    args = vector([0] * 4, gpu), vector([0, 1, 2, 3, 4], gpu), vector(ids, gpu), torch.ones(4, dtype=torch.bool, device=gpu)
    held = *s.states, s.refs, s.table, s.lens, s.attn.cache.k_pages, s.attn.cache.v_pages
    before = [t.clone() for t in held]
    s.turn(inp, *args, 1)                                      # warm: no row grows; then all as it was
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = s.turn(inp, *args, 1)
    for t, x in zip(held, before):
        t.copy_(x)
    args[0].fill_(1)
    other = torch.cuda.Stream()
    for n in range(3):
        inp.copy_(s.rows([1] * 4, 81 + n))
        torch.cuda.synchronize()
        if n == 1:
            with torch.cuda.stream(other):
                graph.replay()
            other.synchronize()
        else:
            graph.replay()
            torch.cuda.synchronize()
        s.check(inp, [1] * 4, got)
        s.step([1, 1, 0, 1], ids, [1] * 4, 90 + n)


def test_refusals(gpu):
    w = layer_weights(gpu, 5)
    cache, rope = pa.PagedKVCache(4, PAGE, gpu, BF16), fa.rotary_table(64, 0, gpu)

    def made(widths, k, n=2):
        return ad.AdapterSet(torch.zeros(n, len(widths), 8, k, dtype=BF16, device=gpu),
                             torch.zeros(n, sum(widths), 8, dtype=BF16, device=gpu), widths)
    qkv, out = made([8192, 512, 512], 2048), made([2048], 4096)
    for into, o in ((None, None), (qkv, made([2048], 4096, 3))):
        with pytest.raises(ValueError, match="as many of each"):
            ad.LayerAdapters(into, o)
    for bad in (ad.LayerAdapters(made([9216], 2048), out), ad.LayerAdapters(qkv, made([2048], 2048)),
                ad.LayerAdapters(None, qkv)):
        with pytest.raises(ValueError, match="adapters of slices"):
            pa.PagedFullAttentionLayer(w, cache, rope, adapters=bad)
    layer = pa.PagedFullAttentionLayer(w, cache, rope, adapters=ad.LayerAdapters(qkv, out))
    x, where = torch.zeros(2, 2048, dtype=BF16, device=gpu), [vector(v, gpu) for v in ([[0]], [0, 2], [2])]
    for batch, match in ((ad.AdapterBatch(where[1], vector([0], gpu), 3, 2), "must be bf16"),
                         (ad.AdapterBatch(where[1], vector([0], gpu), 2, 3), "other adapters")):
        with pytest.raises(ValueError, match=match):
            layer.forward(x, *where, adapter_batch=batch)
