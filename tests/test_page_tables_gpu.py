"""Trimming, forking, growing and compacting rows of a page table against the same by
hand: counts, tables, lengths and every byte of the pages equal."""
import random

import pytest
import torch

from qwen36_attn import page_tables as pt
from qwen36_attn import paged_attention as pa
from qwen36_attn import ragged_deltanet as rd
from tests.page_reference import Tables

pytestmark = pytest.mark.gpu
FP8, BF16 = torch.float8_e4m3fn, torch.bfloat16
NAMES = ("k_pages", "v_pages", "k_exp", "v_exp", "bounds")


def a_cache(pages, page, gpu, dtype, heads, bounds, seed, apart=False):
    g = torch.Generator(device=gpu).manual_seed(seed)

    def of(*shape, kind=torch.uint8):
        x = torch.randint(0, 256, shape, generator=g, device=gpu, dtype=torch.uint8)
        return x.view(kind)
    size = 1 if dtype == FP8 else 2
    shape = (pages, 2, heads, page, 256 * size) if apart else (2, pages, heads, page, 256 * size)
    kv = of(*shape).view(dtype)
    k, v = (kv[:, 0], kv[:, 1]) if apart else (kv[0], kv[1])
    exp = dtype == FP8 or bounds
    return pa.PagedKVCache.of(k, v, of(pages, heads) if exp else None, of(pages, heads) if dtype == FP8 else None,
                              of(pages, heads, 2, 256, kind=torch.int8) if bounds else None)


def raw(cache):
    return {n: getattr(cache, n).clone().contiguous().view(torch.uint8) for n in NAMES if getattr(cache, n) is not None}


class Both:
    """The tables on the GPU and by hand, and the caches' bytes."""

    def __init__(self, rows, width, pages, page, caches, gpu):
        self.refs = pt.new_refs(pages, gpu)
        self.table = torch.full((rows, width + 3), -1, dtype=torch.int32, device=gpu)[:, :width]
        self.lens = torch.zeros(rows, dtype=torch.int32, device=gpu)
        self.hand = Tables(self.refs.tolist(), self.table.tolist(), self.lens.tolist(), page)
        self.caches, self.page, self.gpu = caches, page, gpu
        self.bytes = [raw(c) for c in caches]

    def vector(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.gpu)

    def trim(self, keep):
        pt.trim(self.refs, self.table, self.lens, self.vector(keep), self.page)
        self.hand.trim(keep)
        self.check()

    def fork(self, parents):
        pt.fork(self.refs, self.table, self.lens, self.vector(parents), self.page)
        self.hand.fork(parents)
        self.check()

    def moved(self, copies):
        for b in self.bytes:
            for x in b.values():
                old = x.clone()
                for s, d in copies:
                    x[d] = old[s]

    def extend(self, add):
        got = pt.extend(self.refs, self.table, self.lens, self.vector(add), self.caches)
        granted, copies = self.hand.extend(add)
        assert got.tolist() == granted
        self.moved(copies)
        self.check()
        return granted, copies

    def compact(self, place):
        out = (None, None) if not place else (self.refs, self.table)
        refs, table = pt.compact(self.refs, self.table, self.lens, self.caches, *out)
        moves = self.hand.compact()
        self.refs.copy_(refs)
        self.table.copy_(table)
        self.moved(moves)
        self.check()
        return moves

    def check(self):
        assert self.refs.tolist() == self.hand.refs
        assert self.table.tolist() == self.hand.table
        assert self.lens.tolist() == self.hand.lens
        for c, b in zip(self.caches, self.bytes):
            for n, x in raw(c).items():
                assert torch.equal(x, b[n]), n


@pytest.mark.parametrize("seed,page,kinds", [
    (1, 16, [(FP8, 2, False, False)]), (2, 32, [(FP8, 2, True, False), (BF16, 1, False, True)]),
    (3, 64, [(BF16, 3, True, False), (FP8, 16, False, True)]), (4, 128, [(FP8, 1, True, True)]),
    (5, 16, [(FP8, 2, False, i % 2 == 0) for i in range(18)])])
def test_turns_by_hand(gpu, seed, page, kinds):
    """Random turns over a pool that runs out at times (three of the five)."""
    rng = random.Random(seed)
    rows, width, pages = 9, 7, 23
    b = Both(rows, width, pages, page, [a_cache(pages, page, gpu, d, h, bo, seed * 50 + i, apart)
                                        for i, (d, h, bo, apart) in enumerate(kinds)], gpu)
    copied = moved = 0
    for turn in range(40):
        b.trim([rng.choice([1 << 30, 1 << 30, 0, -5, rng.randint(0, width * page)]) for _ in range(rows)])
        b.fork([rng.choice([-1, -1, rng.randint(-1, rows + 1)]) for _ in range(rows)])
        _, copies = b.extend([rng.choice([0, 1, 1, -3, rng.randint(1, 3 * page), page]) for _ in range(rows)])
        copied += len(copies)
        if turn % 5 == 4:
            moved += len(b.compact(turn % 10 == 9))
    assert copied and moved
    b.trim([0] * rows)
    assert b.refs.tolist() == [0] * pages


def test_children_of_children_stay_empty(gpu):
    b = Both(5, 4, 10, 16, [a_cache(10, 16, gpu, FP8, 2, False, 7)], gpu)
    b.extend([20, 0, 0, 33, 0])
    b.fork([-1, 0, 1, 0, 4])         # 2 forks a child, 3 is not empty, 4 names itself
    assert b.lens.tolist() == [20, 20, 0, 33, 0]
    # both hold the half-full page: each that grows gets a copy of its own
    b.extend([1, 1, 0, 0, 0])
    assert b.refs.tolist()[:2] == [2, 0]


def test_numbers_out_of_range(gpu):
    """Lengths that are none, page ids outside the pool, in rows and tables."""
    b = Both(6, 3, 8, 16, [a_cache(8, 16, gpu, FP8, 2, False, 8)], gpu)
    b.extend([16, 17, 5, 48, 0, 2])
    b.table[1, 1] = 99
    b.lens[2], b.lens[3] = -7, 49
    b.table[5, 0] = -2
    b.hand.table[1][1], b.hand.table[5][0] = 99, -2
    b.hand.lens[2], b.hand.lens[3] = -7, 49
    b.fork([2, -1, -1, -1, 1, -1])
    b.extend([1, 1, 1, 1, 1, 2])
    b.extend([0, 100, 0, 0, 2 ** 31 - 1, 0])
    b.trim([3, 0, 0, 0, 1, 1])
    b.compact(True)


@pytest.mark.parametrize("pages,rows", [(16384, 3), (16385, 5000), (50001, 70)])
def test_large_pools(gpu, pages, rows):
    """Pools of more than one step of the scan, more rows than one pass takes; free pages
    far behind.  Small pages (one head of 16 tokens, bf16 exponents absent)."""
    g = torch.Generator(device=gpu).manual_seed(pages)
    k = torch.randint(0, 120, (pages, 1, 16, 256), generator=g, device=gpu, dtype=torch.uint8).view(FP8)
    e = torch.randint(90, 140, (pages, 1), generator=g, device=gpu, dtype=torch.uint8)
    cache = pa.PagedKVCache.of(k, k.clone(), e, e.clone())
    b = Both(rows, 4, pages, 16, [], gpu)
    b.caches, b.bytes = [cache], [raw(cache)]
    rng = random.Random(pages)
    held = [1 if rng.random() < 0.9 else 0 for _ in range(pages - 100)] + [1] * 99 + [0]
    b.refs.copy_(b.vector(held))
    b.hand.refs = list(held)
    b.extend([rng.choice([1, 17, 40]) for _ in range(rows)])
    b.fork([-1] * (rows - 1) + [0])
    b.trim([rng.choice([0, 5, 1 << 30]) for _ in range(rows)])
    b.fork([rng.randint(-3, rows - 1) if rng.random() < 0.3 else -1 for _ in range(rows)])
    b.extend([1] * rows)
    b.compact(False)


def test_captured_turns(gpu):
    """One captured turn, replayed over other numbers, against the same by hand."""
    b = Both(4, 5, 16, 16, [a_cache(16, 16, gpu, FP8, 2, True, 3)], gpu)
    keep, parents, add = b.vector([99] * 4), b.vector([-1] * 4), b.vector([0] * 4)

    def turn():
        pt.trim(b.refs, b.table, b.lens, keep, 16)
        pt.fork(b.refs, b.table, b.lens, parents, 16)
        got = pt.extend(b.refs, b.table, b.lens, add, b.caches)
        pt.compact(b.refs, b.table, b.lens, b.caches, b.refs, b.table)
        return got
    turn()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = turn()
    for k, p, a in (([99] * 4, [-1] * 4, [40, 0, 3, 0]), ([99] * 4, [-1, 0, -1, 0], [1, 1, 1, 1]),
                    ([0, 99, 20, 99], [-1, -1, -1, -1], [0, 40, 0, 1]), ([99, 0, 99, 7], [2, -1, -1, -1], [90, 1, 1, 20])):
        for x, y in ((keep, k), (parents, p), (add, a)):
            x.copy_(b.vector(y))
        graph.replay()
        torch.cuda.synchronize()
        b.hand.trim(k)
        b.hand.fork(p)
        granted, copies = b.hand.extend(a)
        assert got.tolist() == granted
        b.moved(copies)
        b.moved(b.hand.compact())
        b.check()


def test_fork_states(gpu):
    g = torch.Generator(device=gpu).manual_seed(2)
    conv = torch.randn(6, 2, 8192, 3, generator=g, device=gpu).to(BF16)
    ssm = [torch.randn(6, 32, 128, 128, generator=g, device=gpu) for _ in range(2)]
    odd = torch.randint(0, 256, (6, 48), generator=g, device=gpu, dtype=torch.uint8)
    before = [x.clone() for x in (conv, *ssm, odd)]
    rd.fork_states([conv[:, 1], *ssm, odd], torch.tensor([-1, 0, 1, 5, 9, -4], dtype=torch.int32, device=gpu))
    at = torch.tensor([0, 0, 2, 5, 4, 5], device=gpu)       # 2 forks a child, 9 is no slot
    assert torch.equal(conv[:, 0], before[0][:, 0]) and torch.equal(conv[:, 1], before[0][:, 1][at])
    for x, y in zip((*ssm, odd), before[1:]):
        assert torch.equal(x, y[at])


def test_forked_rows_attend_alike(gpu):
    """A prompt forked three ways and continued with tokens of each: every row's attention
    is that of a row that got the prompt and its tokens alone."""
    from qwen36_attn import full_attention as fa
    from tests.test_paged_use_gpu import layer_weights
    w, rope, page = layer_weights(gpu, 3), fa.rotary_table(256, 0, gpu), 16
    g = torch.Generator(device=gpu).manual_seed(6)
    prompt = torch.randn(37, 2048, generator=g, device=gpu).to(BF16)
    more = torch.randn(4, 3, 2048, generator=g, device=gpu).to(BF16)

    def layer():
        return pa.PagedFullAttentionLayer(w, pa.PagedKVCache(24, page, gpu, BF16), rope)

    def vector(x):
        return torch.tensor(x, dtype=torch.int32, device=gpu)

    def start(rows):
        return pt.new_refs(24, gpu), torch.full((rows, 6), -1, dtype=torch.int32, device=gpu), vector([0] * rows)
    shared, (refs, table, lens) = layer(), start(4)
    assert pt.extend(refs, table, lens, vector([37, 0, 0, 0]), [shared.cache]).tolist() == [1] * 4
    shared.forward(prompt, table, vector([0, 37, 37, 37, 37]), lens)
    pt.fork(refs, table, lens, vector([-1, 0, 0, 0]), page)
    got = []
    for step in range(3):
        assert pt.extend(refs, table, lens, vector([1] * 4), [shared.cache]).tolist() == [1] * 4
        got.append(shared.forward(more[:, step].contiguous(), table, vector([0, 1, 2, 3, 4]), lens))
    assert sorted(refs.tolist())[-3:] == [1, 4, 4]          # two full pages of the prompt stay shared
    for i in range(4):
        alone, (refs1, table1, lens1) = layer(), start(4)
        pt.extend(refs1, table1, lens1, vector([37, 0, 0, 0]), [alone.cache])
        alone.forward(prompt, table1, vector([0, 37, 37, 37, 37]), lens1)
        for step in range(3):
            pt.extend(refs1, table1, lens1, vector([1, 0, 0, 0]), [alone.cache])
            rows = torch.stack([more[i, step]] * 4)         # as many rows, so that the products are the same
            one = alone.forward(rows, table1, vector([0, 1, 1, 1, 1]), lens1)[0]
            # the split of the keys differs with the batch: the P values' bf16 rounding and the output's
            rel = ((got[step][i].double() - one.double()).norm() / one.double().norm()).item()
            assert rel <= 2 * 2.0 ** -8, (i, step, rel)
