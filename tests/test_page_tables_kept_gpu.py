"""Compaction of a table with rows whose length is none: they keep their pages, wherever
these go."""
import pytest
import torch

from qwen36_attn import page_tables as pt
from tests.page_reference import Tables
from tests.test_page_tables_gpu import BF16, FP8, Both, a_cache

pytestmark = pytest.mark.gpu


class Kept(Tables):
    """Entries of a row of no valid length follow their pages as its others do; those that
    name no page stay."""

    def compact(self):
        rows = [list(r) for r in self.table]
        moves = super().compact()
        to = dict(moves)
        for i, row in enumerate(rows):
            if not self.valid(i):
                self.table[i] = [to.get(x, x) for x in row]
        return moves


def tables(rows, width, pages, page, gpu, kinds):
    b = Both(rows, width, pages, page, [a_cache(pages, page, gpu, d, h, bo, 70 + i) for i, (d, h, bo) in enumerate(kinds)], gpu)
    b.hand = Kept(b.refs.tolist(), b.table.tolist(), b.lens.tolist(), page)
    return b


def length(b, row, n):
    b.lens[row] = n
    b.hand.lens[row] = n


@pytest.mark.parametrize("place", [True, False])
@pytest.mark.parametrize("n", [-7, -(1 << 31), 81, 1 << 20])
def test_rows_of_no_length_keep_their_pages(gpu, place, n):
    """Their pages move, the counts go with them, and the row goes on once its length is
    put right: nothing of the pool is lost."""
    b = tables(5, 5, 24, 16, gpu, [(FP8, 2, False), (BF16, 1, True)])
    b.extend([40, 70, 33, 20, 16])
    b.fork([-1] * 5)
    b.trim([0, 99, 99, 0, 99])
    b.extend([5, 0, 0, 0, 0])
    b.trim([0, 99, 99, 0, 99])
    lens = list(b.hand.lens)
    length(b, 2, n)
    length(b, 4, n)
    held = [b.hand.table[i][:-(-lens[i] // 16)] for i in (2, 4)]
    moves = b.compact(place)
    to = dict(moves)
    assert all(any(x in to for x in row) for row in held)
    assert [b.table[i].tolist()[:len(row)] for i, row in zip((2, 4), held)] == [[to.get(x, x) for x in row] for row in held]
    for i in (2, 4):
        length(b, i, lens[i])
    b.extend([0, 0, 3, 0, 20])
    b.compact(place)
    b.trim([0] * 5)
    assert b.refs.tolist() == [0] * 24


def test_numbers_out_of_range(gpu):
    """Lengths that are none and page ids outside the pool, through every call."""
    b = tables(6, 3, 9, 16, gpu, [(FP8, 2, False)])
    b.extend([16, 17, 5, 48, 0, 2])
    b.table[1, 1] = 99
    b.table[5, 0] = -2
    b.table[2, 1], b.table[2, 2] = 1 << 30, -(1 << 31)
    b.hand.table[1][1], b.hand.table[5][0], b.hand.table[2][1:] = 99, -2, [1 << 30, -(1 << 31)]
    length(b, 2, -7)
    length(b, 3, 49)
    b.fork([2, -1, -1, -1, 1, -1])
    b.extend([1, 1, 1, 1, 1, 2])
    b.extend([0, 100, 0, 0, 2 ** 31 - 1, 0])
    b.trim([0, 0, 0, 0, 1, 1])
    assert b.compact(True)
    assert b.table[2].tolist()[1:] == [1 << 30, -(1 << 31)]
    assert [x for x in b.table[3].tolist()] == b.hand.table[3] and min(b.hand.table[3]) >= 0


def test_captured_compaction_keeps_them(gpu):
    b = tables(4, 5, 16, 16, gpu, [(FP8, 2, True)])
    keep, add = b.vector([99] * 4), b.vector([0] * 4)

    def turn():
        pt.trim(b.refs, b.table, b.lens, keep, 16)
        pt.extend(b.refs, b.table, b.lens, add, b.caches)
        pt.compact(b.refs, b.table, b.lens, b.caches, b.refs, b.table)
    turn()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turn()
    for k, a, lost in (([99] * 4, [40, 20, 3, 33], None), ([0, 99, 99, 99], [0, 0, 0, 1], 1), ([99, 99, 0, 99], [20, 1, 5, 0], 3)):
        if lost is not None:
            length(b, lost, -1)
        for x, y in ((keep, k), (add, a)):
            x.copy_(b.vector(y))
        graph.replay()
        torch.cuda.synchronize()
        b.hand.trim(k)
        b.moved(b.hand.extend(a)[1])
        b.moved(b.hand.compact())
        b.check()
