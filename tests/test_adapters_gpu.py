"""Low-rank adapters beside a shared projection against the same in 64 bits: every
rank and slice, requests without an adapter, tiles of both sizes, strides, what stands
behind a rank, captured calls, the layers."""
import pytest
import torch

from qwen36_attn import adapters as ad
from tests import ragged_reference as R

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
QKV, MIXED, ODD = (2048, (8192, 512, 512)), (2048, (8192, 4096, 32, 32)), (128, (8, 264, 72))


def vector(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def make(gpu, proj, n, rank, ranks, seed, behind=float("nan")):
    """Adapters whose matrices hold `behind` where they are not used."""
    k, widths = proj
    g = torch.Generator(device=gpu).manual_seed(seed)
    a = (torch.randn(n, len(widths), rank, k, generator=g, device=gpu) * k ** -0.5).to(BF16)
    b = (torch.randn(n, sum(widths), rank, generator=g, device=gpu) * 0.2).to(BF16)
    for i, r in enumerate(ranks):
        a[i, :, r:] = behind
        b[i, :, r:] = behind
    scales = torch.rand(n, generator=g, device=gpu) * 2 - 0.5
    return a, b, scales, ad.AdapterSet(a, b, widths, vector(ranks, gpu), scales), g


def expected(y, x, a, b, scales, ranks, widths, lens, ids):
    """The rows in 64 bits, and a bound of what fp32 sums (of k and of rank products) and
    a factor kept to 2^-17 leave, before the rounding to bf16."""
    want, slack, at = y.double(), torch.zeros_like(y, dtype=torch.float64), 0
    for n, i in zip(lens, ids):
        if 0 <= i < len(ranks):
            r, c = ranks[i], 0
            for s, width in enumerate(widths):
                u, d, s0 = x[at:at + n].double(), a[i, s, :r].double(), scales[i].double()
                up = b[i, c:c + width, :r].double()
                want[at:at + n, c:c + width] += s0 * (u @ d.T) @ up.T
                slack[at:at + n, c:c + width] = s0.abs() * ((u.abs() @ d.abs().T) @ up.abs().T) \
                    * (2.0 ** -17 + (x.shape[1] + 2 * r + 8) * 2.0 ** -24)
                c += width
        at += n
    return want, slack


CASES = [(QKV, 1, 16, [16], [1], [0]), (QKV, 3, 16, [16, 8, 1], [1, 1, 1, 1, 1], [2, 0, -1, 1, 0]),
         (MIXED, 5, 32, [32, 0, 7, 24, 9], [1] * 37, [(i * 3) % 7 - 1 for i in range(37)]),
         (ODD, 4, 24, [24, 5, 17, 8], [3, 0, 40, 1, 17, 33], [1, 0, 3, 9, 2, 3]),
         (ODD, 2, 8, [8, 3], [500, 524], [1, 0]), (ODD, 2, 8, [8, 3], [501, 524], [1, 0]),
         (QKV, 2, 64, [64, 33], [700, 1, 640], [1, 0, 0]), ((4096, (2048,)), 3, 128, [128, 100, 64], [1200, 5, 77], [0, 2, 1]),
         ((256, (64,)), 300, 8, [1 + i % 8 for i in range(300)], [1 + i % 3 for i in range(700)], [(i * 7) % 301 for i in range(700)]),
         ((16384, (24, 16)), 2, 40, [40, 31], [9, 1], [0, 1])]


@pytest.mark.parametrize("proj,n,rank,ranks,lens,ids", CASES)
def test_rows(gpu, proj, n, rank, ranks, lens, ids):
    k, widths = proj
    t, total = sum(lens) + 3, sum(widths)
    a, b, scales, adapters, g = make(gpu, proj, n, rank, ranks, t)
    x = torch.randn(t, k + 8, generator=g, device=gpu).to(BF16)[:, :k]
    wide = torch.randn(t, total + 16, generator=g, device=gpu).to(BF16)
    before = wide.clone()
    y = wide[:, 8:8 + total]
    print("adapters", proj, ranks[:6], lens[:6], flush=True)
    batch = ad.AdapterBatch(vector(R.cu_of(lens), gpu), vector(ids, gpu), t, n)
    assert ad.apply_adapters(y, x, adapters, batch) is y
    want, slack = expected(before[:, 8:8 + total], x, a, b, scales, ranks, widths, lens, ids)
    err = (y.double() - want).abs()
    tol = 2.0 ** -8 * (want.abs() + slack) + slack
    assert (err <= tol).all(), (err - tol).max().item()
    assert torch.equal(wide[:, :8], before[:, :8]) and torch.equal(wide[:, 8 + total:], before[:, 8 + total:])
    at = 0
    for m, i in zip(lens + [3], ids + [-1]):
        if not 0 <= i < n or ranks[i] == 0:
            assert torch.equal(y[at:at + m], before[at:at + m, 8:8 + total])
        at += m


def test_rows_far_apart(gpu):
    """Rows of x that reach behind 2^31 bytes, in tiles of 64: other loads than where they
    do not, the same sums to their rounding."""
    lens, ids, t = [600, 1, 500], [0, 1, 1], 1101
    a, b, scales, adapters, g = make(gpu, QKV, 2, 64, [64, 17], 4)
    x, y = (torch.randn(t, n, generator=g, device=gpu).to(BF16) for n in (2048, 9216))
    far = torch.empty(t * (1 << 20), dtype=BF16, device=gpu).view(t, 1 << 20)[:, :2048]
    far.copy_(x)
    batch = ad.AdapterBatch(vector(R.cu_of(lens), gpu), vector(ids, gpu), t, 2)
    want, slack = expected(y, x, a, b, scales, [64, 17], QKV[1], lens, ids)
    for rows in (x, far):
        got = ad.apply_adapters(y.clone(), rows, adapters, batch).double()
        assert ((got - want).abs() <= 2.0 ** -8 * (want.abs() + slack) + slack).all()


def test_no_ranks_and_no_scales(gpu):
    a, b, _, _, g = make(gpu, ODD, 2, 16, [16, 16], 5)
    x, y = (torch.randn(30, n, generator=g, device=gpu).to(BF16) for n in (128, 344))
    before = y.clone()
    lens, ids = [10, 20], [1, 0]
    ad.apply_adapters(y, x, ad.AdapterSet(a, b, ODD[1]), ad.AdapterBatch(vector(R.cu_of(lens), gpu), vector(ids, gpu), 30, 2))
    want, slack = expected(before, x, a, b, torch.ones(2, device=gpu), [16, 16], ODD[1], lens, ids)
    assert ((y.double() - want).abs() <= 2.0 ** -8 * (want.abs() + slack) + slack).all()


def test_requests_in_any_order(gpu):
    """The same requests in another order: the same bits for each; NaN in one request's rows
    stays there."""
    a, b, scales, adapters, g = make(gpu, QKV, 3, 32, [32, 20, 16], 8)
    lens, ids = [1, 4, 1, 30, 2, 1, 17], [0, 1, 2, 0, 1, -1, 0]
    x = [torch.randn(n, 2048, generator=g, device=gpu).to(BF16) for n in lens]
    y = [torch.randn(n, 9216, generator=g, device=gpu).to(BF16) for n in lens]
    got = []
    for order in (list(range(7)), [6, 3, 0, 5, 1, 4, 2]):
        xx = torch.cat([x[i] for i in order])
        if order[0]:
            at = sum(lens[i] for i in order[:2])        # request 0's only row
            xx[at] = float("nan")
        yy = torch.cat([y[i] for i in order])
        batch = ad.AdapterBatch(vector(R.cu_of([lens[i] for i in order]), gpu), vector([ids[i] for i in order], gpu), 56, 3)
        ad.apply_adapters(yy, xx, adapters, batch)
        parts = yy.split([lens[i] for i in order])
        got.append({i: p for i, p in zip(order, parts)})
    for i in range(1, 7):
        assert torch.equal(got[0][i], got[1][i]), i
    assert got[1][0].isnan().all()


def test_offsets_that_make_no_sense(gpu):
    """Offsets behind the rows, falling and overlapping: rows of no sequence stay, the call
    ends, and what is behind the tensors stays."""
    a, b, scales, adapters, g = make(gpu, ODD, 3, 16, [16, 8, 4], 2)
    for cu, rows in (([0, 900, -5, 30, 50], range(0, 50)), ([40, 20, 10, 5, 2 ** 31 - 1], range(5, 50)), ([60, 70, 80, 90, 99], range(0))):
        x = torch.randn(50, 128, generator=g, device=gpu).to(BF16)
        wide = torch.randn(60, 344, generator=g, device=gpu).to(BF16)
        before = wide.clone()
        batch = ad.AdapterBatch(vector(cu, gpu), vector([0, 1, 2, 0], gpu), 50, 3)
        ad.apply_adapters(wide[:50], x, adapters, batch)
        same = (wide == before).all(1).tolist()
        assert all(same[i] for i in range(60) if i not in rows)


def test_captured_calls_follow_the_requests(gpu):
    a, b, scales, adapters, g = make(gpu, MIXED, 4, 16, [16, 8, 12, 3], 6)
    x, y = (torch.randn(20, n, generator=g, device=gpu).to(BF16) for n in (2048, sum(MIXED[1])))
    before = y.clone()
    cu, ids = vector([0, 5, 6, 20], gpu), vector([0, 1, 2], gpu)

    def step():
        return ad.apply_adapters(y, x, adapters, ad.AdapterBatch(cu, ids, 20, 4))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for c, i in (([0, 5, 6, 20], [0, 1, 2]), ([0, 0, 19, 20], [3, -1, 0]), ([0, 1, 2, 3], [7, 2, 2]), ([0, 20, 20, 20], [1, 1, 1])):
        y.copy_(before)
        cu.copy_(vector(c, gpu))
        ids.copy_(vector(i, gpu))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone()
        y.copy_(before)
        assert torch.equal(step(), got), c


def test_on_another_stream(gpu):
    a, b, scales, adapters, g = make(gpu, QKV, 2, 16, [16, 16], 1)
    x, y = (torch.randn(70, n, generator=g, device=gpu).to(BF16) for n in (2048, 9216))
    cu, ids, other = vector([0, 30, 70], gpu), vector([1, 0], gpu), y.clone()
    ad.apply_adapters(y, x, adapters, ad.AdapterBatch(cu, ids, 70, 2))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ad.apply_adapters(other, x, adapters, ad.AdapterBatch(cu, ids, 70, 2))
    s.synchronize()
    assert torch.equal(other, y)


def test_refusals(gpu):
    a, b, scales, adapters, g = make(gpu, ODD, 2, 16, [16, 8], 1)
    x, y = (torch.zeros(6, n, dtype=BF16, device=gpu) for n in (128, 344))
    cu, ids = vector([0, 6], gpu), vector([0], gpu)
    batch = ad.AdapterBatch(cu, ids, 6, 2)
    for bad in (lambda: ad.AdapterSet(a, b, (8, 264)), lambda: ad.AdapterSet(a, b, (8, 264, 70)),
                lambda: ad.AdapterSet(a.float(), b, ODD[1]), lambda: ad.AdapterSet(a[..., :120], b, ODD[1]),
                lambda: ad.AdapterSet(a[:, :, :12].contiguous(), b[:, :, :12].contiguous(), ODD[1]),
                lambda: ad.AdapterSet(a, b, ODD[1], scales), lambda: ad.AdapterSet(a, b, ODD[1], None, scales[:1]),
                lambda: ad.AdapterBatch(cu.long(), ids, 6, 2), lambda: ad.AdapterBatch(cu, cu, 6, 2),
                lambda: ad.AdapterBatch(cu, ids, 0, 2), lambda: ad.AdapterBatch(cu, ids, 6, 4097),
                lambda: ad.AdapterBatch(cu.cpu(), ids, 6, 2),
                lambda: ad.apply_adapters(y, x, adapters, ad.AdapterBatch(cu, ids, 6, 3)),
                lambda: ad.apply_adapters(y[:5], x, adapters, batch), lambda: ad.apply_adapters(y, x[:, :120], adapters, batch),
                lambda: ad.apply_adapters(y, x.float(), adapters, batch),
                lambda: ad.apply_adapters(torch.zeros(6, 347, dtype=BF16, device=gpu)[:, :344], x, adapters, batch)):
        with pytest.raises(ValueError):
            bad()
