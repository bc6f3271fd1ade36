"""Plain forms of the paged-cache operators on the CPU, in 64 bits and whole
numbers, and the batches that their tests use."""
import math

import torch

D, GROUP = 256, 8


class Batch:
    """Sequences of lengths ``lens`` whose last ``new`` tokens are the call's
    rows, their pages dealt over a pool in random order."""

    def __init__(self, lens, new, page, seed=0, spare=3, rows_behind=0, room=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.page = list(lens), list(new), page
        need = [max(1, -(-(x + room) // page)) for x in lens]
        self.width = max(need)
        self.pool = sum(need) + spare
        order = torch.randperm(self.pool, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.cu = torch.tensor([0] + self.new).cumsum(0).to(torch.int32)
        self.tokens = int(self.cu[-1]) + rows_behind

    def where(self, dev):
        return (self.table.to(dev), self.cu.to(dev),
                torch.tensor(self.lens, dtype=torch.int32, device=dev))

    def rows(self):
        """(row, sequence, position) of every row of a sequence."""
        for i, n in enumerate(self.new):
            for j in range(n):
                yield int(self.cu[i]) + j, i, self.lens[i] - n + j


def least_byte(amax: float) -> int:
    """Least e >= 16 with amax <= 448 * 2^(e - 127)."""
    if amax == 0:
        return 16
    m, x = math.frexp(amax)
    return max(16, x + 118 + (m > 0.875))


def to_e4m3(x):
    """bf16/fp64 values to e4m3 bits, nearest even; what is not finite is a NaN."""
    b = x.float().to(torch.float8_e4m3fn).view(torch.uint8)
    return torch.where(torch.isfinite(x), b, torch.full_like(b, 0x7F))


def from_e4m3(b):
    return b.view(torch.float8_e4m3fn).double()


def same_e4m3(a, b):
    """Equal bits, any NaN being one."""
    nan = ((a & 0x7F) == 0x7F) & ((b & 0x7F) == 0x7F)
    return bool(((a == b) | nan).all())


class CacheState:
    """A cache's tensors on the CPU: e4m3 pages as bytes, bf16 pages as bf16."""

    def __init__(self, cache):
        fp8 = cache.k_pages.dtype == torch.float8_e4m3fn
        self.fp8 = fp8
        self.k, self.v = (p.cpu().view(torch.uint8) if fp8 else p.cpu() for p in (cache.k_pages, cache.v_pages))
        self.k, self.v = self.k.clone(), self.v.clone()
        self.ke = None if cache.k_exp is None else cache.k_exp.cpu().clone()
        self.ve = None if cache.v_exp is None else cache.v_exp.cpu().clone()
        self.bounds = None if cache.bounds is None else cache.bounds.cpu().clone()

    def append(self, b: Batch, k, v):
        """k, v [T, kv_heads, 256] bf16: the normed and rotated keys, raw values."""
        heads = k.shape[1]
        for i, n in enumerate(b.new):
            if n == 0 or b.lens[i] == 0 or b.lens[i] > b.width * b.page:
                continue
            p0, end = max(0, b.lens[i] - n), b.lens[i]
            for p in range(p0 // b.page, (end - 1) // b.page + 1):
                pid = int(b.table[i, p])
                if not 0 <= pid < self.k.shape[0]:
                    continue
                lo, hi = max(p0, p * b.page), min(end, (p + 1) * b.page)
                r0, r1 = lo - p * b.page, hi - p * b.page
                row = int(b.cu[i]) + n - (end - lo)
                for h in range(heads):
                    self._page(pid, h, r0, r1, k[row:row + hi - lo, h], v[row:row + hi - lo, h])

    def _page(self, pid, h, r0, r1, k, v):
        for name, pages, exps, x in (("k", self.k, self.ke, k), ("v", self.v, self.ve, v)):
            if exps is None:
                pages[pid, h, r0:r1] = x
                continue
            fin = x[torch.isfinite(x)].double()
            e = least_byte(fin.abs().max().item() if fin.numel() else 0.0)
            old = int(exps[pid, h])
            if r0 > 0:
                e = max(e, old)
            exps[pid, h] = e
            if name == "k" and self.bounds is not None:
                step = 4.0 * 2.0 ** (e - 127)
                z = torch.nan_to_num(x.double(), nan=0.0, posinf=math.inf, neginf=-math.inf)
                top = torch.ceil(z.amax(0) / step).clamp(-127, 127)
                low = torch.floor(z.amin(0) / step).clamp(-127, 127)
                if r0 > 0:
                    was = self.bounds[pid, h].double() * 2.0 ** (old - e)
                    top, low = torch.maximum(top, was[0].ceil()), torch.minimum(low, was[1].floor())
                self.bounds[pid, h] = torch.stack((top, low)).to(torch.int8)
            if not self.fp8:
                pages[pid, h, r0:r1] = x
                continue
            if r0 > 0 and e > old:
                kept = from_e4m3(pages[pid, h, :r0]) * 2.0 ** (old - e)
                pages[pid, h, :r0] = to_e4m3(kept)
            pages[pid, h, r0:r1] = to_e4m3(x.double() * 2.0 ** (127 - e))

    def same(self, cache):
        o = CacheState(cache)
        for name in ("ke", "ve", "bounds"):
            a, b = getattr(self, name), getattr(o, name)
            assert (a is None) == (b is None)
            if a is not None:
                assert torch.equal(a, b), name
        for name in ("k", "v"):
            a, b = getattr(self, name), getattr(o, name)
            if self.fp8:
                assert same_e4m3(a, b), name
            else:
                assert torch.equal(a.view(torch.int16), b.view(torch.int16)), name

    def page_values(self, pid, h):
        """K and V of a page and head, [page, 256] in 64 bits."""
        if not self.fp8:
            return self.k[pid, h].double(), self.v[pid, h].double()
        return (from_e4m3(self.k[pid, h]) * 2.0 ** (int(self.ke[pid, h]) - 127),
                from_e4m3(self.v[pid, h]) * 2.0 ** (int(self.ve[pid, h]) - 127))


def attend_row(state, b, q, i, h, pos, pages):
    """One row's 8 heads over the positions <= pos of the listed pages of
    sequence i: (output, bound of the error of a kernel that sums in fp32, rounds
    P to bf16 and the output to bf16)."""
    ks, vs = [], []
    for p in pages:
        pid = int(b.table[i, p])
        if not 0 <= pid < state.k.shape[0]:
            continue
        k, v = state.page_values(pid, h)
        n = min(b.page, pos + 1 - p * b.page)
        if n > 0:
            ks.append(k[:n])
            vs.append(v[:n])
    if not ks:
        return torch.zeros(GROUP, D, dtype=torch.float64), torch.zeros(GROUP, D, dtype=torch.float64)
    k, v = torch.cat(ks), torch.cat(vs)
    q = q.double()
    p = torch.softmax(q @ k.t() / 16, -1)
    o = p @ v
    # fp32 scores: 256 products and sums of 2^-24 each, once in p and once in its sum;
    # exp2, its argument and the fp32 sums of n keys; P rounded to bf16 (2^-8)
    score = (q.abs() @ k.abs().t()).amax(-1, keepdim=True) / 16 * 258 * 2.0 ** -24
    # a query as the sum of two e4m3 values: to 2^-22 of the largest of its 64 dims
    score = score + q.abs().amax(-1, keepdim=True) * k.abs().sum(-1).amax() / 16 * 2.0 ** -22
    rel = 2.0 ** -8 + 2 * score + (2 * k.shape[0] + 64) * 2.0 ** -24
    return o, rel * (p @ v.abs()) + 2.0 ** -8 * o.abs() + 1e-30


def attend(state, b, q, gate=None, pages=None):
    """(outputs, error bounds) [T, heads * 256] and the rows that have one."""
    t, hq, _ = q.shape
    out = torch.zeros(t, hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    rows = []
    for row, i, pos in b.rows():
        rows.append(row)
        if pos < 0 or b.lens[i] > b.width * b.page:
            continue
        for h in range(hq // GROUP):
            mine = range(pos // b.page + 1) if pages is None else [
                int(x) for x in pages[row, h] if 0 <= int(x) <= pos // b.page]
            s = slice(h * GROUP, (h + 1) * GROUP)
            out[row, s], tol[row, s] = attend_row(state, b, q[row, s], i, h, pos, mine)
    if gate is not None:
        g = torch.sigmoid(gate.double().view(t, hq, 2, D)[:, :, 1])
        out, tol = out * g, tol * g + 2.0 ** -20 * (out * g).abs()
    return out.flatten(1), tol.flatten(1), rows


def select(state, b, q, budget, sinks, recents):
    """Selected pages per (row, head), as lists."""
    t, hq, _ = q.shape
    out = {}
    for row, i, pos in b.rows():
        for h in range(hq // GROUP):
            n = pos // b.page + 1 if pos >= 0 and b.lens[i] <= b.width * b.page else 0
            if n <= budget:
                out[row, h] = list(range(n))
                continue
            x = q[row, h * GROUP:(h + 1) * GROUP].double()
            fin = x[torch.isfinite(x)].abs()
            top = fin.max().item() if fin.numel() else 0.0
            step = 2.0 ** (math.frexp(top)[1] - 7) if top else 1.0
            qi = torch.nan_to_num(torch.round(x / step), nan=0.0, posinf=127, neginf=-127).clamp(-127, 127)
            scores = []
            for p in range(n):
                pid = int(b.table[i, p])
                if not 0 <= pid < state.k.shape[0]:
                    scores.append(-math.inf)
                    continue
                bd = state.bounds[pid, h].double()
                s = torch.maximum(qi * bd[0], qi * bd[1]).sum(-1).max().item()
                scores.append(s * 2.0 ** (int(state.ke[pid, h]) - 127))
            forced = [p for p in range(n) if p < sinks or p >= n - recents]
            rest = sorted((p for p in range(n) if p not in forced), key=lambda p: (-scores[p], p))
            out[row, h] = sorted(forced + rest[:budget - len(forced)])
    return out
