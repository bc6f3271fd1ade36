"""Operators of a server that runs many requests at once beside the paged cache:
the Gated DeltaNet layer's convolution and delta rule over a ragged batch with
states in slots, low-rank adapters of many requests beside a shared projection,
and the page table's turn (trim, fork, extend with copies) and compaction.

``listed()`` and ``draw()`` give cases, ``prepare()`` what a serving program
holds before the call, ``run()`` one call, ``exact()`` its result in 64 bits and
``work()`` what it cannot do without.  With ``own`` false, ``run`` computes the
operators from elementary torch operations in 32 bits.

A batch is ``cu_tokens`` [seqs + 1] and one number for each sequence: the slot of
its states, or its adapter.  Value head h of the delta rule reads key head h // 2,
heads of 128; a page holds ``page`` tokens of two KV heads of 256 as e4m3.
"""
import math
import os
import sys

import torch

own = False

HK, HV, DK = 16, 32, 128
CONV, IN_ROWS = 8192, 12352          # conv channels; rows of the layer's fused input projection
CHUNK = 64
KV_HEADS, D = 2, 256
# inputs and the widths of the stacked weights of the projections that carry adapters
PROJ = {"qkv": (2048, (8192, 512, 512)), "out": (4096, (2048,)), "mixed": (2048, (8192, 4096, 32, 32))}


def listed():
    return [
        # the convolution of a full server's decode step
        {"name": "conv decode batch of 64", "op": "conv", "seqs": 64, "new": 1, "ragged": False},
        # prompts and turns of odd lengths in one call
        {"name": "conv ragged prompts", "op": "conv", "seqs": 13, "new": 1531, "ragged": True},
        # one user's next token
        {"name": "delta 1 token", "op": "delta", "seqs": 1, "new": 1, "ragged": False},
        # a full server's decode step
        {"name": "delta decode batch of 64", "op": "delta", "seqs": 64, "new": 1, "ragged": False},
        # prompts and turns of odd lengths in one call, some of them with a state
        {"name": "delta ragged prompts", "op": "delta", "seqs": 13, "new": 1531, "ragged": True},
        # one user's next token through an adapter of rank 16
        {"name": "adapter 1 token", "op": "adapter", "proj": "qkv", "seqs": 1, "new": 1, "ragged": False,
         "adapters": 4, "rank": 16},
        # a decode step of requests with adapters of several ranks, some with none
        {"name": "adapter decode batch of 61", "op": "adapter", "proj": "mixed", "seqs": 61, "new": 1,
         "ragged": False, "adapters": 17, "rank": 32},
        # a step of long prompts with two adapters and one without
        {"name": "adapter prompts of 8190", "op": "adapter", "proj": "qkv", "seqs": 3, "new": 2730,
         "ragged": False, "adapters": 2, "rank": 64},
        # the prompt of one user continued four ways, its last page copied for each
        {"name": "turn of 1 by 4", "op": "turn", "page": 64, "layers": 2, "parents": 1, "children": 4, "ctx": 1000,
         "pool": 512},
        # a server's turn: a third of its rows are given up, forked again and grow
        {"name": "turn of 43 by 1", "op": "turn", "page": 64, "layers": 10, "parents": 43, "children": 43, "ctx": 6000,
         "pool": 3300},
        # a small cache whose pages lie apart
        {"name": "compaction of 300 pages", "op": "compact", "page": 16, "layers": 2, "parents": 7, "children": 0,
         "ctx": 1100, "pool": 511},
        # what a server does before it gives memory back
        {"name": "compaction of 2600 pages", "op": "compact", "page": 64, "layers": 6, "parents": 33, "children": 12,
         "ctx": 5000, "pool": 2600},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "delta", "delta", "adapter", "adapter", "turn", "compact"])
    if op in ("turn", "compact"):
        c = {"op": op, "page": rng.choice([16, 32, 64, 128]), "layers": rng.randint(1, 10), "parents": _log(rng, 1, 43)}
        c["children"] = c["parents"] * rng.randint(1, max(1, 43 // c["parents"])) if op == "turn" else _log(rng, 1, 12)
        c["ctx"] = _log(rng, 1, 6000)
        # no more bytes of pages than the largest listed
        most = 2600 * 64 * 10 // (c["page"] * c["layers"])
        held = c["parents"] * -(-c["ctx"] // c["page"]) + c["children"]
        if held > most * 3 // 4:
            c["ctx"] = max(1, (most * 3 // 4 - c["children"]) // c["parents"] * c["page"])
            held = c["parents"] * -(-c["ctx"] // c["page"]) + c["children"]
        c["pool"] = held + rng.randint(c["children"] + 1, held + c["children"] + 50)
        if op == "compact":
            c["layers"] = max(1, min(c["layers"], 2600 * 64 * 6 // (c["pool"] * c["page"])))
        return c
    c = {"op": op, "ragged": rng.random() < 0.6, "seqs": _log(rng, 1, 64)}
    c["new"] = 1 if rng.random() < 0.4 else _log(rng, 2, 8190)
    c["new"] = max(1, min(c["new"], 4096 if op == "delta" else 8190, 9000 // c["seqs"]))
    if op == "adapter":
        c["proj"] = rng.choice(["qkv", "out", "mixed"])
        c["adapters"], c["rank"] = _log(rng, 1, 24), rng.choice([8, 16, 24, 32, 64])
        if c["proj"] == "mixed":
            c["new"] = max(1, min(c["new"], 6000 // c["seqs"]))
    return c


def _lengths(case):
    b, new = case["seqs"], case["new"]
    if not case["ragged"]:
        return [new] * b
    return [1 + (i * 7919 + new - 1) % new for i in range(b)]


def _ranks(case):
    """The adapters' ranks: the largest, and fewer."""
    r = case["rank"]
    return [max(4, r >> (i % 3)) for i in range(case["adapters"])]


def _wants(case):
    """Each sequence's adapter; every seventh request and one out of range have none."""
    n = case["adapters"]
    return [(-1 if i % 7 == 5 else (i * 5 + 1) % n) if i else 0 for i in range(case["seqs"])]


def _held(case):
    """Tokens of each parent."""
    p, ctx = case["parents"], case["ctx"]
    return [max(1, int(ctx * (1.0 - 0.7 * ((i * 0.6180339887) % 1.0)))) for i in range(p)]


def _copied(case):
    """Children of a parent whose last page is not full: one page of every layer is copied for each."""
    held, p = _held(case), case["parents"]
    return sum(held[i % p] % case["page"] > 0 for i in range(case["children"]))


def _moved(case):
    """Pages that lie behind the number of pages held: about their share of the pool."""
    held = sum(-(-x // case["page"]) for x in _held(case))
    return held * (case["pool"] - held) // case["pool"]


def work(case):
    op = case["op"]
    if op in ("turn", "compact"):
        page = 2 * KV_HEADS * (case["page"] * D + 1) * case["layers"]
        table = 4 * (sum(-(-x // case["page"]) for x in _held(case)) + case["pool"])
        n = _copied(case) if op == "turn" else _moved(case)
        return {"bytes": 2 * n * page + 2 * table, "flops": 0}
    new = _lengths(case)
    t, b = sum(new), case["seqs"]
    if op == "conv":
        return {"bytes": t * CONV * 4 + CONV * 8 + b * CONV * 12, "flops": t * CONV * 12}
    if op == "delta":
        with_state = b if t == b else sum(i % 3 == 0 for i in range(b))
        return {"bytes": t * (2 * HK * DK + 2 * HV * DK) * 2 + t * HV * 8 + (b + with_state) * HV * DK * DK * 4,
                "flops": t * HV * DK * DK * 7}
    k, widths = PROJ[case["proj"]]
    ranks, wants = _ranks(case), _wants(case)
    used = sum(ranks[i] for i in set(wants) if i >= 0)
    rows = sum(n for n, w in zip(new, wants) if w >= 0)
    per = sum(n * ranks[w] for n, w in zip(new, wants) if w >= 0)
    return {"bytes": used * 2 * (k * len(widths) + sum(widths)) + rows * 2 * (k + 2 * sum(widths)),
            "flops": 2 * per * (k * len(widths) + sum(widths))}


# ---------------------------------------------------------------- inputs

def _randn(shape, g, dev, scale=1.0):
    return (torch.randn(shape, generator=g, device=dev) * scale).to(torch.bfloat16)


def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "aima-amd395-qwen36-35b-linux-engine_amd")
    if at not in sys.path:
        sys.path.insert(0, at)


def _prepare_pages(case, g, dev, s):
    page, rows, pool = case["page"], case["parents"] + case["children"], case["pool"]
    held = _held(case)
    pages = [-(-x // page) for x in held]
    s["width"] = max(pages) + 2
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.full((rows, s["width"]), -1, dtype=torch.int32, device=dev)
    refs = torch.zeros(pool, dtype=torch.int32, device=dev)
    at, lens = 0, held + [0] * case["children"]
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    if case["op"] == "compact":          # rows that share all full pages of another
        for i in range(case["children"]):
            src = i % case["parents"]
            n = held[src] // page
            table[case["parents"] + i, :n] = table[src, :n]
            lens[case["parents"] + i] = n * page
    taken = table[table >= 0].long()
    refs.index_add_(0, taken, torch.ones_like(taken, dtype=torch.int32))
    s |= {"page": page, "rows": rows, "table": table, "refs": refs,
          "lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
    # pages as an append leaves them: finite e4m3 values, a scale for each page and head
    shape = (pool, KV_HEADS, page, D)
    s["layers"] = []
    for _ in range(case["layers"]):
        s["layers"].append({
            **{n: torch.randint(0, 0x78, shape, generator=g, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn)
               for n in ("k_pages", "v_pages")},
            **{n: torch.randint(100, 140, (pool, KV_HEADS), generator=g, device=dev, dtype=torch.uint8)
               for n in ("k_exp", "v_exp")}})
    # a turn: the children's rows are given up, taken from a parent again and grow by a token
    p, n = case["parents"], case["children"]
    def vector(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)
    s["keep"] = vector([1 << 30] * p + [0] * n)
    s["parent"] = vector([-1] * p + [i % p for i in range(n)])
    s["add"] = vector([0] * p + [1] * n)
    if own:
        _package()
        from qwen36_attn import page_tables, paged_attention
        s["pt"] = page_tables
        s["caches"] = [paged_attention.PagedKVCache.of(c["k_pages"], c["v_pages"], c["k_exp"], c["v_exp"])
                       for c in s["layers"]]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] in ("turn", "compact"):
        _prepare_pages(case, g, dev, s)
        return s
    new, b = _lengths(case), case["seqs"]
    t = sum(new)
    s["longest"] = max(new)
    s["cu"] = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
    if case["op"] == "adapter":
        k, widths = PROJ[case["proj"]]
        n, r = case["adapters"], case["rank"]
        s["x"] = _randn((t, k), g, dev)                      # normed rows
        s["y"] = _randn((t, sum(widths)), g, dev)            # the shared projection's rows
        s["a"] = _randn((n, len(widths), r, k), g, dev, k ** -0.5)
        s["b"] = _randn((n, sum(widths), r), g, dev, 0.1)
        s["ranks"] = torch.tensor(_ranks(case), dtype=torch.int32, device=dev)
        s["scales"] = torch.rand(n, generator=g, device=dev) + 0.5
        s["ids"] = torch.tensor(_wants(case), dtype=torch.int32, device=dev)
        if own:
            _package()
            from qwen36_attn import adapters
            s["ad"] = adapters
            s["set"] = adapters.AdapterSet(s["a"], s["b"], widths, s["ranks"], s["scales"])
            # the step's rows by adapter: made once, used by every projection of every layer
            s["batch"] = adapters.AdapterBatch(s["cu"], s["ids"], t, n)
        return s
    slots = b + 3
    s["slots"] = torch.randperm(slots, generator=g, device=dev)[:b].to(torch.int32)
    # a step of single tokens carries every state; of prompts a third go on from one
    s["has"] = torch.tensor([t == b or i % 3 == 0 for i in range(b)], device=dev)
    if case["op"] == "conv":
        s["mixed"] = _randn((t, IN_ROWS), g, dev)[:, :CONV]
        s["w"] = _randn((CONV, 4), g, dev, 0.5)
        s["states"] = _randn((slots, CONV, 3), g, dev)
    else:
        x = torch.nn.functional.silu(_randn((t, CONV), g, dev))   # the convolution's rows
        s["q"] = x[:, :HK * DK].view(t, HK, DK)
        s["k"] = x[:, HK * DK:2 * HK * DK].view(t, HK, DK)
        s["v"] = x[:, 2 * HK * DK:].view(t, HV, DK)
        a = torch.rand(HV, generator=g, device=dev) * 16.0
        s["g"] = -torch.nn.functional.softplus(torch.randn(t, HV, generator=g, device=dev)) * a
        s["beta"] = torch.sigmoid(torch.randn(t, HV, generator=g, device=dev))
        s["states"] = torch.randn(slots, HV, DK, DK, generator=g, device=dev) * 0.2
    if own:
        _package()
        from qwen36_attn import ragged_deltanet
        s["rd"] = ragged_deltanet
    return s


# ------------------------------------------------------------ plain forms

def _rows(s, t):
    """Sequence of every row and its place there."""
    i = torch.arange(t, device=s["cu"].device)
    seq = torch.searchsorted(s["cu"][1:], i.to(torch.int32), right=True)
    return seq, i - s["cu"][seq].long()


def _conv(s):
    x, states, t = s["mixed"].float(), s["states"], s["mixed"].shape[0]
    seq, col = _rows(s, t)
    old = torch.where(s["has"][:, None, None], states[s["slots"].long()].float(), 0.0)     # [b, C, 3]

    def tap(j, seq, col, last):
        """The input 3 - j rows before."""
        back = col - 3 + j
        here = x[(last - 3 + j).clamp(min=0)]
        return torch.where(back[:, None] >= 0, here, old[seq, :, (back + 3).clamp(max=2)])

    w = s["w"].float()
    last = torch.arange(t, device=x.device)
    y = tap(0, seq, col, last) * w[:, 0]
    y = y + tap(1, seq, col, last) * w[:, 1]
    y = y + tap(2, seq, col, last) * w[:, 2]
    y = (y + x * w[:, 3]).to(torch.bfloat16).float()
    out = (y / (1.0 + torch.exp(-y))).to(torch.bfloat16)
    b = torch.arange(s["case"]["seqs"], device=x.device)
    n, z = (s["cu"][1:] - s["cu"][:-1]).long(), s["cu"][1:].long()
    new = torch.stack((tap(0, b, n, z), tap(1, b, n, z), tap(2, b, n, z)), -1)
    states[s["slots"].long()] = new.to(torch.bfloat16)
    return out


def _normed(x):
    return x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()


def _padded(s, length):
    """q, k, v, g and beta of every sequence [b, heads, length, ...], zeros behind its end."""
    b = s["case"]["seqs"]
    at = s["cu"][:-1, None].long() + torch.arange(length, device=s["cu"].device)
    there = at < s["cu"][1:, None]
    at = at.clamp(max=s["q"].shape[0] - 1)

    def rows(x):
        x = torch.where(there.view(b, length, *[1] * (x.dim() - 1)), x[at], 0.0)
        return x.transpose(1, 2)
    q, k = (_normed(s[n].float()).repeat_interleave(HV // HK, 1) for n in ("q", "k"))
    return rows(q * DK ** -0.5), rows(k), rows(s["v"].float()), rows(s["g"]), rows(s["beta"]), at, there


def _delta_steps(s, state):
    """Token by token."""
    q, k, v, g, beta, at, there = _padded(s, s["longest"])
    outs = []
    for t in range(s["longest"]):
        state = state * torch.exp(g[:, :, t, None, None])
        d = (v[:, :, t] - (state * k[:, :, t, :, None]).sum(2)) * beta[:, :, t, None]
        state = state + k[:, :, t, :, None] * d[:, :, None]
        outs.append((state * q[:, :, t, :, None]).sum(2))
    return torch.stack(outs, 1), state, at, there


def _delta_chunks(s, state):
    """Chunks of 64 tokens: the rows of a chunk are solved for at once, chunks follow one another."""
    n = -(-s["longest"] // CHUNK)
    q, k, v, g, beta, at, there = _padded(s, n * CHUNK)
    q, k, v, g, beta = (x.unflatten(2, (n, CHUNK)) for x in (q, k, v, g, beta))
    g = g.cumsum(-1)
    i = torch.arange(CHUNK, device=g.device)
    low = i[:, None] >= i
    decay = torch.exp(torch.where(low, g[..., :, None] - g[..., None, :], -math.inf))
    kb = k * beta[..., None]
    left = torch.matmul(kb, k.transpose(-1, -2)) * decay * (i[:, None] > i)
    inv = torch.eye(CHUNK, device=g.device).expand_as(left)
    for m in (1, 2, 4, 8, 16, 32):      # the inverse of I + left, from blocks of m to blocks of 2m
        off = left * ((i[:, None] // (2 * m) == i // (2 * m)) & (i[:, None] // m % 2 > i // m % 2))
        inv = inv - torch.matmul(inv, torch.matmul(off, inv))
    u, w = torch.matmul(inv, v * beta[..., None]), torch.matmul(inv, kb * torch.exp(g)[..., None])
    inner = torch.matmul(q, k.transpose(-1, -2)) * decay
    q = q * torch.exp(g)[..., None]
    k = k * torch.exp(g[..., -1:] - g)[..., None]
    outs = []
    for c in range(n):
        d = u[:, :, c] - torch.matmul(w[:, :, c], state)
        outs.append(torch.matmul(q[:, :, c], state) + torch.matmul(inner[:, :, c], d))
        state = state * torch.exp(g[:, :, c, -1])[..., None, None] + torch.matmul(k[:, :, c].transpose(-1, -2), d)
    return torch.cat(outs, 2).transpose(1, 2), state, at, there


def _delta(s):
    slots = s["slots"].long()
    state = torch.where(s["has"][:, None, None, None], s["states"][slots], 0.0)
    o, state, at, there = (_delta_steps if s["longest"] <= 4 else _delta_chunks)(s, state)
    s["states"][slots] = state
    return o[there].to(torch.bfloat16)       # the rows in the batch's order


def _adapter(s):
    t, n, r = s["x"].shape[0], s["case"]["adapters"], s["case"]["rank"]
    widths = PROJ[s["case"]["proj"]][1]
    seq, _ = _rows(s, t)
    mine = s["ids"][seq].long()
    use = torch.arange(r, device=mine.device) < s["ranks"][:, None]                       # [n, r]
    use = use & (mine[:, None] == torch.arange(n, device=mine.device))[:, :, None]        # [t, n, r]
    use = torch.where(use, s["scales"][:, None], 0.0)
    x = s["x"].float()
    parts, at = [], 0
    for i, width in enumerate(widths):
        h = torch.matmul(x, s["a"][:, i].float().flatten(0, 1).transpose(0, 1)).view(t, n, r) * use
        up = s["b"][:, at:at + width].float().transpose(1, 2).reshape(n * r, width)
        parts.append(torch.matmul(h.flatten(1), up))
        at += width
    s["y"].copy_((s["y"].float() + torch.cat(parts, 1)).to(torch.bfloat16))
    return s["y"]


def _count(refs, table, lens, page, by):
    """Adds `by` to the count of every page that the rows hold."""
    held = torch.arange(table.shape[1], device=table.device) * page < lens[:, None]
    at = torch.where(held & (table >= 0), table, 0).long()
    refs.index_add_(0, at.flatten(), torch.where(held & (table >= 0), by, 0).to(torch.int32).flatten())


def _trim(s):
    refs, table, lens, page = s["refs"], s["table"], s["lens"], s["page"]
    kept = torch.minimum(lens, s["keep"].clamp(min=0))
    _count(refs, table, lens, page, -1)
    _count(refs, table, kept, page, 1)
    column = torch.arange(table.shape[1], device=table.device) * page
    table.copy_(torch.where((column >= kept[:, None]) & (column < lens[:, None]), -1, table))
    lens.copy_(kept)


def _fork(s):
    refs, table, lens, page, p = s["refs"], s["table"], s["lens"], s["page"], s["parent"]
    at = p.clamp(min=0).long()
    ok = (p >= 0) & (lens == 0) & (p[at] < 0)
    column = torch.arange(table.shape[1], device=table.device) * page
    take = ok[:, None] & (column < lens[at][:, None])
    rows = torch.where(take, table[at], table)
    new = torch.where(ok, lens[at], lens)
    _count(refs, rows, torch.where(ok, new, 0), page, 1)
    table.copy_(rows)
    lens.copy_(new)


def _extend(s):
    refs, table, lens, page, add = s["refs"], s["table"], s["lens"], s["page"], s["add"].clamp(min=0)
    have, want = -(-lens // page), -(-(lens + add) // page)
    last = table.gather(1, (have - 1).clamp(min=0).long()[:, None])[:, 0]
    copy = (add > 0) & (lens % page > 0) & (last >= 0) & (refs[last.clamp(min=0).long()] > 1)
    need = torch.where(add > 0, want - have + copy, 0)
    until = need.cumsum(0)
    free = refs <= 0
    ok = (add > 0) & (until <= free.sum()) & (want <= table.shape[1])
    # free pages in ascending order, then the others
    order = torch.sort((~free).to(torch.int32), stable=True)[1].to(torch.int32)
    column = torch.arange(table.shape[1], device=table.device)
    first = have - copy.to(torch.int32)
    new = ok[:, None] & (column >= first[:, None]) & (column < want[:, None])
    place = (until - need)[:, None] + column - first[:, None]
    rows = torch.where(new, order[place.clamp(0, refs.shape[0] - 1).long()], table)
    refs.index_add_(0, torch.where(copy & ok, last, 0).long(), -(copy & ok).to(torch.int32))
    refs.index_add_(0, torch.where(new, rows, 0).long().flatten(), new.to(torch.int32).flatten())
    src = last[copy & ok].long()
    dst = rows.gather(1, (have - 1).clamp(min=0).long()[:, None])[:, 0][copy & ok].long()
    _copy(s, src, dst)
    table.copy_(rows)
    lens.copy_(torch.where(ok, lens + add, lens))
    return (ok | (add == 0)).to(torch.int32)


def _copy(s, src, dst):
    for c in s["layers"]:
        for x in c.values():
            x = x.view(torch.uint8)
            x[dst] = x[src]


def _compact(s):
    """Pages held behind the number of pages held go to the free ones before it, in ascending order."""
    refs, table = s["refs"], s["table"]
    held = refs > 0
    n = held.sum()
    i = torch.arange(refs.shape[0], device=refs.device)
    src, dst = i[held & (i >= n)], i[~held & (i < n)]
    _copy(s, src, dst)
    to = i.clone()
    to[src] = dst
    rows = torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), table)
    new = torch.where(i < n, refs, 0)
    new[dst] = refs[src]
    return new, rows


def _pools(s):
    return [[c[n] for n in ("k_pages", "v_pages", "k_exp", "v_exp")] for c in s["layers"]]


def run(s):
    op = s["case"]["op"]
    if op == "conv":
        if own:
            out = s["rd"].ragged_conv1d(s["mixed"], s["w"], s["states"], s["cu"], s["slots"], has_state=s["has"])
        else:
            out = _conv(s)
        return out, s["states"]
    if op == "delta":
        if own:
            out = s["rd"].ragged_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], s["states"], s["cu"],
                                            s["slots"], has_state=s["has"], longest=s["longest"])
        else:
            out = _delta(s)
        return out, s["states"]
    if op == "adapter":
        return s["ad"].apply_adapters(s["y"], s["x"], s["set"], s["batch"]) if own else _adapter(s)
    if op == "compact":
        if own:
            refs, table = s["pt"].compact(s["refs"], s["table"], s["lens"], s["caches"])
        else:
            refs, table = _compact(s)
        return refs, table, _pools(s)
    if own:
        s["pt"].trim(s["refs"], s["table"], s["lens"], s["keep"], s["page"])
        s["pt"].fork(s["refs"], s["table"], s["lens"], s["parent"], s["page"])
        granted = s["pt"].extend(s["refs"], s["table"], s["lens"], s["add"], s["caches"])
    else:
        _trim(s)
        _fork(s)
        granted = _extend(s)
    return granted, s["refs"], s["table"], s["lens"], _pools(s)


# ------------------------------------------------------------ in 64 bits

def _exact_conv(s):
    cu, slots, has = s["cu"].tolist(), s["slots"].tolist(), s["has"].tolist()
    states, w = s["states"].double(), s["w"].double()
    outs = []
    for i, slot in enumerate(slots):
        old = states[slot].T if has[i] else torch.zeros(3, CONV, dtype=torch.float64, device=w.device)
        x = torch.cat((old, s["mixed"][cu[i]:cu[i + 1]].double()))
        y = (x.unfold(0, 4, 1) * w).sum(-1).to(torch.bfloat16).double()
        outs.append(y * torch.sigmoid(y))
        states[slot] = x[-3:].T
    return torch.cat(outs), states


def _exact_delta(s):
    b, cu = s["case"]["seqs"], s["cu"].long()
    slots = s["slots"].long()
    state = s["states"][slots].double() * s["has"][:, None, None, None]
    out = torch.zeros(s["q"].shape[0], HV, DK, dtype=torch.float64, device=state.device)
    which = torch.arange(HV, device=state.device) // (HV // HK)
    for j in range(s["longest"]):
        live = torch.nonzero(cu[1:] - cu[:-1] > j)[:, 0]
        if live.numel() == b:
            live = slice(None)
        at = cu[:-1][live] + j
        q, k, v = (s[n][at].double() for n in ("q", "k", "v"))
        q = (q / (q.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt() / math.sqrt(DK))[:, which]
        k = (k / (k.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt())[:, which]
        x = state[live] * s["g"][at].double().exp()[..., None, None]
        d = (v - torch.einsum("bhkv,bhk->bhv", x, k)) * s["beta"][at].double()[..., None]
        x = x + torch.einsum("bhk,bhv->bhkv", k, d)
        out[at] = torch.einsum("bhkv,bhk->bhv", x, q)
        state[live] = x
    states = s["states"].double()
    states[slots] = state
    return out, states


def _exact_adapter(s):
    widths = PROJ[s["case"]["proj"]][1]
    cu, y = s["cu"].tolist(), s["y"].double()
    for i, w in enumerate(s["ids"].tolist()):
        if 0 <= w < s["case"]["adapters"]:
            x, r = s["x"][cu[i]:cu[i + 1]].double(), s["ranks"][w].item()
            scale, at = s["scales"][w].double(), 0
            for j, width in enumerate(widths):
                h = x @ s["a"][w, j, :r].double().T
                y[cu[i]:cu[i + 1], at:at + width] += scale * (h @ s["b"][w, at:at + width, :r].double().T)
                at += width
    return y


def _exact_pages(s):
    """The tables by hand, on the host; the pages as the values that they hold."""
    page, pool = s["page"], s["case"]["pool"]
    refs, lens = s["refs"].tolist(), s["lens"].tolist()
    table = s["table"].tolist()
    moves, granted = [], []
    if s["case"]["op"] == "compact":
        n = sum(r > 0 for r in refs)
        moves = list(zip([i for i in range(n, pool) if refs[i] > 0], [i for i in range(n) if refs[i] <= 0]))
        to = dict(moves)
        table = [[to.get(x, x) for x in row] for row in table]
        for a, z in moves:
            refs[a], refs[z] = 0, refs[a]
    else:
        for i, parent in enumerate(s["parent"].tolist()):
            if parent >= 0:
                n = -(-lens[parent] // page)
                table[i][:n] = table[parent][:n]
                lens[i] = lens[parent]
                for x in table[i][:n]:
                    refs[x] += 1
        free, before = [i for i in range(pool) if refs[i] <= 0], list(refs)
        for i, add in enumerate(s["add"].tolist()):
            granted.append(1)
            if add:
                n = -(-lens[i] // page)
                first = n - (lens[i] % page > 0 and before[table[i][n - 1]] > 1)
                for j in range(first, -(-(lens[i] + add) // page)):
                    z = free.pop(0)
                    if j < n:
                        moves.append((table[i][j], z))
                        refs[table[i][j]] -= 1
                    table[i][j] = z
                    refs[z] += 1
                lens[i] += add
    dev = s["refs"].device
    at = torch.arange(pool, device=dev)
    if moves:
        src, dst = torch.tensor(moves, device=dev).unbind(1)
        at[dst] = src
    pools = [[c["k_pages"][at].float(), c["v_pages"][at].float(), c["k_exp"][at], c["v_exp"][at]] for c in s["layers"]]
    refs, table = (torch.tensor(x, dtype=torch.int32, device=dev) for x in (refs, table))
    if s["case"]["op"] == "compact":
        return refs, table, pools
    return (torch.tensor(granted, dtype=torch.int32, device=dev), refs, table,
            torch.tensor(lens, dtype=torch.int32, device=dev), pools)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "conv":
        return _exact_conv(s)
    if op == "delta":
        return _exact_delta(s)
    return _exact_adapter(s) if op == "adapter" else _exact_pages(s)
