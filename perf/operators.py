"""The paged-cache operators: appending rotated keys and values, attention over
pages of 8 or 16 bits, and attention over pages that a cheap score selects.

``listed()`` and ``draw()`` give cases, ``prepare()`` what a serving program
holds before the call, ``run()`` one call, ``exact()`` its result in 64 bits and
``work()`` what it cannot do without.  With ``own`` false, ``run`` computes the
operators from elementary torch operations in 32 bits.

Head layout: query head h reads KV head h // 8, head dim 256.  A page holds
``page`` tokens of every KV head, [KV head][token][dim]; an e4m3 page has a
power-of-two scale for each KV head, kept as the byte e of 2^(e - 127).
"""
import math
import os
import sys

import torch

own = False

D, GROUP, PAIRS = 256, 8, 32
LOWEST, MAX_POS = 16, 262144


def listed():
    return [
        # one user's next token: nothing but latency
        {"name": "append 1 token", "op": "append", "cache": "e4m3", "heads": 2, "page": 64, "seqs": 1, "ctx": 1000,
         "new": 1, "ragged": False, "bounds": False},
        # a decode step of a full server, the cache ready for selection
        {"name": "append decode batch of 64", "op": "append", "cache": "e4m3", "heads": 2, "page": 64, "seqs": 64,
         "ctx": 32768, "new": 1, "ragged": True, "bounds": True},
        # seven short prompts and turns of odd lengths in one call, cache of 16 bits
        {"name": "append ragged prompts bf16", "op": "append", "cache": "bf16", "heads": 2, "page": 16, "seqs": 7,
         "ctx": 1531, "new": 517, "ragged": True, "bounds": False},
        # a long prompt's second part
        {"name": "append 8192 tokens", "op": "append", "cache": "e4m3", "heads": 2, "page": 64, "seqs": 1, "ctx": 4096,
         "new": 8192, "ragged": False, "bounds": True},
        # one user's next token over a short conversation
        {"name": "attend 1 token over 1000", "op": "attend", "cache": "e4m3", "heads": 2, "page": 64, "seqs": 1,
         "ctx": 1000, "new": 1, "ragged": False, "gate": True},
        # the longest conversation that the benchmark decodes over
        {"name": "attend 1 token over 128K", "op": "attend", "cache": "e4m3", "heads": 2, "page": 64, "seqs": 1,
         "ctx": 131071, "new": 1, "ragged": False, "gate": True},
        # a full server's decode step over conversations of every length, small pages
        {"name": "attend decode batch of 32", "op": "attend", "cache": "e4m3", "heads": 2, "page": 16, "seqs": 32,
         "ctx": 32768, "new": 1, "ragged": True, "gate": True},
        # five drafted tokens of each sequence under verification, one KV head of a split model, 16 bits
        {"name": "attend 5 drafts of 16 bf16", "op": "attend", "cache": "bf16", "heads": 1, "page": 32, "seqs": 16,
         "ctx": 12001, "new": 5, "ragged": False, "gate": False},
        # a chunk of a long document's prompt
        {"name": "attend chunk of 2048 over 30K", "op": "attend", "cache": "e4m3", "heads": 2, "page": 64, "seqs": 1,
         "ctx": 30001, "new": 2048, "ragged": False, "gate": True},
        # one user's next token over 128K, one page of 32 read
        {"name": "sparse 1 token over 128K", "op": "sparse", "cache": "e4m3", "heads": 2, "page": 64, "seqs": 1,
         "ctx": 131071, "new": 1, "ragged": False, "budget": 64, "gate": True},
        # a decode step of 16 long conversations
        {"name": "sparse decode batch of 16", "op": "sparse", "cache": "e4m3", "heads": 2, "page": 32, "seqs": 16,
         "ctx": 65536, "new": 1, "ragged": True, "budget": 96, "gate": True},
        # a turn's tokens, each with pages of its own, 16 bits
        {"name": "sparse turn of 300 over 16K bf16", "op": "sparse", "cache": "bf16", "heads": 2, "page": 64, "seqs": 1,
         "ctx": 16001, "new": 300, "ragged": False, "budget": 24, "gate": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "sparse"])
    c = {"op": op, "cache": rng.choice(["e4m3", "e4m3", "bf16"]), "heads": rng.choice([1, 2, 2, 4]),
         "page": rng.choice([16, 32, 64, 128]), "ragged": rng.random() < 0.5}
    c["seqs"] = _log(rng, 1, 64)
    c["ctx"] = _log(rng, 1, 131071)
    c["new"] = 1 if rng.random() < 0.5 else _log(rng, 1, 2048)
    # at most what the largest listed cases hold: tokens in the cache, new tokens, pairs of them
    c["new"] = max(1, min(c["new"], 8192 // c["seqs"]))
    c["ctx"] = max(1, min(c["ctx"], (1 << 19) // (c["seqs"] * c["heads"])))
    pairs = c["seqs"] * c["heads"] * c["new"] * (c["ctx"] + c["new"])
    if op == "attend" and pairs > 1 << 26:
        c["new"] = max(1, (1 << 26) // (c["seqs"] * c["heads"] * (c["ctx"] + c["new"])))
    if op == "append":
        c["bounds"] = rng.random() < 0.5
    else:
        c["gate"] = rng.random() < 0.5
    if op == "sparse":
        c["budget"] = _log(rng, 3, 128)
        most = max(1, (1 << 21) // (c["seqs"] * c["heads"] * c["budget"] * c["page"]))
        c["new"] = min(c["new"], most)
    return c


def _lengths(case):
    """(tokens in the cache before, new tokens) of each sequence."""
    b, ctx, new = case["seqs"], case["ctx"], case["new"]
    if not case["ragged"]:
        return [ctx] * b, [new] * b
    part = [1.0 - 0.9 * ((i * 0.6180339887) % 1.0) for i in range(b)]
    return [max(0, int(ctx * p)) for p in part], [1 + (i * 7919 + new - 1) % new for i in range(b)]


def _old_rows(case):
    """Cache rows that an append reads and writes again: the sequence's last page, where it is not full."""
    return sum(x % case["page"] for x in _lengths(case)[0])


def work(case):
    before, new = _lengths(case)
    h, elem, t = case["heads"], 1 if case["cache"] == "e4m3" else 2, sum(new)
    hq = h * GROUP
    if case["op"] == "append":
        rows = t * (hq + 2 * h) * D * 2 + t * hq * D * 2 + t * 2 * h * D * elem + t * PAIRS * 8
        pages = sum((x + n - 1) // case["page"] - x // case["page"] + 1 for x, n in zip(before, new))
        return {"bytes": rows + pages * h * (2 if case["cache"] == "e4m3" else 0) + (pages * h * 2 * D if case["bounds"] else 0),
                "flops": t * (hq + h) * D * 6}
    io = t * hq * D * 2 * (3 if case["gate"] else 2)
    if case["op"] == "attend":
        pairs = sum(n * x + n * (n + 1) // 2 for x, n in zip(before, new))
        return {"bytes": io + 2 * sum(x + n for x, n in zip(before, new)) * h * D * elem, "flops": 4 * D * hq * pairs}
    page, budget = case["page"], case["budget"]
    pages = [-(-(x + n) // page) for x, n in zip(before, new)]
    read = sum(min(p, n * budget) for p, n in zip(pages, new))
    keys = sum(n * min(budget * page, x + n) for x, n in zip(before, new))
    scored = sum(n * p for p, n in zip(pages, new))
    return {"bytes": io + sum(pages) * h * 2 * D + 2 * read * page * h * D * elem + t * h * budget * 4,
            "flops": 4 * D * hq * keys + 4 * D * hq * scored}


# ---------------------------------------------------------------- inputs

def _least(amax):
    """The least byte e with amax <= 448 * 2^(e - 127)."""
    m, x = torch.frexp(amax)
    return torch.where(amax > 0, x + 118 + (m > 0.875), torch.full_like(x, LOWEST)).clamp(min=LOWEST)


def _power(e):
    return torch.exp2(e.to(torch.float32) - 127.0)


def _randn(shape, g, dev, scale=1.0):
    return (torch.randn(shape, generator=g, device=dev) * scale).to(torch.bfloat16)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    before, new = _lengths(case)
    b, h, page = case["seqs"], case["heads"], case["page"]
    t, hq = sum(new), case["heads"] * GROUP
    lens = [x + n for x, n in zip(before, new)]
    wide = max(-(-x // page) for x in lens)
    pool = sum(-(-x // page) for x in lens) + 3
    # keys as a head norm leaves them, with channels of unequal size; values of a projection
    size = torch.exp(0.4 * torch.randn(h, 1, D, generator=g, device=dev))
    k = _randn((pool, h, page, D), g, dev) * size.to(torch.bfloat16)
    v = _randn((pool, h, page, D), g, dev, 0.7)
    s = {"case": case, "seqs": b, "page": page, "heads": h, "most": max(new)}
    k_exp = _least(k.abs().amax((2, 3)).float()).to(torch.uint8)
    v_exp = _least(v.abs().amax((2, 3)).float()).to(torch.uint8)
    if case["op"] == "sparse" or case.get("bounds"):
        step = _power(k_exp)[:, :, None] * 4.0
        top, low = k.amax(2).float() / step, k.amin(2).float() / step
        s["bounds"] = torch.stack((top.ceil(), low.floor()), 2).to(torch.int8)
    else:
        s["bounds"] = None
    if case["cache"] == "e4m3":
        k = (k.float() / _power(k_exp)[:, :, None, None]).to(torch.float8_e4m3fn)
        v = (v.float() / _power(v_exp)[:, :, None, None]).to(torch.float8_e4m3fn)
        s["k_exp"], s["v_exp"] = k_exp, v_exp
    else:
        s["k_exp"], s["v_exp"] = (k_exp if s["bounds"] is not None else None), None
    s["k_pages"], s["v_pages"] = k, v
    # the sequences' pages lie anywhere in the pool
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(b, wide, dtype=torch.int32, device=dev)
    at = 0
    for i, x in enumerate(lens):
        p = -(-x // page)
        table[i, :p] = order[at:at + p]
        at += p
    s["table"] = table
    s["cu"] = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["qkv"] = _randn((t, (2 * hq + 2 * h) * D), g, dev)   # [q | gate] of each head, k, v
    s["q_gate"] = s["qkv"][:, :2 * hq * D]
    if case["op"] == "append":
        s["k"] = s["qkv"][:, 2 * hq * D:(2 * hq + h) * D]
        s["v"] = s["qkv"][:, (2 * hq + h) * D:]
        s["q_norm"], s["k_norm"] = _randn((D,), g, dev, 0.3), _randn((D,), g, dev, 0.3)
        inv = 1.0e7 ** (-torch.arange(PAIRS, dtype=torch.float64, device=dev) / PAIRS)
        angle = torch.arange(max(lens), dtype=torch.float64, device=dev)[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    else:
        s["q"] = _randn((t, hq, D), g, dev, 1.2)
    if own:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "aima-amd395-qwen36-35b-linux-engine_amd"))
        from qwen36_attn import paged_attention as pa
        s["pa"] = pa
        s["cache"] = pa.PagedKVCache.of(s["k_pages"], s["v_pages"], s["k_exp"], s["v_exp"], s["bounds"])
    return s


# ------------------------------------------------------------ plain forms

def _slots(s):
    """Sequence and position of every new token."""
    i = torch.arange(s["qkv"].shape[0], device=s["cu"].device)
    seq = torch.searchsorted(s["cu"][1:], i.to(torch.int32), right=True)
    return seq, (s["lens"][seq] - (s["cu"][seq + 1] - i)).long()


def _normed(x, w, c, sn):
    """Head norm with weight w + 1, rounded to bf16, then the rotation of dims 0..63, rounded.  In 32 bits with
    every product and sum rounded, the squares summed in the framework's order (four neighbours, then halves): a
    key next to a border of the 8-bit values has to fall on its one side."""
    x = x.float()
    a = (x * x).unflatten(-1, (64, 4))
    a = (a[..., 0] + a[..., 1]) + (a[..., 2] + a[..., 3])
    a = a[..., :32] + a[..., 32:]
    a = a[..., :16] + a[..., 16:]
    a = a[..., :8] + a[..., 8:]
    a = a[..., :4] + a[..., 4:]
    a = a[..., :2] + a[..., 2:]
    a = a[..., :1] + a[..., 1:]
    inv = (1.0 / (a * (1.0 / 256.0) + 1e-6).double().sqrt()).float()
    y = ((x * inv) * (w.float() + 1.0)).to(torch.bfloat16).float()
    lo, hi = y[..., :PAIRS], y[..., PAIRS:2 * PAIRS]
    return torch.cat((lo * c - hi * sn, hi * c + lo * sn, y[..., 2 * PAIRS:]), -1).to(torch.bfloat16)


def _append(s):
    h, page, t = s["heads"], s["page"], s["qkv"].shape[0]
    seq, pos = _slots(s)
    c, sn = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = _normed(s["q_gate"].view(t, h * GROUP, 2 * D)[..., :D], s["q_norm"], c, sn)
    k = _normed(s["k"].reshape(t, h, D), s["k_norm"], c, sn)
    v = s["v"].reshape(t, h, D)
    at, row = s["table"][seq, pos // page].long(), pos % page
    first = s["lens"] - (s["cu"][1:] - s["cu"][:-1])            # the first new position
    held = s["table"].gather(1, (first // page).long()[:, None])[:, 0].long()
    mine, at_mine = torch.unique(at, return_inverse=True)       # the pages that get rows
    kept = torch.zeros(s["k_pages"].shape[0], dtype=torch.long, device=at.device)
    kept[held] = (first % page).long()                          # rows of a sequence's last page that stay
    kept = kept[mine]
    for pages, exp, x in ((s["k_pages"], s["k_exp"], k), (s["v_pages"], s["v_exp"], v)):
        if exp is not None:
            a = torch.zeros(mine.shape[0], h, device=x.device).index_reduce_(0, at_mine, x.abs().amax(-1).float(), "amax")
            was = exp[mine].int()
            e = torch.where(kept[:, None] > 0, torch.maximum(was, _least(a)), _least(a))
            less = torch.exp2((was - e).float())
            exp[mine] = e.to(torch.uint8)
            if pages is s["k_pages"] and s["bounds"] is not None:
                step = _power(e)[:, :, None] * 4.0
                old = s["bounds"][mine].float() * less[:, :, None, None]
                some, none = (kept > 0)[:, None, None], torch.full_like(old[:, :, 0], math.inf)
                top = torch.where(some, old[:, :, 0].ceil() * step, -none).index_reduce_(0, at_mine, x.float(), "amax")
                low = torch.where(some, old[:, :, 1].floor() * step, none).index_reduce_(0, at_mine, x.float(), "amin")
                s["bounds"][mine] = torch.stack(((top / step).ceil(), (low / step).floor()), 2).to(torch.int8)
        if pages.dtype == torch.float8_e4m3fn:
            old = torch.searchsorted(mine, held)                # the page of each sequence that may hold older rows
            there = pages[held].float() * less[old][:, :, None, None]
            stay = torch.arange(page, device=x.device) < (first % page)[:, None]
            seq_of, row_of = torch.nonzero(stay, as_tuple=True)
            pages.view(torch.uint8)[held[seq_of], :, row_of] = there[seq_of, :, row_of].to(pages.dtype).view(torch.uint8)
            x = (x.float() / _power(exp)[at][:, :, None]).to(pages.dtype)
        pages.view(torch.uint8 if pages.element_size() == 1 else torch.int16)[at, :, row] = x.view(
            torch.uint8 if pages.element_size() == 1 else torch.int16)
    return q


def _values(pages, exp, at):
    """Pages at [...] as 32-bit values."""
    x = pages[at].float()
    return x if exp is None or pages.dtype != torch.float8_e4m3fn else x * _power(exp[at])[..., None, None]


def _gated(s, o):
    if s["case"]["gate"]:
        t, hq = o.shape[:2]
        o = o * torch.sigmoid(s["q_gate"].view(t, hq, 2 * D)[..., D:].float())
    return o.flatten(1).to(torch.bfloat16)


def _attend(s):
    b, h, n = s["seqs"], s["heads"], s["most"]
    t = s["q"].shape[0]
    at = s["table"].long()
    k = _values(s["k_pages"], s["k_exp"], at).transpose(1, 2).flatten(2, 3)            # [b, h, keys, D]
    v = _values(s["v_pages"], s["v_exp"], at).transpose(1, 2).flatten(2, 3)
    seq, pos = _slots(s)
    col = torch.arange(t, device=seq.device) - s["cu"][seq]
    q = torch.zeros(b, n, h * GROUP, D, device=seq.device)
    q[seq, col] = s["q"].float()
    last = torch.full((b, n), -1, dtype=torch.long, device=seq.device)
    last[seq, col] = pos
    q = q.view(b, n, h, GROUP, D).transpose(1, 2).reshape(b, h, n * GROUP, D)
    x = torch.matmul(q, k.transpose(2, 3)).view(b, h, n, GROUP, -1) * 0.0625
    seen = torch.arange(k.shape[2], device=seq.device) <= last[:, None, :, None, None]
    x = torch.where(seen, x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    x = x / x.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(x.view(b, h, n * GROUP, -1), v).view(b, h, n, GROUP, D)
    return _gated(s, o.transpose(1, 2).reshape(b, n, h * GROUP, D)[seq, col])


def _select(s, seq, pos):
    """For each token and KV head the pages to read: the first, the last and those of the highest scores, ties to
    the lower page; ascending, -1 behind the last."""
    h, page, budget = s["heads"], s["page"], s["case"]["budget"]
    t, n = s["q"].shape[0], s["table"].shape[1]
    q = s["q"].view(t, h, GROUP * D).float()
    _, x = torch.frexp(q.abs().amax(-1, keepdim=True))
    q = torch.round(q * torch.exp2(7.0 - x)).clamp(-127, 127).view(t, h, GROUP, D)
    at = s["table"].long()
    bound = s["bounds"][at].float().permute(0, 2, 1, 3, 4)                            # [b, h, n, 2, D]
    b = s["seqs"]
    most, col = s["most"], torch.arange(t, device=seq.device) - s["cu"][seq]
    qs = torch.zeros(b, most, h, GROUP, D, device=seq.device)
    qs[seq, col] = q
    qs = qs.permute(0, 2, 1, 3, 4).reshape(b, h, most * GROUP, D)
    # whole numbers below 2^24: exact in 32 bits whatever the order
    score = torch.matmul(qs.clamp(min=0), bound[:, :, :, 0].transpose(2, 3)) + torch.matmul(
        qs.clamp(max=0), bound[:, :, :, 1].transpose(2, 3))
    score = score.view(b, h, most, GROUP, n).amax(3).transpose(1, 2)[seq, col]        # [t, h, n]
    e = s["k_exp"][at].transpose(1, 2)[seq]
    score = score.double() * torch.exp2(e.double() - 127.0)
    i = torch.arange(n, device=seq.device)
    last = (pos // page)[:, None, None]
    score = torch.where((i < 1) | (i == last), math.inf, score)
    score = torch.where(i <= last, score, -math.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :budget]
    best = torch.where(best <= last, best, n)
    best = torch.sort(torch.nn.functional.pad(best, (0, budget - best.shape[-1]), value=n), -1)[0]
    return torch.where(best < n, best, -1).to(torch.int32)


def _sparse(s):
    h, page = s["heads"], s["page"]
    seq, pos = _slots(s)
    picked = _select(s, seq, pos)
    t, _, budget = picked.shape
    at = s["table"].long()[seq[:, None, None], picked.clamp(min=0).long()]            # [t, h, budget]
    head = torch.arange(h, device=at.device)[None, :, None]

    def rows(pages, exp):
        x = pages[at, head].float()                                                    # [t, h, budget, page, D]
        if pages.dtype == torch.float8_e4m3fn:
            x = x * _power(exp[at, head])[..., None, None]
        return x.flatten(2, 3)

    key = picked.long()[..., None] * page + torch.arange(page, device=at.device)
    seen = ((picked >= 0)[..., None] & (key <= pos[:, None, None, None])).flatten(2)[:, :, None]
    q = s["q"].float().view(t, h, GROUP, D)
    x = torch.matmul(q, rows(s["k_pages"], s["k_exp"]).transpose(2, 3)) * 0.0625
    x = torch.where(seen, x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    o = torch.matmul(x, rows(s["v_pages"], s["v_exp"]))
    return picked, _gated(s, o.reshape(t, h * GROUP, D))


def run(s):
    op = s["case"]["op"]
    if own:
        pa, cache = s["pa"], s["cache"]
        where = (s["table"], s["cu"], s["lens"])
        gate = s["q_gate"] if op != "append" and s["case"]["gate"] else None
        if op == "append":
            q = pa.paged_append(s["q_gate"], s["k"], s["v"], s["q_norm"], s["k_norm"], (s["cos"], s["sin"]), cache, *where)
        elif op == "attend":
            return pa.paged_attention(s["q"], cache, *where, q_gate=gate)
        else:
            picked = pa.select_pages(s["q"], cache, *where, budget=s["case"]["budget"], sink_pages=1, recent_pages=1)
            return picked, pa.sparse_paged_attention(s["q"], cache, *where, picked, q_gate=gate)
    elif op == "append":
        q = _append(s)
    else:
        return _attend(s) if op == "attend" else _sparse(s)
    return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"], "k_exp": s["k_exp"], "v_exp": s["v_exp"],
            "bounds": s["bounds"]}


# ------------------------------------------------------------ in 64 bits

def _exact_row(x, w, c, s):
    """One head's rows: the norm, rounded to bf16 as the operator has it, and the rotation."""
    x = x.double()
    y = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * (w.double() + 1.0)
    y = y.to(torch.bfloat16).double()
    z = y.clone()
    z[..., :32] = y[..., :32] * c - y[..., 32:64] * s
    z[..., 32:64] = y[..., 32:64] * c + y[..., :32] * s
    return z.to(torch.bfloat16).double()


def _exact_append(s):
    h, page = s["heads"], s["page"]
    lens, cu, table = s["lens"].tolist(), s["cu"].tolist(), s["table"].tolist()
    t = s["qkv"].shape[0]
    q = torch.empty(t, h * GROUP, D, dtype=torch.float64, device=s["qkv"].device)
    out = {}
    for name in ("k", "v"):
        exp = s[name + "_exp"] if s["case"]["cache"] == "e4m3" else None
        out[name] = (s[name + "_pages"].to(torch.float64), None if exp is None else exp.double())
    for i in range(s["seqs"]):
        a, b = cu[i], cu[i + 1]
        p0 = lens[i] - (b - a)
        c, sn = s["cos"][p0:lens[i], None].double(), s["sin"][p0:lens[i], None].double()
        q[a:b] = _exact_row(s["q_gate"][a:b].reshape(b - a, h * GROUP, 2, D)[:, :, 0], s["q_norm"], c, sn)
        rows = {"k": _exact_row(s["k"][a:b].reshape(b - a, h, D), s["k_norm"], c, sn),
                "v": s["v"][a:b].reshape(b - a, h, D).double()}
        for name, x in rows.items():
            pages, exp = out[name]
            for j in range(p0 // page, (lens[i] - 1) // page + 1):
                lo, hi = max(p0, j * page), min(lens[i], (j + 1) * page)
                r0, r1, at = lo - j * page, hi - j * page, table[i][j]
                y = x[lo - p0:hi - p0].transpose(0, 1)                                 # [h, rows, D]
                if exp is not None:
                    need = torch.ceil(torch.log2(y.abs().amax((1, 2)) / 448.0)) + 127.0
                    need = need.clamp(min=LOWEST)
                    if r0:
                        need = torch.maximum(need, exp[at])
                        old = pages[at, :, :r0] * torch.exp2(exp[at] - need)[:, None, None]
                        pages[at, :, :r0] = old.float().to(torch.float8_e4m3fn).double()
                    exp[at] = need
                    y = (y / torch.exp2(need - 127.0)[:, None, None]).float().to(torch.float8_e4m3fn).double()
                pages[at, :, r0:r1] = y
    return {"q": q, "k_pages": out["k"][0], "v_pages": out["v"][0], "k_exp": None, "v_exp": None, "bounds": None}


def _exact_softmax(q, k, v, seen):
    """q [8, D], k and v [keys, D] or with leading axes, in 64 bits."""
    x = (q @ k.transpose(-1, -2)) / 16.0
    x = x.masked_fill(~seen, -math.inf).softmax(-1)
    return x @ v


def _exact_pages(s, name, at, j):
    x = s[name + "_pages"][at, j].double()
    if s["case"]["cache"] == "e4m3":
        x = x * torch.pow(2.0, s[name + "_exp"][at, j].double() - 127.0)[:, None, None]
    return x.reshape(-1, D)


def _exact_attend(s):
    h, t = s["heads"], s["q"].shape[0]
    out = torch.empty(t, h * GROUP, D, dtype=torch.float64, device=s["q"].device)
    lens, cu = s["lens"].tolist(), s["cu"].tolist()
    for i in range(s["seqs"]):
        at = s["table"][i, :-(-lens[i] // s["page"])].long()
        for j in range(h):
            k, v = (_exact_pages(s, x, at, j)[:lens[i]] for x in ("k", "v"))
            for a in range(cu[i], cu[i + 1], 128):
                z = min(a + 128, cu[i + 1])
                last = lens[i] - (cu[i + 1] - torch.arange(a, z, device=k.device))
                seen = torch.arange(lens[i], device=k.device) <= last[:, None]
                q = s["q"][a:z, j * GROUP:(j + 1) * GROUP].double()
                out[a:z, j * GROUP:(j + 1) * GROUP] = _exact_softmax(q.transpose(0, 1), k, v, seen).transpose(0, 1)
    return out


def _exact_pick(s, i, j, a, pos):
    """The pages of token a (position pos of sequence i) for KV head j."""
    page, budget, n = s["page"], s["case"]["budget"], pos // s["page"] + 1
    if n <= budget:
        return list(range(n))
    at = s["table"][i, :n].long()
    q = s["q"][a, j * GROUP:(j + 1) * GROUP].double()
    q = torch.round(q / 2.0 ** (math.floor(math.log2(q.abs().max().item())) - 6)).clamp(-127, 127)
    b = s["bounds"][at, j].double()                                                    # [n, 2, D]
    x = torch.maximum(q[:, None] * b[None, :, 0], q[:, None] * b[None, :, 1]).sum(-1).amax(0)
    x = (x * torch.pow(2.0, s["k_exp"][at, j].double())).tolist()
    rest = sorted(range(1, n - 1), key=lambda p: (-x[p], p))[:budget - 2]
    return sorted([0, n - 1] + rest)[:budget]


def _exact_sparse(s):
    h, t, page, budget = s["heads"], s["q"].shape[0], s["page"], s["case"]["budget"]
    out = torch.empty(t, h * GROUP, D, dtype=torch.float64, device=s["q"].device)
    picked = torch.full((t, h, budget), -1, dtype=torch.int32)
    lens, cu = s["lens"].tolist(), s["cu"].tolist()
    for i in range(s["seqs"]):
        for a in range(cu[i], cu[i + 1]):
            pos = lens[i] - (cu[i + 1] - a)
            for j in range(h):
                mine = _exact_pick(s, i, j, a, pos)
                picked[a, j, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
                mine = torch.tensor(mine, device=out.device)
                at = s["table"][i].long()[mine]
                key = (mine[:, None] * page + torch.arange(page, device=out.device)).flatten()
                out[a, j * GROUP:(j + 1) * GROUP] = _exact_softmax(
                    s["q"][a, j * GROUP:(j + 1) * GROUP].double(), _exact_pages(s, "k", at, j),
                    _exact_pages(s, "v", at, j), key <= pos)
    return picked, out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s)
    t = sum(_lengths(case)[1])
    if case["op"] == "sparse":
        if t * case["heads"] > 4000:
            return None          # a selection of its own for every token and head: too long
        picked, o = _exact_sparse(s)
    else:
        o = _exact_attend(s)
    if case["gate"]:
        o = o / (1.0 + torch.exp(-s["q_gate"].unflatten(1, (-1, 2, D))[:, :, 1].double()))
    return (picked.to(o.device), o.flatten(1)) if case["op"] == "sparse" else o.flatten(1)
