"""Attention over a paged KV cache: appending, dense and sparse reads.

No counterpart in the reference, whose caches are dense and hold one sequence
(``full_attention_kv_caches``, four_layer_mini_engine.py:4190).  A pool of pages
serves a ragged batch: prompts, drafted tokens and single tokens of any number
of sequences go through the same calls.  Pages are bf16, or e4m3 with a
power-of-two scale for each page and KV head.

The batch of a call is three int32 GPU tensors, read when the launch runs:
``page_table`` [seqs, width], ``cu_tokens`` [seqs + 1] (row offsets of the call)
and ``seq_lens`` [seqs] (lengths with the call's tokens): the last row of
sequence i is at position ``seq_lens[i] - 1``.  Rows behind the last sequence
are left as they were.  All arithmetic runs in ``libqwen36_attn.so``.
"""
from __future__ import annotations

import torch

from . import _lib
from ._tensors import ptr, require
from .full_attention import HEAD_DIM, HKV, HQ, MAX_TOKENS

GROUP = HQ // HKV
PAGE_TOKENS = (16, 32, 64, 128)
MAX_LISTED = 1024
# torch.cuda.current_stream(device).cuda_stream without the Stream object (1.9 us a call)
_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch.cuda.current_device
_WEIGHT = (HEAD_DIM,)
_TYPES = {torch.bfloat16: 0, torch.float8_e4m3fn: 1}
_FIXED = frozenset(("k_pages", "v_pages", "k_exp", "v_exp", "bounds", "num_pages", "kv_heads",
                    "page_tokens", "heads", "device", "_index", "_max_width", "_args"))


class PagedKVCache:
    """A pool of KV pages of one layer: ``k_pages``, ``v_pages`` [num_pages,
    kv_heads, page_tokens, 256] in bf16 or e4m3; for e4m3 ``k_exp``, ``v_exp``
    [num_pages, kv_heads] uint8, the scale of a page and head being
    2^(byte - 127); ``bounds`` [num_pages, kv_heads, 2, 256] int8 where pages are
    to be selected: each channel's largest and smallest key in steps of
    4 * 2^(k_exp - 127).  ``kv_heads`` is 2, or a tensor-parallel share.  The
    attributes are fixed; the tensors' contents are the caller's to change."""

    def __init__(self, num_pages: int, page_tokens: int, device, dtype=torch.float8_e4m3fn,
                 kv_heads: int = HKV, bounds: bool = False) -> None:
        if dtype not in _TYPES:
            raise ValueError("pages must be torch.bfloat16 or torch.float8_e4m3fn")
        if num_pages < 1 or page_tokens not in PAGE_TOKENS or not 1 <= kv_heads <= 16:
            raise ValueError("pages hold 16, 32, 64 or 128 tokens of 1 to 16 KV heads")
        shape = (num_pages, kv_heads, page_tokens, HEAD_DIM)
        fp8 = dtype == torch.float8_e4m3fn

        def byte(*more):
            return torch.zeros(num_pages, kv_heads, *more, dtype=torch.uint8, device=device)
        self._set(torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) if fp8
                  else torch.zeros(shape, dtype=dtype, device=device),
                  torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) if fp8
                  else torch.zeros(shape, dtype=dtype, device=device),
                  byte() if fp8 or bounds else None, byte() if fp8 else None,
                  byte(2, HEAD_DIM).view(torch.int8) if bounds else None)

    @classmethod
    def of(cls, k_pages: torch.Tensor, v_pages: torch.Tensor, k_exp: torch.Tensor | None = None,
           v_exp: torch.Tensor | None = None, bounds: torch.Tensor | None = None) -> "PagedKVCache":
        """A cache over the caller's tensors (pages may be apart: only their
        [kv_heads, page_tokens, 256] has to be contiguous)."""
        self = cls.__new__(cls)
        self._set(k_pages, v_pages, k_exp, v_exp, bounds)
        return self

    def _set(self, k_pages, v_pages, k_exp, v_exp, bounds) -> None:
        if not isinstance(k_pages, torch.Tensor) or k_pages.dtype not in _TYPES:
            raise ValueError("pages must be torch.bfloat16 or torch.float8_e4m3fn")
        for name, t in (("k_pages", k_pages), ("v_pages", v_pages)):
            require(t, name, k_pages.dtype, contiguous=False)
            if t.dim() != 4 or t.shape != k_pages.shape or t.shape[3] != HEAD_DIM:
                raise ValueError(f"{name} must be [num_pages, kv_heads, page_tokens, 256]")
            if t.stride()[1:] != (t.shape[2] * HEAD_DIM, HEAD_DIM, 1):
                raise ValueError(f"{name}: a page must be contiguous")
        n, heads, page, _ = k_pages.shape
        if n < 1 or page not in PAGE_TOKENS or not 1 <= heads <= 16:
            raise ValueError("pages hold 16, 32, 64 or 128 tokens of 1 to 16 KV heads")
        fp8 = k_pages.dtype == torch.float8_e4m3fn
        if fp8 and (k_exp is None or v_exp is None):
            raise ValueError("e4m3 pages need k_exp and v_exp")
        if bounds is not None and k_exp is None:
            raise ValueError("bounds need k_exp")
        for name, t in (("k_exp", k_exp), ("v_exp", v_exp)):
            if t is not None:
                require(t, name, torch.uint8, shape=(n, heads))
        if bounds is not None:
            require(bounds, "bounds", torch.int8, shape=(n, heads, 2, HEAD_DIM))
        for t in (v_pages, k_exp, v_exp, bounds):
            if t is not None and t.device != k_pages.device:
                raise ValueError("the cache's tensors must be on one device")
        stride = [t.stride(0) if n > 1 else heads * page * HEAD_DIM for t in (k_pages, v_pages)]
        self.__dict__.update(
            k_pages=k_pages, v_pages=v_pages, k_exp=k_exp, v_exp=v_exp, bounds=bounds,
            num_pages=n, kv_heads=heads, page_tokens=page, heads=heads * GROUP,
            device=k_pages.device, _index=k_pages.get_device(), _max_width=(MAX_TOKENS + 127) // page,
            _args=_lib.PagedCacheArgs(ptr(k_pages), ptr(v_pages), ptr(k_exp),
                                      ptr(v_exp) if fp8 else None, ptr(bounds), stride[0],
                                      stride[1], n, page, heads, _TYPES[k_pages.dtype]))

    # The calls use the addresses and sizes of ``_args``: another tensor in an
    # attribute's place would go unseen, and the old one's memory would be reused.
    def __setattr__(self, name: str, value) -> None:
        if name in _FIXED:
            raise AttributeError(f"{name}: a cache's tensors and sizes are fixed (PagedKVCache.of makes one "
                                 "over other tensors)")
        object.__setattr__(self, name, value)

    def __delattr__(self, name: str) -> None:
        if name in _FIXED:
            raise AttributeError(f"{name}: a cache's tensors and sizes are fixed")
        object.__delattr__(self, name)

    def values(self) -> tuple[torch.Tensor, torch.Tensor]:
        """K and V pages as the bf16 values that they hold (e4m3 values times a
        power of two are bf16 values)."""
        if self.k_pages.dtype == torch.bfloat16:
            return self.k_pages, self.v_pages
        return tuple((p.float() * torch.exp2(e.float() - 127.0)[:, :, None, None]).to(torch.bfloat16)
                     for p, e in ((self.k_pages, self.k_exp), (self.v_pages, self.v_exp)))


_BATCH = "a batch is page_table [seqs, width], contiguous cu_tokens [seqs + 1] and seq_lens [seqs]"


def _batch(cache: PagedKVCache, tokens: int, page_table, cu_tokens, seq_lens) -> _lib.PagedBatchArgs:
    index, kind = cache._index, torch.int32
    if not (isinstance(page_table, torch.Tensor) and isinstance(cu_tokens, torch.Tensor)
            and isinstance(seq_lens, torch.Tensor) and page_table.dtype is kind
            and cu_tokens.dtype is kind and seq_lens.dtype is kind
            and page_table.get_device() == index and cu_tokens.get_device() == index
            and seq_lens.get_device() == index):
        raise ValueError("page_table, cu_tokens and seq_lens must be int32 tensors on the cache's device")
    if page_table.dim() != 2 or not cu_tokens.is_contiguous() or not seq_lens.is_contiguous():
        raise ValueError(_BATCH)
    rows, width = page_table.shape
    if seq_lens.shape != (rows,) or cu_tokens.shape != (rows + 1,) or rows < 1 or width < 1:
        raise ValueError(_BATCH)
    stride, inner = page_table.stride()
    if width > 1 and inner != 1 or rows > 1 and stride < width:
        raise ValueError("page_table must have contiguous rows that do not overlap")
    if width > cache._max_width:
        raise ValueError(f"a sequence has at most {MAX_TOKENS} tokens")
    if not 0 < tokens <= MAX_TOKENS or rows > 65536:
        raise ValueError(f"a call has 1 to {MAX_TOKENS} rows of at most 65536 sequences")
    return _lib.PagedBatchArgs(page_table.data_ptr(), cu_tokens.data_ptr(), seq_lens.data_ptr(),
                               stride if rows > 1 else width, width, rows, tokens)


def _rows(t, name: str, rows: int, width: int, index: int) -> tuple[int, int]:
    """Address and row stride of a bf16 [rows, width] tensor with unit inner stride."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.bfloat16 or t.get_device() != index:
        raise ValueError(f"{name} must be a bf16 tensor on the cache's device")
    if t.shape != (rows, width):
        raise ValueError(f"{name} must be [{rows}, {width}]")
    stride, inner = t.stride()
    if rows == 1:
        stride = width
    at = t.data_ptr()
    if inner != 1 or not width <= stride < 1 << 32 or (at | 2 * stride) & 7:
        raise ValueError(f"{name} must have unit inner stride and 8-byte aligned rows that do not overlap")
    return at, stride


def _queries(q, cache: PagedKVCache) -> int:
    if not isinstance(q, torch.Tensor) or q.dtype is not torch.bfloat16 or q.get_device() != cache._index:
        raise ValueError("q must be a bf16 tensor on the cache's device")
    t = q.shape[0] if q.dim() == 3 else 0
    if q.shape != (t, cache.heads, HEAD_DIM) or not q.is_contiguous() or q.data_ptr() & 15:
        raise ValueError(f"q must be contiguous [T, {cache.heads}, 256], 16-byte aligned")
    return t


def _out(out, shape, dtype, device) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if not isinstance(out, torch.Tensor) or out.dtype != dtype or out.device != device \
            or tuple(out.shape) != shape or not out.is_contiguous() or out.data_ptr() % 8:
        raise ValueError(f"out must be contiguous {dtype} {list(shape)} on the cache's device")
    return out


def _call(cache: PagedKVCache, name: str, *args) -> None:
    """The entry point on the cache's device and its current stream."""
    fn = getattr(_lib._LIB or _lib.load(), name)
    index = cache._index
    if _current_device() == index:
        status = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _stream(index))
    if status != 0:
        raise _lib.KernelError(f"{name} failed: hip_status={status}")


# The workspaces below are allocated per call: calls on several streams, and
# graphs captured apart, then never share one.

def paged_append(q_gate: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_norm: torch.Tensor,
                 k_norm: torch.Tensor, rope: tuple[torch.Tensor, torch.Tensor],
                 cache: PagedKVCache, page_table: torch.Tensor, cu_tokens: torch.Tensor,
                 seq_lens: torch.Tensor, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Head norm and rotation of the new rows, K (normed, rotated) and raw V
    into their pages: ``full_attention.head_norm_rope_kv_write`` for a paged
    cache, with its arithmetic.  q_gate [T, heads * 512] ([q | gate] of each
    head), k, v [T, kv_heads * 256], unit inner strides; ``rope``: fp32 (cos,
    sin) [positions, 32], e.g. ``full_attention.rotary_table(capacity, 0,
    device)``.  An e4m3 page's scale fits its largest value and grows with it;
    a page that gets rows must belong to one sequence.  Returns q [T, heads,
    256] bf16.  A sequence longer than ``rope`` or than the page table has no tokens:
    neither its pages nor its q are written (as rows of negative position and rows
    behind the last sequence).  The calls that attend do not know ``rope``; give them
    such a sequence with a length of 0."""
    dev, index = cache.device, cache._index
    t = q_gate.shape[0] if isinstance(q_gate, torch.Tensor) and q_gate.dim() == 2 else 0
    batch = _batch(cache, t, page_table, cu_tokens, seq_lens)
    qp, qs = _rows(q_gate, "q_gate", t, 2 * cache.heads * HEAD_DIM, index)
    kp, ks = _rows(k, "k", t, cache.kv_heads * HEAD_DIM, index)
    vp, vs = _rows(v, "v", t, cache.kv_heads * HEAD_DIM, index)
    cos, sin = rope
    if not (isinstance(q_norm, torch.Tensor) and isinstance(k_norm, torch.Tensor)
            and q_norm.dtype is k_norm.dtype is torch.bfloat16 and q_norm.get_device() == index
            and k_norm.get_device() == index and q_norm.shape == k_norm.shape == _WEIGHT
            and q_norm.is_contiguous() and k_norm.is_contiguous()):
        raise ValueError("q_norm and k_norm must be contiguous bf16 [256] on the cache's device")
    if not (isinstance(cos, torch.Tensor) and isinstance(sin, torch.Tensor)
            and cos.dtype is sin.dtype is torch.float32 and cos.get_device() == index
            and sin.get_device() == index and cos.dim() == 2 and cos.is_contiguous()
            and sin.is_contiguous()):
        raise ValueError("rope must be two contiguous fp32 tensors on the cache's device")
    positions, pairs = cos.shape
    cp, sp = cos.data_ptr(), sin.data_ptr()
    if pairs != 32 or positions < 1 or sin.shape != (positions, 32) or (cp | sp) & 15:
        raise ValueError("rope must be two 16-byte aligned [positions, 32]")
    q_out = _out(q_out, (t, cache.heads, HEAD_DIM), torch.bfloat16, dev)
    _call(cache, "qwen36_paged_append", qp, qs, kp, ks, vp, vs, q_norm.data_ptr(), k_norm.data_ptr(),
          cp, sp, positions, cache._args, batch, q_out.data_ptr())
    return q_out


def _gate(q_gate, t: int, cache: PagedKVCache) -> tuple[int | None, int]:
    if q_gate is None:
        return None, 0
    return _rows(q_gate, "q_gate", t, 2 * cache.heads * HEAD_DIM, cache._index)


def paged_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor,
                    cu_tokens: torch.Tensor, seq_lens: torch.Tensor,
                    q_gate: torch.Tensor | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal GQA attention of each row over its sequence's positions up to its
    own, scale 1/16; the rows' own keys must have been appended.  q [T, heads,
    256] bf16 as ``paged_append`` returns it.  ``q_gate`` (its input rows): the
    output is ``attention * sigmoid(gate)``, rounded once.  Rows that see
    nothing are zeros.  The workspace of a call grows with its rows (two KV heads:
    259 MiB for 8,192, 4.2 GiB for 262,144).  Returns bf16 [T, heads * 256]."""
    dev = cache.device
    t = _queries(q, cache)
    batch = _batch(cache, t, page_table, cu_tokens, seq_lens)
    gate, gs = _gate(q_gate, t, cache)
    out = _out(out, (t, cache.heads * HEAD_DIM), torch.bfloat16, dev)
    nb = _lib.load().qwen36_paged_attention_workspace_bytes(cache._args, batch)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)
    _call(cache, "qwen36_paged_attention", q.data_ptr(), cache._args, batch, gate, gs, out.data_ptr(),
          ws.data_ptr(), nb)
    return out


def select_pages(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor,
                 cu_tokens: torch.Tensor, seq_lens: torch.Tensor, budget: int,
                 sink_pages: int = 1, recent_pages: int = 1,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """For each row and KV head the pages that a sparse attention reads: int32
    [T, kv_heads, budget] logical page indices, ascending, -1 behind the last.
    Rows of at most ``budget`` pages take all; others the first
    ``sink_pages``, the last ``recent_pages`` and those of the highest scores,
    estimates of the page's largest q.k from its bounds in whole numbers (so the
    choice is exact; ties to the lower page).  The cache needs ``bounds``."""
    dev = cache.device
    t = _queries(q, cache)
    batch = _batch(cache, t, page_table, cu_tokens, seq_lens)
    if cache.bounds is None:
        raise ValueError("the cache has no bounds")
    if not (sink_pages >= 0 and recent_pages >= 1 and sink_pages + recent_pages <= budget <= MAX_LISTED):
        raise ValueError(f"sink_pages + recent_pages (>= 1) <= budget <= {MAX_LISTED}")
    out = _out(out, (t, cache.kv_heads, budget), torch.int32, dev)
    nb = _lib.load().qwen36_paged_select_workspace_bytes(cache._args, batch)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)
    _call(cache, "qwen36_paged_select", q.data_ptr(), cache._args, batch, budget, sink_pages,
          recent_pages, out.data_ptr(), ws.data_ptr(), nb)
    return out


def sparse_paged_attention(q: torch.Tensor, cache: PagedKVCache, page_table: torch.Tensor,
                           cu_tokens: torch.Tensor, seq_lens: torch.Tensor, pages: torch.Tensor,
                           q_gate: torch.Tensor | None = None,
                           out: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_attention`` over the positions up to the row's own in the listed
    pages only.  pages: int32 [T, kv_heads, listed] logical page indices, any
    order, listed <= 1024; an index outside the row's pages lists nothing, a
    page listed twice counts twice."""
    dev = cache.device
    t = _queries(q, cache)
    batch = _batch(cache, t, page_table, cu_tokens, seq_lens)
    if not isinstance(pages, torch.Tensor) or pages.dtype != torch.int32 or pages.get_device() != cache._index:
        raise ValueError("pages must be an int32 tensor on the cache's device")
    if (pages.dim() != 3 or pages.shape[:2] != (t, cache.kv_heads) or not pages.is_contiguous()
            or not 1 <= pages.shape[2] <= MAX_LISTED):
        raise ValueError(f"pages must be contiguous [T, {cache.kv_heads}, 1..{MAX_LISTED}]")
    gate, gs = _gate(q_gate, t, cache)
    out = _out(out, (t, cache.heads * HEAD_DIM), torch.bfloat16, dev)
    listed = pages.shape[2]
    nb = _lib.load().qwen36_paged_sparse_attention_workspace_bytes(cache._args, batch, listed)
    ws = torch.empty(nb, dtype=torch.uint8, device=dev)
    _call(cache, "qwen36_paged_sparse_attention", q.data_ptr(), cache._args, batch, pages.data_ptr(),
          listed, gate, gs, out.data_ptr(), ws.data_ptr(), nb)
    return out


class PagedFullAttentionLayer:
    """One gated GQA layer over a paged cache, ``full_attention.FullAttentionLayer``
    for a ragged batch: the projections, the append, the attention (over selected
    pages if ``budget`` is given) with the output gate, and o_proj.  ``weights`` as
    there, for all of the model's heads; ``rope``: fp32 (cos, sin) tables that reach the
    longest sequence; ``adapters``: an ``adapters.LayerAdapters`` of q | k | v and o_proj.
    A sequence longer than they or the page table has no tokens: its
    rows are zeros and its pages stay as they are."""

    def __init__(self, weights: dict, cache: PagedKVCache,
                 rope: tuple[torch.Tensor, torch.Tensor], budget: int | None = None,
                 sink_pages: int = 1, recent_pages: int = 1, adapters=None) -> None:
        if cache.kv_heads != HKV:
            raise ValueError(f"the layer has {HKV} KV heads")
        if budget is not None and cache.bounds is None:
            raise ValueError("the cache has no bounds")
        from .projections import FusedProjection
        self.w, self.cache, self.rope = weights, cache, rope
        self.budget, self.sink_pages, self.recent_pages = budget, sink_pages, recent_pages
        self._qkv = FusedProjection(weights["q_proj"], weights["k_proj"], weights["v_proj"])
        if adapters is not None:
            adapters.check(self._qkv.splits, [weights["o_proj"].shape[0]], self._qkv.w.shape[1], weights["o_proj"].shape[1])
        self._into, self._out = (None, None) if adapters is None else (adapters.into, adapters.out)

    def forward(self, inp: torch.Tensor, page_table: torch.Tensor, cu_tokens: torch.Tensor,
                seq_lens: torch.Tensor, adapter_batch=None) -> torch.Tensor:
        """inp [T, 2048]: the new rows of the batch's sequences.  ``adapter_batch``: the
        ``adapters.AdapterBatch`` of these rows (None: no request has an adapter).  Returns
        [T, 2048]."""
        from .adapters import project
        w = self.w
        q_gate, k, v = self._qkv.split_rows(project(inp, self._qkv.w, self._into, adapter_batch))
        where = (page_table, cu_tokens, seq_lens)
        q = paged_append(q_gate, k, v, w["q_norm"], w["k_norm"], self.rope, self.cache, *where)
        positions = self.rope[0].shape[0]
        if min(page_table.shape[1] * self.cache.page_tokens, MAX_TOKENS) > positions:
            # a longer sequence has no tokens for the append, so neither for the attention
            where = (page_table, cu_tokens, seq_lens.masked_fill(seq_lens > positions, 0))
        if self.budget is None:
            attn = paged_attention(q, self.cache, *where, q_gate=q_gate)
        else:
            pages = select_pages(q, self.cache, *where, self.budget, self.sink_pages,
                                 self.recent_pages)
            attn = sparse_paged_attention(q, self.cache, *where, pages, q_gate=q_gate)
        return project(attn, w["o_proj"], self._out, adapter_batch)
