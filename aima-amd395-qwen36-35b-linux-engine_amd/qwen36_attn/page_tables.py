"""Who holds which page of a ``PagedKVCache``: giving rows up, forking and growing
them, and moving the held pages together.

No counterpart in the reference, whose caches are dense.  A server keeps one table
for all its sequences, ``page_table`` int32 [rows, width] with ``seq_lens`` int32
[rows] (0: an empty row), and ``refs`` int32 [num_pages]: how many table entries name
each page (0: free), all on the GPU and shared by the caches of every layer.  The
calls read and write them on the current stream, so that nothing waits for the host
and captured calls follow them.  They take a number for every row (``keep``,
``parents``, ``add``), so that no row can be named twice.  A row whose length is
negative or above what its table holds is left as it is, and a page id outside the
pool holds nothing.

A turn of a server: ``trim`` the rows that end (or whose drafts were refused),
``fork`` rows whose prompt is shared, ``extend`` the rows that get tokens, then
``paged_append`` and the attention over the rows of the batch.  A page that several
rows hold is never written: ``extend`` gives a row that would write one a copy of it.
A row that it could not serve has its old length and pages, so that tokens of it in the
turn's batch would be written over its last ones, in pages that others may hold: such a
row has no tokens there (``cu_tokens``) until it is served.
"""
from __future__ import annotations

import torch

from . import _lib
from ._tensors import launch
from .full_attention import MAX_TOKENS
from .paged_attention import PAGE_TOKENS, PagedKVCache


def new_refs(num_pages: int, device) -> torch.Tensor:
    """Counts of a pool whose pages are all free."""
    return torch.zeros(num_pages, dtype=torch.int32, device=device)


def _vector(t, name: str, index: int, n: int) -> int:
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.get_device() != index \
            or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor [{n}] on the device of refs")
    return t.data_ptr()


def _table(t, name: str, index: int) -> tuple[int, int, int]:
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.get_device() != index or t.dim() != 2:
        raise ValueError(f"{name} must be an int32 tensor [rows, width] on the device of refs")
    rows, width = t.shape
    stride, inner = t.stride()
    if rows < 1 or width < 1 or rows > 65536 or width > 1 and inner != 1 or rows > 1 and stride < width:
        raise ValueError(f"{name} must have contiguous rows that do not overlap, 65536 at most")
    return rows, width, stride if rows > 1 else width


def _args(refs, page_table, seq_lens, page_tokens: int) -> tuple[int, _lib.PageTablesArgs]:
    if not isinstance(refs, torch.Tensor) or refs.dtype is not torch.int32 or not refs.is_cuda \
            or refs.dim() != 1 or not refs.is_contiguous() or refs.shape[0] < 1:
        raise ValueError("refs must be a contiguous int32 GPU tensor [num_pages]")
    index = refs.get_device()
    rows, width, stride = _table(page_table, "page_table", index)
    lens = _vector(seq_lens, "seq_lens", index, rows)
    if page_tokens not in PAGE_TOKENS:
        raise ValueError("pages hold 16, 32, 64 or 128 tokens")
    if width > (MAX_TOKENS + 127) // page_tokens:
        raise ValueError(f"a sequence has at most {MAX_TOKENS} tokens")
    return index, _lib.PageTablesArgs(refs.data_ptr(), page_table.data_ptr(), lens, stride, refs.shape[0],
                                      page_tokens, width, rows)


def _caches(caches, refs):
    """The caches as the C calls take them, and their page size."""
    caches = list(caches)
    if not caches or not all(isinstance(c, PagedKVCache) for c in caches):
        raise ValueError("caches must be one or more PagedKVCache")
    page, pages = caches[0].page_tokens, refs.shape[0] if isinstance(refs, torch.Tensor) and refs.dim() else 0
    seen = set()
    for c in caches:
        if c.page_tokens != page or c.num_pages != pages or c.device != refs.device:
            raise ValueError("the caches must have the pages that refs counts, of one size, on its device")
        seen.add(c._args.k_pages)
        seen.add(c._args.v_pages)
    if len(seen) < 2 * len(caches):
        raise ValueError("a cache is listed twice")
    return (_lib.PagedCacheArgs * len(caches))(*[c._args for c in caches]), page


def trim(refs: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, keep: torch.Tensor,
         page_tokens: int) -> None:
    """Row i keeps its first ``keep[i]`` tokens (all, if it has fewer; 0 gives the row
    up).  Pages without tokens leave the row (entries of -1) and lose a count."""
    index, t = _args(refs, page_table, seq_lens, page_tokens)
    launch(index, "qwen36_pages_trim", t, _vector(keep, "keep", index, t.rows))


def fork(refs: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, parents: torch.Tensor,
         page_tokens: int) -> None:
    """Row i becomes a fork of row ``parents[i]`` (-1: it stays): its tokens and pages,
    each of which gains a count.  A row that is not empty stays, and so does a child of
    a row that is a child of the same call.  ``ragged_deltanet.fork_states`` copies the
    states in slots by such numbers, but slots have no lengths: where a row stays because
    it is not empty, or its parent is, its slot is copied over all the same.  One vector
    serves both if it names no such row."""
    index, t = _args(refs, page_table, seq_lens, page_tokens)
    launch(index, "qwen36_pages_fork", t, _vector(parents, "parents", index, t.rows))


def extend(refs: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, add: torch.Tensor,
           caches) -> torch.Tensor:
    """Row i grows by ``add[i]`` tokens (none, if not positive): pages for them, and a
    copy of its last page, in every one of ``caches`` (the layers' PagedKVCache), if that
    is not full and other rows hold it too.  The lowest free pages go to the rows in
    their order, to each row all that it needs or nothing: once the pool cannot serve a
    row, it serves no later one that needs pages.  Returns int32 [rows]: 0 where a row
    could not grow (its length is unchanged), else 1."""
    args, page = _caches(caches, refs)
    index, t = _args(refs, page_table, seq_lens, page)
    ap = _vector(add, "add", index, t.rows)
    granted = torch.empty(t.rows, dtype=torch.int32, device=refs.device)
    nb = (_lib._LIB or _lib.load()).qwen36_pages_extend_workspace_bytes(t)
    ws = torch.empty(nb, dtype=torch.uint8, device=refs.device)
    launch(index, "qwen36_pages_extend", t, ap, granted.data_ptr(), args, len(args), ws.data_ptr(), nb)
    return granted


def compact(refs: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor, caches,
            refs_out: torch.Tensor | None = None,
            table_out: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Moves the held pages together: with n of them, those at n or behind go, in every
    one of ``caches``, to the free pages before n, in ascending order.  Returns the counts
    and the table after it (``refs_out`` and ``table_out``, which may be ``refs`` and
    ``page_table`` themselves); entries behind a row's length come out as -1.  A row whose
    length is negative or above what its table holds keeps all of its entries, which name
    its pages where they are then."""
    args, page = _caches(caches, refs)
    index, t = _args(refs, page_table, seq_lens, page)
    if refs_out is None:
        refs_out = torch.empty_like(refs)
    if table_out is None:
        table_out = torch.empty(page_table.shape, dtype=torch.int32, device=refs.device)
    rp = _vector(refs_out, "refs_out", index, t.num_pages)
    rows, width, stride = _table(table_out, "table_out", index)
    if (rows, width) != (t.rows, t.table_width):
        raise ValueError("table_out must have the shape of page_table")
    nb = (_lib._LIB or _lib.load()).qwen36_pages_compact_workspace_bytes(t)
    ws = torch.empty(nb, dtype=torch.uint8, device=refs.device)
    launch(index, "qwen36_pages_compact", t, rp, table_out.data_ptr(), stride, args, len(args), ws.data_ptr(), nb)
    return refs_out, table_out
