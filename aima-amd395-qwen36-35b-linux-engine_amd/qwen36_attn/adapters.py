"""Low-rank adapters of many requests beside a shared projection.

No counterpart in the reference.  The projections of a ragged batch are shared
products (``projections.FusedProjection``, ``prefill_gemm.linear``); a request with
an adapter of its own gets ``scale * (x A^T) B^T`` added to its rows, for every slice
of the stacked weights (q | k | v ...) with matrices of its own.  Requests choose
their adapter by a number on the GPU, which the launch that makes an
``AdapterBatch`` reads: a captured step follows new numbers where the batch is
made within the capture.  All arithmetic runs in ``libqwen36_attn.so``.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._tensors import launch
from .full_attention import MAX_TOKENS


class AdapterSet:
    """The adapters of one projection: ``a`` bf16 [adapters, slices, rank, K] and ``b``
    bf16 [adapters, sum(widths), rank], for a projection whose stacked weights are slices
    of ``widths`` rows (1 to 4, multiples of 8) over K inputs (a multiple of 128).
    ``ranks`` int32 [adapters]: each adapter's rank if it is below ``rank`` (a multiple of
    8, 128 at most); what stands behind it in a and b is not used.  ``scales`` fp32
    [adapters], or None: 1.  The tensors' contents are the caller's to change."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, widths, ranks: torch.Tensor | None = None,
                 scales: torch.Tensor | None = None) -> None:
        widths = tuple(int(w) for w in widths)
        for name, t in (("a", a), ("b", b)):
            if not isinstance(t, torch.Tensor) or t.dtype is not torch.bfloat16 or not t.is_cuda \
                    or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"{name} must be a contiguous bf16 GPU tensor, 16-byte aligned")
        if not 1 <= len(widths) <= 4 or any(w < 8 or w % 8 for w in widths) or sum(widths) > 65536:
            raise ValueError("widths must be 1 to 4 multiples of 8, 65536 together at most")
        if a.dim() != 4 or a.shape[1] != len(widths) or b.shape != (a.shape[0], sum(widths), a.shape[2]):
            raise ValueError("a must be [adapters, slices, rank, K] and b [adapters, sum(widths), rank]")
        n, _, rank, k = a.shape
        if not 1 <= n <= 4096 or not 8 <= rank <= 128 or rank % 8 or not 128 <= k <= 16384 or k % 128:
            raise ValueError("1 to 4096 adapters, a rank of 8 to 128 (a multiple of 8), K a multiple of 128")
        for name, t, kind in (("ranks", ranks, torch.int32), ("scales", scales, torch.float32)):
            if t is not None and (not isinstance(t, torch.Tensor) or t.dtype is not kind or t.shape != (n,)
                                  or not t.is_contiguous() or t.device != a.device):
                raise ValueError(f"{name} must be a contiguous {kind} tensor [{n}] on the adapters' device")
        if b.device != a.device:
            raise ValueError("the adapters' tensors must be on one device")
        self._held = a, b, ranks, scales
        self.adapters, self.slices, self.rank, self.k, self.widths, self.total = n, len(widths), rank, k, widths, sum(widths)
        self.device, self._index = a.device, a.get_device()
        self._args = _lib.AdaptersArgs(a.data_ptr(), b.data_ptr(), None if ranks is None else ranks.data_ptr(),
                                       None if scales is None else scales.data_ptr(), n, rank, k, len(widths),
                                       (ctypes.c_uint * 4)(*widths))


class AdapterBatch:
    """The rows of a ragged batch by adapter: made once for all projections of a step.
    ``cu_tokens`` int32 [seqs + 1]: row offsets of the call's ``tokens`` rows (cut to them);
    ``adapter_ids`` int32 [seqs]: each sequence's adapter; one outside [0, ``adapters``)
    means none.  Both are read by a launch on the current stream, here and not again: a
    batch stays what it was when they change, in a graph that was captured over it too.
    Made within a capture, it is made anew by every replay."""

    def __init__(self, cu_tokens: torch.Tensor, adapter_ids: torch.Tensor, tokens: int, adapters: int) -> None:
        for t in (cu_tokens, adapter_ids):
            if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or not t.is_cuda or t.dim() != 1 \
                    or not t.is_contiguous() or t.device != cu_tokens.device:
                raise ValueError("cu_tokens [seqs + 1] and adapter_ids [seqs] must be contiguous int32 tensors on one GPU")
        seqs = adapter_ids.shape[0]
        if cu_tokens.shape[0] != seqs + 1 or not 1 <= seqs <= 65536:
            raise ValueError("a batch is cu_tokens [seqs + 1] and adapter_ids [seqs] of 1 to 65536 sequences")
        if not 0 < tokens <= MAX_TOKENS or not 1 <= adapters <= 4096:
            raise ValueError(f"a call has 1 to {MAX_TOKENS} rows and 1 to 4096 adapters")
        self.seqs, self.tokens, self.adapters, self._index = seqs, tokens, adapters, cu_tokens.get_device()
        self._bytes = _lib.load().qwen36_adapter_plan_bytes(seqs, tokens, adapters)
        self._plan = torch.empty(self._bytes, dtype=torch.uint8, device=cu_tokens.device)
        launch(self._index, "qwen36_adapter_plan", cu_tokens.data_ptr(), adapter_ids.data_ptr(), seqs, tokens, adapters,
               self._plan.data_ptr(), self._bytes)


def _rows(t, name: str, rows: int, width: int, index: int) -> tuple[int, int]:
    """Address and row stride of a bf16 [rows, width] tensor with unit inner stride."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.bfloat16 or t.get_device() != index \
            or t.shape != (rows, width):
        raise ValueError(f"{name} must be bf16 [{rows}, {width}] on the adapters' device")
    stride, inner = t.stride()
    if rows == 1:
        stride = width
    at = t.data_ptr()
    if inner != 1 or stride < width or (at | 2 * stride) & 15:
        raise ValueError(f"{name} must have unit inner stride and 16-byte aligned rows that do not overlap")
    return at, stride


def apply_adapters(y: torch.Tensor, x: torch.Tensor, adapters: AdapterSet, batch: AdapterBatch) -> torch.Tensor:
    """Adds to the rows of y [T, sum(widths)] bf16, the shared projection of x [T, K] bf16,
    what their adapters give: y = bf16(y + scale * (x A^T) B^T), in place; rows without an
    adapter stay as they are.  x A^T is kept to 2^-17 of it, sums are fp32.  Returns y."""
    if batch.adapters != adapters.adapters or batch._index != adapters._index:
        raise ValueError("the batch was made for other adapters")
    index, t = adapters._index, batch.tokens
    xp, xs = _rows(x, "x", t, adapters.k, index)
    yp, ys = _rows(y, "y", t, adapters.total, index)
    nb = (_lib._LIB or _lib.load()).qwen36_adapter_workspace_bytes(adapters._args, batch.seqs, t)
    # allocated per call: calls on several streams, and graphs captured apart, never share one
    ws = torch.empty(nb, dtype=torch.uint8, device=adapters.device)
    launch(index, "qwen36_adapter_apply", xp, xs, yp, ys, adapters._args, batch._plan.data_ptr(), batch._bytes,
           batch.seqs, t, ws.data_ptr(), nb)
    return y


class LayerAdapters:
    """The adapters of a layer's two projections, either of which may be None:
    ``into`` for the stacked one that its input goes through (q with its gate | k | v;
    qkv | z | b | a), ``out`` for its o_proj or out_proj, of as many adapters."""

    def __init__(self, into: AdapterSet | None = None, out: AdapterSet | None = None) -> None:
        if into is None and out is None or into is not None and out is not None and into.adapters != out.adapters:
            raise ValueError("a layer has adapters of one or both of its projections, as many of each")
        self.into, self.out = into, out

    def check(self, into: list[int], out: list[int], k: int, inner: int) -> None:
        """Refuses adapters of other projections than the layer's."""
        for name, s, widths, n in (("into", self.into, into, k), ("out", self.out, out, inner)):
            if s is not None and (s.widths != tuple(widths) or s.k != n):
                raise ValueError(f"{name} must be adapters of slices of {list(widths)} rows over {n} inputs")


def project(x: torch.Tensor, w: torch.Tensor, adapters: AdapterSet | None = None,
            batch: AdapterBatch | None = None) -> torch.Tensor:
    """x W^T [T, N] bf16, with what the rows' adapters give if there are any."""
    from .prefill_gemm import linear
    from .projections import gemv
    y = gemv(w, x) if x.shape[0] == 1 else linear(x, w)
    return y if adapters is None or batch is None else apply_adapters(y, x, adapters, batch)
