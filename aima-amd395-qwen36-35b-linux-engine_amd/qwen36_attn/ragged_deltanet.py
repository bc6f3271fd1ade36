"""Gated DeltaNet over ragged batches, states in slots.

No counterpart in the reference, which runs one sequence
(``linear_attention``, four_layer_mini_engine.py:6378-6544).  Prompts, drafted
tokens and single tokens of any number of sequences go through the same calls,
next to ``paged_attention`` for the full-attention layers.

The batch of a call is ``cu_tokens`` int32 [seqs + 1] (row offsets of the call),
``slots`` int32 [seqs] (where each sequence's states are) and ``has_state`` bool
[seqs] or None (all True): where False the sequence begins with zeros, whatever
its slot holds.  They are GPU tensors, read when the launch runs.  A sequence
without rows, or with a slot outside the pool, is padding: its rows and slot stay
as they are, as do rows behind the last sequence.  A slot must belong to one
sequence of the batch.  All arithmetic runs in ``libqwen36_attn.so``.
"""
from __future__ import annotations

import torch

from . import _lib
from ._tensors import launch
from .full_attention import MAX_TOKENS
from .gated_deltanet import CONV_DIM, DK, DV, HK, HV, KEY_DIM, VALUE_DIM

_STATE, _CONV = ((HV, DK, DV), (DK * DV, DV, 1)), ((CONV_DIM, 3), (3, 1))     # a slot's shape and strides


def _pool(t, name: str, dtype, shape: tuple, strides: tuple) -> tuple[int, int, int, int]:
    """Device index, slots, address and slot stride in elements of a [slots, ...] pool
    whose slots have ``strides``."""
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or not t.is_cuda:
        raise ValueError(f"{name} must be a {dtype} GPU tensor")
    size, step, at = t.shape, t.stride(), t.data_ptr()
    if len(size) != len(shape) + 1 or size[1:] != shape or size[0] < 1:
        raise ValueError(f"{name} must be [slots, {', '.join(map(str, shape))}]")
    n, least = size[0], shape[0] * strides[0]
    stride = step[0] if n > 1 else least
    if step[1:] != strides or stride < least or (stride * t.itemsize | at) & 15:
        raise ValueError(f"{name}: a slot must be contiguous, 16-byte aligned and apart from the others")
    return t.get_device(), n, at, stride


def _batch(index: int, tokens: int, n_slots: int, cu_tokens, slots, has_state) -> _lib.StateBatchArgs:
    for t in (cu_tokens, slots):
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.get_device() != index \
                or t.dim() != 1 or not t.is_contiguous():
            raise ValueError("cu_tokens [seqs + 1] and slots [seqs] must be contiguous int32 tensors "
                             "on the pool's device")
    seqs = len(slots)
    if len(cu_tokens) != seqs + 1 or not 1 <= seqs <= 65536:
        raise ValueError("a batch is cu_tokens [seqs + 1] and slots [seqs] of 1 to 65536 sequences")
    has = None
    if has_state is not None:
        if not isinstance(has_state, torch.Tensor) or has_state.dtype is not torch.bool \
                or has_state.get_device() != index or has_state.shape != (seqs,) or not has_state.is_contiguous():
            raise ValueError("has_state must be a contiguous bool tensor [seqs] on the pool's device")
        has = has_state.data_ptr()
    if not 0 < tokens <= MAX_TOKENS:
        raise ValueError(f"a call has 1 to {MAX_TOKENS} rows")
    return _lib.StateBatchArgs(cu_tokens.data_ptr(), slots.data_ptr(), has, seqs, tokens, n_slots)


def _heads(t, name: str, tokens: int, heads: tuple, index: int) -> tuple[int, int, int]:
    """Address, heads and token stride of a bf16 [tokens, heads, 128] tensor with
    contiguous rows."""
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.bfloat16 or t.get_device() != index:
        raise ValueError(f"{name} must be a bf16 tensor on the pool's device")
    size = t.shape
    if len(size) != 3 or size[0] != tokens or size[1] not in heads or size[2] != DK:
        raise ValueError(f"{name} must be [{tokens}, {' or '.join(map(str, heads))}, 128]")
    at, (stride, head, inner) = t.data_ptr(), t.stride()
    width = size[1] * DK
    if tokens == 1:
        stride = width
    if inner != 1 or head != DK or not width <= stride <= 1 << 24 or stride & 7 or at & 15:
        raise ValueError(f"{name} must have contiguous, 16-byte aligned rows, apart by 2^24 elements at most")
    return at, size[1], stride


def _scalars(t, name: str, tokens: int, index: int) -> int:
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.float32 or t.get_device() != index \
            or t.shape != (tokens, HV) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous fp32 [{tokens}, 32] on the pool's device")
    return t.data_ptr()


def _out(out, shape: tuple, device) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=torch.bfloat16, device=device)
    if not isinstance(out, torch.Tensor) or out.dtype is not torch.bfloat16 or out.device != device \
            or tuple(out.shape) != shape or not out.is_contiguous() or out.data_ptr() % 16:
        raise ValueError(f"out must be contiguous bf16 {list(shape)} on the pool's device")
    return out


def ragged_conv1d(mixed_qkv: torch.Tensor, weight: torch.Tensor, states: torch.Tensor,
                  cu_tokens: torch.Tensor, slots: torch.Tensor, has_state: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """``gated_deltanet.causal_conv1d`` for a batch, with its arithmetic: mixed_qkv
    [T, 8192] bf16 (unit inner stride), weight [8192, 4] bf16, states [slots, 8192, 3]
    bf16, replaced in place by each sequence's last three inputs.  Returns SiLU(conv)
    [T, 8192] bf16; ``out`` overlaps no input."""
    index, n, sp, ss = _pool(states, "states", torch.bfloat16, *_CONV)
    t = mixed_qkv.shape[0] if isinstance(mixed_qkv, torch.Tensor) and mixed_qkv.dim() == 2 else 0
    if t == 0 or mixed_qkv.dtype is not torch.bfloat16 or mixed_qkv.get_device() != index \
            or mixed_qkv.shape[1] != CONV_DIM:
        raise ValueError("mixed_qkv must be bf16 [T, 8192] on the pool's device")
    at, (stride, inner) = mixed_qkv.data_ptr(), mixed_qkv.stride()
    if t == 1:
        stride = CONV_DIM
    if inner != 1 or not CONV_DIM <= stride < 1 << 32 or stride & 7 or at & 15:
        raise ValueError("mixed_qkv must have unit inner stride and 16-byte aligned rows that do not overlap")
    if not isinstance(weight, torch.Tensor) or weight.dtype is not torch.bfloat16 or weight.get_device() != index \
            or weight.shape != (CONV_DIM, 4) or not weight.is_contiguous() or weight.data_ptr() & 15:
        raise ValueError("weight must be contiguous bf16 [8192, 4] on the pool's device")
    batch = _batch(index, t, n, cu_tokens, slots, has_state)
    out = _out(out, (t, CONV_DIM), states.device)
    launch(index, "qwen36_gdn_ragged_conv1d", at, stride, weight.data_ptr(), sp, ss, batch,
           out.data_ptr())
    return out


def ragged_delta_rule(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                      states: torch.Tensor, cu_tokens: torch.Tensor, slots: torch.Tensor,
                      has_state: torch.Tensor | None = None, out: torch.Tensor | None = None,
                      longest: int | None = None, flags: int = 0) -> torch.Tensor:
    """The gated delta rule for a batch: q, k [T, 16 (or 32 repeated), 128], v [T, 32,
    128] bf16 (q and k are l2-normalised in the kernel), g (log decay, at most 0, -inf
    among them), beta (0 to 2) [T, 32] fp32, states [slots, 32, 128 (k), 128 (v)] fp32,
    replaced in place by the sequences' last states.  ``longest``: the most rows that a
    sequence of the call has, where the caller knows it; it only chooses between the forms
    for few and for many tokens (a sequence may have more).  ``flags``:
    ``gated_deltanet.QK_NORMALIZED`` (q and k, of norm 1 at most, are used as given) and
    ``STATE_VK`` (states are [slots, 32, 128 (v), 128 (k)]).  Returns [T, 32, 128] bf16;
    ``out`` overlaps no input.  A value that is not finite may reach any row of its chunk of
    64, those before it too, where a sequence has 8 and more rows.  A call of more than 12
    rows takes 824 KiB of workspace for every 64 rows and every sequence that may have 8 and
    more of them, an eighth of the rows at most (none where ``longest`` is less: a decode
    step of many sequences says 1)."""
    index, n, sp, ss = _pool(states, "states", torch.float32, *_STATE)
    t = v.shape[0] if isinstance(v, torch.Tensor) and v.dim() == 3 else 0
    (qp, heads, qs), (kp, *same) = _heads(q, "q", t, (HK, HV), index), _heads(k, "k", t, (HK, HV), index)
    if same != [heads, qs]:
        raise ValueError("q and k must share shape and token stride")
    vp, _, vs = _heads(v, "v", t, (HV,), index)
    gp, bp = _scalars(g, "g", t, index), _scalars(beta, "beta", t, index)
    if longest is not None and longest < 1:
        raise ValueError("longest must be positive")
    batch = _batch(index, t, n, cu_tokens, slots, has_state)
    out = _out(out, (t, HV, DV), states.device)
    most = min(longest or 0, MAX_TOKENS)
    nb = 0 if t == 1 else (_lib._LIB or _lib.load()).qwen36_gdn_ragged_delta_workspace_bytes(batch, most)
    # allocated per call: calls on several streams, and graphs captured apart, never share one
    ws = torch.empty(nb, dtype=torch.uint8, device=states.device) if nb else None
    launch(index, "qwen36_gdn_ragged_delta_ex", qp, kp, vp, heads, qs, vs, gp, bp,
           sp, ss, batch, most, flags, out.data_ptr(), None if ws is None else ws.data_ptr(), nb)
    return out


def fork_states(pools, parents: torch.Tensor) -> None:
    """Slot i of every pool (the layers' [slots, ...] conv and recurrent states) becomes a
    copy of its slot ``parents[i]`` (int32 [slots], -1: it stays; a child of a slot that
    is a child of the same call stays too): what ``page_tables.fork`` is for pages, but
    for rows that are not empty, which stay there and are copied over here."""
    pools = list(pools)
    if not pools or not isinstance(parents, torch.Tensor) or parents.dtype is not torch.int32 \
            or parents.dim() != 1 or not parents.is_cuda or not parents.is_contiguous() \
            or not 1 <= parents.shape[0] <= 65536:
        raise ValueError("pools must be one or more tensors and parents a contiguous int32 GPU tensor [slots]")
    n, index, args = parents.shape[0], parents.get_device(), []
    for t in pools:
        if not isinstance(t, torch.Tensor) or t.get_device() != index or t.dim() < 2 or t.shape[0] != n \
                or not t[0].is_contiguous():
            raise ValueError("a pool must be [slots, ...] with contiguous slots on the device of parents")
        size = t.nbytes // n
        stride = t.stride(0) * t.itemsize if n > 1 else size
        if size < 1 or (size | stride | t.data_ptr()) & 15 or stride < size:
            raise ValueError("a pool's slots must be 16-byte aligned, multiples of 16 bytes and apart")
        args.append(_lib.SlotPoolArgs(t.data_ptr(), size, stride))
    if len({a.data for a in args}) < len(args):
        raise ValueError("a pool is listed twice")
    launch(index, "qwen36_slots_fork", (_lib.SlotPoolArgs * len(args))(*args), len(args), n,
           parents.data_ptr())


class RaggedLinearAttentionLayer:
    """One Gated-DeltaNet layer over ragged batches, ``gated_deltanet.
    LinearAttentionLayer`` for many sequences: the projections, the convolution and the
    delta rule with their states in ``conv_states`` [slots, 8192, 3] bf16 and
    ``ssm_states`` [slots, 32, 128, 128] fp32, the gated norm and out_proj.
    ``weights`` as there; ``adapters``: an ``adapters.LayerAdapters`` of in_proj and
    out_proj."""

    def __init__(self, weights: dict, conv_states: torch.Tensor, ssm_states: torch.Tensor, adapters=None) -> None:
        if _pool(conv_states, "conv_states", torch.bfloat16, *_CONV)[:2] \
                != _pool(ssm_states, "ssm_states", torch.float32, *_STATE)[:2]:
            raise ValueError("conv_states and ssm_states must have the same slots on one device")
        from .projections import FusedProjection
        self.w, self.conv_states, self.ssm_states = weights, conv_states, ssm_states
        self._in_proj = FusedProjection(weights["in_proj_qkv"], weights["in_proj_z"], weights["in_proj_b"],
                                        weights["in_proj_a"])
        if adapters is not None:
            adapters.check(self._in_proj.splits, [weights["out_proj"].shape[0]], self._in_proj.w.shape[1], VALUE_DIM)
        self._into, self._out = (None, None) if adapters is None else (adapters.into, adapters.out)

    def forward(self, inp: torch.Tensor, cu_tokens: torch.Tensor, slots: torch.Tensor,
                has_state: torch.Tensor | None = None, longest: int | None = None,
                adapter_batch=None) -> torch.Tensor:
        """inp [T, 2048]: the new rows of the batch's sequences.  ``adapter_batch``: the
        ``adapters.AdapterBatch`` of these rows (None: no request has an adapter).  Returns
        [T, 2048]; rows of padding hold nothing of use."""
        from .adapters import project
        from .gated_deltanet import gated_rmsnorm, gating
        w, t = self.w, inp.shape[0]
        mixed, z, b, a = self._in_proj.split_rows(project(inp, self._in_proj.w, self._into, adapter_batch))
        conv = ragged_conv1d(mixed, w["conv1d"], self.conv_states, cu_tokens, slots, has_state)
        q = conv[:, :KEY_DIM].view(t, HK, DK)
        k = conv[:, KEY_DIM:2 * KEY_DIM].view(t, HK, DK)
        v = conv[:, 2 * KEY_DIM:].view(t, HV, DV)
        g, beta = gating(a, b, w["A_log"], w["dt_bias"])
        core = ragged_delta_rule(q, k, v, g, beta, self.ssm_states, cu_tokens, slots, has_state, longest=longest)
        gated = gated_rmsnorm(core, z, w["norm"])
        return project(gated.view(t, VALUE_DIM), w["out_proj"], self._out, adapter_batch)
