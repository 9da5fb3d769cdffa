"""Several rollouts on one cache of pages.

A server generates many videos at a time.  Their keys and values lie in one pool, ``[pages, page size, Hk, D]`` a layer, of which each request has as many
pages as it needs; ``tables[b]`` names request ``b``'s, in order, and ``lens[b]`` its tokens.  One step of it:

    plan = plan_pages(tables, lens, new_lens, q.shape[0], n_pages=k_pages.shape[0], page_size=k_pages.shape[1])      # once
    for each layer:
        q = prepare_qkv_pages(q, k, v, positions, axes, k_pages, v_pages, plan.slots, norm="rms", ...)               # or append_pages(k, v, ...)
        out, lse = paged_attention(q, k_pages, v_pages, tables, plan.lens, plan.cu_seqlens, served=plan.served, left=7, right=0, frame=1350, sinks=226)
    lens = plan.lens

The new tokens of all requests are packed, one request behind the other.  Nothing here reads device memory on the host, so a step can be captured in a
graph and follows lengths that change.  No counterpart in the reference, which caches whole attention states (core/cache.py:75-84).
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _hip
from .producer import _NORMS, RotaryAxes
from .window import _limit

_INT32 = torch.int32


class PagePlan(NamedTuple):
    """What a step needs to know.  The results of a plan are parts of one allocation (``lens`` with ``in_place`` apart): whoever keeps ``lens`` for long
    keeps the 8 bytes a row of ``slots`` with it, and ``torch.save``, which refuses tensors of different types in one storage, takes clones of them."""

    lens: torch.Tensor          # int32 [B]: tokens of each request, the new ones among them where it is served
    cu_seqlens: torch.Tensor    # int32 [B + 1]: rows of each request's new tokens
    slots: torch.Tensor         # int64 [n_tokens]: page * page_size + place of each row; -1: nowhere
    served: torch.Tensor        # bool [B]: whether there were pages for all of its new tokens


def plan_pages(tables: torch.Tensor, lens: torch.Tensor, new_lens: torch.Tensor, n_tokens: int, *, n_pages: int, page_size: int,
               in_place: bool = False) -> PagePlan:
    """Pages for the new tokens of each request.  ``tables`` int32 ``[B, entries]``, ``lens`` and ``new_lens`` int32 ``[B]``, on the GPU; ``n_tokens``: rows
    of the packed tensors, at least the sum of ``new_lens`` (tokens beyond them do not exist).

    A request holds the first ``ceil(len / page_size)`` entries of its row of ``tables``; what stands behind them means nothing.  Pages that no request
    holds are free: a request ends by its length going to 0, and requests may share the whole pages of a common beginning.  Requests take free pages in
    order, the lowest first, and their entries go into ``tables``.  A request whose tokens do not fit its row gets none, and from the first one that finds too
    few free pages on, no request gets any: ``served`` says whose tokens have a place; the rows of the others stay without a slot, and their length as it
    was, so that the attention behind it needs ``served`` as well.  With ``in_place`` ``lens`` itself becomes the new lengths, for a captured step that is
    replayed."""
    if lens.dtype is not _INT32 or new_lens.dtype is not _INT32 or tables.dtype is not _INT32:
        raise ValueError(f"tables, lens and new_lens must be int32, got {tables.dtype}, {lens.dtype}, {new_lens.dtype}")
    return PagePlan(*_hip.plan_pages(tables, lens, new_lens, n_tokens, n_pages, page_size, in_place))


def append_pages(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, slots: torch.Tensor) -> None:
    """Writes row ``t`` of k and v ``[T,Hk,D]`` (bf16 or fp16, any strides with a contiguous last dimension) into slot ``slots[t]`` of the pages
    ``[pages, page size, Hk, D]``; rows without a slot (-1) are left out.  Slots are distinct, as ``plan_pages`` makes them: of rows that share one, elements of
    either remain."""
    _hip.append_pages(k, v, k_pages, v_pages, slots)


def prepare_qkv_pages(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, axes: RotaryAxes, k_pages: torch.Tensor,
                      v_pages: torch.Tensor, slots: torch.Tensor, *, norm: Optional[str] = None, q_weight: Optional[torch.Tensor] = None,
                      q_bias: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, k_bias: Optional[torch.Tensor] = None,
                      eps: float = 1e-6, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``producer.prepare_qk_axes`` of q ``[T,H,D]`` and k ``[T,Hk,D]`` by ``positions`` int32 ``[T, axes]``, whose keys go straight into their slots, and
    ``append_pages`` of v, in one launch.  Returns q, contiguous; q of rows without a slot is computed as well."""
    if norm not in _NORMS:
        raise ValueError(f"unknown norm {norm!r}")
    if positions.dtype is not _INT32:
        raise ValueError(f"positions must be int32, got {positions.dtype}")
    if positions.dim() != 2 or positions.size(-1) != len(axes.dims):
        raise ValueError(f"positions must be [T, {len(axes.dims)}] for these axes, got {tuple(positions.shape)}")
    return _hip.prepare_pages([(q, q_weight, q_bias, out, 1.0), (k, k_weight, k_bias, None, 1.0)], v,
                              positions if positions.is_contiguous() else positions.contiguous(), axes.table, _NORMS[norm], eps, k_pages, v_pages, slots)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor, lens: torch.Tensor, cu_seqlens: torch.Tensor, *,
                    served: Optional[torch.Tensor] = None, max_seqlen_q: Optional[int] = None, left: Optional[int] = None, right: Optional[int] = None,
                    frame: int = 1, sinks: int = 0, softmax_scale: float = 0.0, out: Optional[torch.Tensor] = None,
                    lse: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """q ``[T,H,D]`` (bf16 or fp16, D 64 or 128; H a multiple of the pages' key heads) holds the new tokens of request ``b`` in rows ``cu_seqlens[b] ..
    cu_seqlens[b + 1]``: the last ones of its ``lens[b]`` tokens, whose keys and values are in the pages already.  Returns (out ``[T,H,D]``, lse fp32
    ``[H,T]``).

    Row ``i`` of a request's ``n`` stands at position ``lens[b] - n + i`` and sees the frames that ``left``, ``right``, ``frame`` and ``sinks`` name in
    ``window.window_attention`` (``right=0``: causal, by tokens or by whole frames).  Rows that see no key, and rows that belong to no request, get 0 and an
    lse of -inf; so do the rows of a request that ``served`` (bool ``[B]``, as ``plan_pages`` makes it) leaves out, whose keys are not in the pages.  Without
    ``served`` every request's are.  ``max_seqlen_q`` is the most rows a request has, where the caller knows it: the launch is made for that; without it
    for ``T``.  An entry of ``tables`` that a window needs and that names no page stands for keys and values of zeros."""
    if tables.dtype is not _INT32 or lens.dtype is not _INT32 or cu_seqlens.dtype is not _INT32:
        raise ValueError(f"tables, lens and cu_seqlens must be int32, got {tables.dtype}, {lens.dtype}, {cu_seqlens.dtype}")
    if served is not None and served.dtype is not torch.bool:
        raise ValueError(f"served must be bool, got {served.dtype}")
    if frame < 1:
        raise ValueError(f"frame must be at least 1, got {frame}")
    rows = q.shape[0] if max_seqlen_q is None else _limit("max_seqlen_q", max_seqlen_q)
    return _hip.attn_pages_fwd(q, k_pages, v_pages, tables, lens, cu_seqlens, rows, _limit("left", left),
                               _limit("right", right), _limit("frame", frame), _limit("sinks", sinks), softmax_scale, out, lse, served)
