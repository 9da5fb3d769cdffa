"""Attention in a window of frames or tokens, with first tokens that stay visible.

A rolled-out video grows without end; its queries attend to the frames around their own and to the first tokens of the sequence (the prompt,
the first frame), which hold a softmax together that has lost everything else.  The result is an attention state ``(out, lse)`` like those
of ``proAttention``'s launches: it merges with them (``utils.update_out_and_lse``, ``core.cache.merge_any``).  No counterpart in the
reference, whose chunks are attended to whole.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _hip


def _limit(name: str, value: Optional[int]) -> int:
    if value is None:
        return -1
    if type(value) is not int:
        if isinstance(value, bool) or not hasattr(value, "__index__"):
            raise ValueError(f"{name} must be None or a whole number of at least 0, got {value!r}")
        value = value.__index__()
    if not 0 <= value < 1 << 31:
        raise ValueError(f"{name} must be None or a whole number of at least 0, got {value!r}")
    return value


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, left: Optional[int] = None, right: Optional[int] = None,
                     frame: int = 1, sinks: int = 0, q_begin: Optional[int] = None, kv_lens: Optional[torch.Tensor] = None,
                     softmax_scale: float = 0.0, out: Optional[torch.Tensor] = None,
                     lse: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """q ``[B,Sq,H,D]``, k / v ``[B,Sk,Hk,D]``, bf16 or fp16, D 64 or 128; only the last dimension must be contiguous; ``H`` is a multiple of
    ``Hk`` (query heads share key heads).  Returns (out ``[B,Sq,H,D]`` in q's dtype, lse fp32 ``[B,H,Sq]``).

    Query row ``i`` stands at position ``p = q_begin + i`` among the keys; by default behind them, ``p = len - Sq + i``.  It sees the frames of
    ``frame`` tokens from ``left`` before its own to ``right`` behind it (``None``: no border; ``right = 0`` with ``frame = 1`` is causal) and,
    up to the right border, the first ``sinks`` keys.  Frames are counted from key ``sinks``: with ``sinks`` text tokens in front of the
    video, frame ``f`` is the tokens ``sinks + f * frame ..``.  A row that sees no key gets 0 and an lse of -inf.

    ``kv_lens`` int32 ``[B]`` on the GPU: the keys that each sample has (``len``; otherwise ``Sk``).  The host does not read it, so a captured launch
    follows a cache that grows.  What stands behind the length, or is masked otherwise, adds nothing, whatever it holds."""
    if kv_lens is not None and kv_lens.dtype is not torch.int32:
        raise ValueError(f"kv_lens must be int32, got {kv_lens.dtype}")
    if frame < 1:
        raise ValueError(f"frame must be at least 1, got {frame}")
    return _hip.attn_window_fwd(q, k, v, _limit("left", left), _limit("right", right), _limit("frame", frame), _limit("sinks", sinks),
                                _limit("q_begin", q_begin), kv_lens, softmax_scale, out, lse)
