"""Attention of new tokens, one or many of each sequence, over a cache of keys and values in pages (``cache.Cache``).  The reference's attention
crate (crates/cubek-attention) takes contiguous floats.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

from . import _ffi
from .cache import Cache
from .scheme import ElemType
from .tensor import ComputeClient, TensorHandleRef


@dataclass(frozen=True)
class Scores:
    """What stands between queries and weights: t = scale * q k (None: dim^-0.5), then cap * tanh(t / cap) where ``cap`` > 0, then
    - slopes[head] * distance; a query sees the keys up to its own position and, where given, those before ``prefix`` of its sequence, and of
    them, where ``window`` > 0, only those less than ``window`` behind."""

    scale: Optional[float] = None
    cap: float = 0.0
    window: int = 0
    slopes: Optional[TensorHandleRef] = None  # f32 [heads]
    prefix: Optional[TensorHandleRef] = None  # i32 [sequences]


DEFAULT = Scores()


def workspace_bytes(cache: Cache, q: TensorHandleRef, table: TensorHandleRef, elem: ElemType) -> int:
    return int(_ffi.attention_lib().cq_attention_workspace_bytes(_ffi.cache_to_c(cache), q.as_c(), table.as_c(), int(elem)))


def launch_ref(client: ComputeClient, cache: Cache, q: TensorHandleRef, y: TensorHandleRef, table: TensorHandleRef, offsets: TensorHandleRef,
               lengths: TensorHandleRef, elem: ElemType, scores: Scores = DEFAULT, workspace: int = 0, workspace_size: int = 0) -> None:
    """``q``, ``y``: [tokens, heads, dim] of ``elem``; i32 on the device: ``table`` [sequences, pages] of each sequence, ``offsets``
    [sequences + 1] of its tokens, ``lengths`` [sequences] of its keys with the new ones, which are in the cache already.
    ``workspace``: device memory of ``workspace_bytes()``, optional."""
    scale = scores.scale
    if scale is None:
        scale = q.shape[-1] ** -0.5 if q.shape and q.shape[-1] else 1.0  # heads without entries are the library's to refuse
    rc = _ffi.calls().attention(client.stream, cache.keys, cache.key_scales, cache.values, cache.value_scales, cache.scheme, q, y, table, offsets, lengths,
                                scale, scores.cap, scores.window, scores.slopes, scores.prefix, elem, workspace, workspace_size)
    if rc:
        _ffi.check_attention(rc)
