"""A cache of keys and values in pages, quantized or not: new tokens appended to it (with rotary positions on the way) and pages copied
within it.  ``attention`` reads it.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

from . import _ffi
from .rotary import Rotary
from .scheme import ElemType, QuantScheme
from .tensor import ComputeClient, TensorHandleRef


@dataclass(frozen=True)
class Cache:
    """Keys and values of a layer, each [pages, kv_heads, page_size, dim / num_quants] (any strides but the last dimension's), and their
    scales [pages, kv_heads, page_size, dim / block].  ``scheme``: 8- or 4-bit values in blocks along the last dimension; None: floats, no
    scales.  Slot ``page * page_size + place`` is one token's place."""

    keys: TensorHandleRef
    values: TensorHandleRef
    scheme: Optional[QuantScheme] = None
    key_scales: Optional[TensorHandleRef] = None
    value_scales: Optional[TensorHandleRef] = None


def append(client: ComputeClient, cache: Cache, k: TensorHandleRef, v: TensorHandleRef, slots: TensorHandleRef, elem: ElemType,
           q: Optional[TensorHandleRef] = None, q_out: Optional[TensorHandleRef] = None, positions: Optional[TensorHandleRef] = None,
           rotary: Optional[Rotary] = None) -> None:
    """``k``, ``v`` [tokens, kv_heads, dim] of ``elem`` into their ``slots`` (i32; one outside of the cache: not stored), keys turned by
    ``positions`` (i32) as ``rotary`` says, both quantized as ``quantize.launch_dynamic`` does; ``q`` [tokens, heads, dim], turned, to
    ``q_out`` (which may be ``q``)."""
    rc = _ffi.calls().append(client.stream, cache.keys, cache.key_scales, cache.values, cache.value_scales, cache.scheme, k, v, slots, q, q_out, positions,
                             None if rotary is None else rotary.frequencies, 1.0 if rotary is None else rotary.magnitude,
                             False if rotary is None else rotary.interleaved, elem)
    if rc:
        _ffi.check_attention(rc)


def copy_pages(client: ComputeClient, tensors: Sequence[TensorHandleRef], pairs: TensorHandleRef) -> None:
    """Page ``pairs[i, 0]`` to page ``pairs[i, 1]`` (i32 on the device) in each of ``tensors``, whose first dimension is that of the pages:
    a sequence forks, or a pool is compacted.  No page may be the destination of two pairs, nor source and destination."""
    rc = _ffi.calls().copy_pages(client.stream, tensors, pairs)
    if rc:
        _ffi.check_attention(rc)
