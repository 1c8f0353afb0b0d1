"""The choice of each token's experts, the positions of (token, choice) sorted by expert, and the weighted sum of the experts' results:
what stands before and behind ``experts``.
"""
from __future__ import annotations

import enum
from typing import Optional

from . import _ffi
from .scheme import ElemType
from .tensor import ComputeClient, TensorHandleRef


class Score(enum.IntEnum):
    Softmax = 0  # over all experts of the token
    Sigmoid = 1


def workspace_bytes(tokens: int, experts: int, chosen: int) -> int:
    return int(_ffi.matmul_lib().cq_route_workspace_bytes(tokens, experts, chosen))


def launch_ref(client: ComputeClient, logits: TensorHandleRef, weights: TensorHandleRef, experts: TensorHandleRef, offsets: TensorHandleRef,
               rows: TensorHandleRef, slots: TensorHandleRef, elem: ElemType, score: Score = Score.Softmax, normalize: bool = True,
               workspace: int = 0, workspace_size: int = 0) -> None:
    """``logits``: [tokens, experts] of ``elem``.  Writes ``weights`` (f32) and ``experts`` (i32) [tokens, chosen], the largest
    logits first, equal ones by rising expert; ``offsets`` [experts + 1], ``rows`` [tokens * chosen] and ``slots``
    [tokens, chosen] (i32) as ``experts.launch_ref`` and ``combine`` take them."""
    rc = _ffi.calls().route(client.stream, logits, weights, experts, offsets, rows, slots, elem, score, normalize, workspace, workspace_size)
    if rc:
        _ffi.check_matmul(rc)


def combine(client: ComputeClient, h: TensorHandleRef, slots: TensorHandleRef, weights: TensorHandleRef, y: TensorHandleRef,
            h_elem: ElemType, y_elem: ElemType, residual: Optional[TensorHandleRef] = None) -> None:
    """``y[t] = residual[t] + sum_j weights[t, j] * h[slots[t, j]]``, in f32, rounded once; ``residual`` may be ``y``."""
    rc = _ffi.calls().combine(client.stream, h, slots, weights, residual, y, h_elem, y_elem)
    if rc:
        _ffi.check_matmul(rc)
