"""What stands behind a product: bias, activation, gate and residual (``cq_epilogue`` of include/cubek_matmul.h)."""
from __future__ import annotations

import enum
from dataclasses import dataclass
from typing import Optional

from .tensor import TensorHandleRef


class Activation(enum.IntEnum):
    Identity = 0
    Relu = 1
    Silu = 2
    Gelu = 3       # by the error function
    GeluTanh = 4


@dataclass(frozen=True)
class Epilogue:
    """``y = act(v) + residual`` with ``v = x W^T + bias``; gated: ``y = act(v[:, :n]) * v[:, n:] + residual`` for a weight
    of ``2 n`` rows.  ``bias``: [rows of W] ([experts, rows of W]) typed like x or f32; ``residual``: shaped and typed like y, may be y."""

    activation: Activation = Activation.Identity
    gated: bool = False
    bias: Optional[TensorHandleRef] = None
    residual: Optional[TensorHandleRef] = None


IDENTITY = Epilogue()
