"""``y = epilogue(x @ dequantize(W)^T)`` for any number of tokens, with the weights read in their quantized form and each
entering as the value dequantize would store (the quantized-input arm of the reference's matmul,
crates/cubek-matmul/src/base.rs:309-317).  ``matvec`` is its form for up to sixteen bare vectors.
"""
from __future__ import annotations

from . import _ffi
from .epilogue import IDENTITY, Epilogue
from .scheme import ElemType, QuantScheme
from .tensor import ComputeClient, TensorHandleRef


def workspace_bytes(values: TensorHandleRef, scheme: QuantScheme, x: TensorHandleRef, elem: ElemType, epilogue: Epilogue = IDENTITY) -> int:
    return int(_ffi.matmul_lib().cq_matmul_workspace_bytes(values.as_c(), scheme.to_c(), x.as_c(), int(elem), _ffi.epilogue_to_c(epilogue)))


def launch_ref(client: ComputeClient, values: TensorHandleRef, params: TensorHandleRef, scheme: QuantScheme, x: TensorHandleRef,
               y: TensorHandleRef, elem: ElemType, y_elem: ElemType, epilogue: Epilogue = IDENTITY, workspace: int = 0,
               workspace_size: int = 0) -> None:
    """``values``: packed [rows, cols / num_quants]; ``params``: the scales; ``x``: [tokens, cols] of ``elem``; ``y``: [tokens, rows]
    of ``y_elem`` ([tokens, rows / 2] where gated).  ``workspace``: device memory of ``workspace_bytes()``, optional."""
    rc = _ffi.calls().matmul(client.stream, values, params, scheme, x, y, elem, y_elem, epilogue.activation, epilogue.gated,
                             epilogue.bias, epilogue.residual, workspace, workspace_size)
    if rc:
        _ffi.check_matmul(rc)
