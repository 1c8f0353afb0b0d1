"""Products grouped by expert: rows of y with a weight of their own for every group, of any sizes that only the device knows.
``routing`` makes the groups and adds the experts' results up.
"""
from __future__ import annotations

from typing import Optional

from . import _ffi
from .epilogue import IDENTITY, Epilogue
from .scheme import ElemType, QuantScheme
from .tensor import ComputeClient, TensorHandleRef


def workspace_bytes(values: TensorHandleRef, scheme: QuantScheme, y: TensorHandleRef, elem: ElemType, epilogue: Epilogue = IDENTITY) -> int:
    return int(_ffi.matmul_lib().cq_experts_workspace_bytes(values.as_c(), scheme.to_c(), y.as_c(), int(elem), _ffi.epilogue_to_c(epilogue)))


def launch_ref(client: ComputeClient, values: TensorHandleRef, params: TensorHandleRef, scheme: QuantScheme, x: TensorHandleRef,
               offsets: TensorHandleRef, y: TensorHandleRef, elem: ElemType, y_elem: ElemType, rows: Optional[TensorHandleRef] = None,
               epilogue: Epilogue = IDENTITY, workspace: int = 0, workspace_size: int = 0) -> None:
    """``y[p] = epilogue(x[rows[p]] @ dequantize(W[e])^T)`` for ``offsets[e] <= p < offsets[e + 1]``; without ``rows``
    position p takes row p of x.  ``values``: packed [experts, rows, cols / num_quants]; ``offsets``, ``rows``: i32 on the device."""
    rc = _ffi.calls().experts(client.stream, values, params, scheme, x, offsets, rows, y, elem, y_elem, epilogue.activation,
                              epilogue.gated, epilogue.bias, epilogue.residual, workspace, workspace_size)
    if rc:
        _ffi.check_matmul(rc)
