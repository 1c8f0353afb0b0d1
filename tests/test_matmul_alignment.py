"""Scales and x that do not start on a multiple of their elements' size, which the kernels read by the words around them, are refused."""
import pytest

from cubek_amd import ElemType, QuantParam, _ffi, experts, matmul
from test_matmul_refusals import BF16, BLOCK, CLIENT, F32, GOOD, GROUPED, P, status, t

HALF = BLOCK.with_param(QuantParam.F16)


@pytest.mark.parametrize("changes", [dict(x=t(5, 128, ptr=P + 1)), dict(x=t(5, 128, size=4, ptr=P + 2), elem=F32), dict(params=t(64, 4, size=4, ptr=P + 2)),
                                     dict(params=t(64, 4, size=4, ptr=P + 1)), dict(params=t(64, 4, ptr=P + 3), scheme=HALF)])
def test_products(changes):
    a = {**GOOD, **changes}
    assert status(matmul.launch_ref, CLIENT, a["values"], a["params"], a["scheme"], a["x"], a["y"], a["elem"], a["y_elem"]) == _ffi.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("changes", [dict(x=t(5, 128, ptr=P + 1)), dict(params=t(3, 64, 4, size=4, ptr=P + 2))])
def test_grouped_products(changes):
    a = {**GROUPED, **changes}
    assert status(experts.launch_ref, CLIENT, a["values"], a["params"], a["scheme"], a["x"], a["offsets"], a["y"], BF16, ElemType.BF16, a["rows"]) == _ffi.ERR_INVALID_ARGUMENT
