"""The calls of include/cubek_matmul.h refuse what they do not take before anything touches a GPU, and header, binding and library agree."""
import os
import re

import pytest

from cubek_amd import (Activation, ComputeClient, ElemType, Epilogue, QuantError, QuantLevel, QuantScheme, QuantStore, QuantValue, Score, TensorHandleRef,
                       _ffi, experts, matmul, routing)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # never read: every call here is refused
CLIENT = ComputeClient(0)
BF16, F32 = ElemType.BF16, ElemType.F32
BLOCK = QuantScheme.default().with_value(QuantValue.Q4S).with_level(QuantLevel.block([32]))


def t(*shape, size=2, strides=None, ptr=P):
    if strides is None:
        strides, n = [], 1
        for s in reversed(shape):
            strides.insert(0, n)
            n *= s
    return TensorHandleRef(ptr, tuple(shape), tuple(strides), size)


def status(call, *args, **kwargs):
    with pytest.raises(QuantError) as e:
        call(*args, **kwargs)
    return e.value.status


def test_header_binding_and_library_agree():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "cubek_matmul.h")).read(), flags=re.S)
    assert sorted(set(re.findall(r"\b(cq_[a-z0-9_]+)\s*\(", text))) == sorted(_ffi.MATMUL_SYMBOLS)
    lib = _ffi.matmul_lib()
    assert all(getattr(lib, s) is not None for s in _ffi.MATMUL_SYMBOLS)


GOOD = dict(values=t(64, 16, size=4), params=t(64, 4, size=4), scheme=BLOCK, x=t(5, 128), y=t(5, 64), elem=BF16, y_elem=BF16, epilogue=Epilogue())
OTHER = [
    ("INVALID_ARGUMENT", dict(values=t(64, 16, size=4, ptr=0))),
    ("INVALID_ARGUMENT", dict(x=t(5, 128, ptr=0))),
    ("INVALID_ARGUMENT", dict(y=t(5, 64, ptr=0))),
    ("INVALID_ARGUMENT", dict(params=t(64, 4, size=4, ptr=0))),
    ("INVALID_ARGUMENT", dict(elem=7)),
    ("INVALID_ARGUMENT", dict(y_elem=-1)),
    ("INVALID_ARGUMENT", dict(x=t(1, 1, 1, 1, 1, 1, 1, 5, 128))),
    ("INVALID_ARGUMENT", dict(epilogue=Epilogue(5))),
    ("INVALID_ARGUMENT", dict(epilogue=Epilogue(Activation.Silu, gated=2))),
    ("INVALID_ARGUMENT", dict(epilogue=Epilogue(bias=t(64, ptr=0)))),
    ("UNSUPPORTED_SCHEME", dict(scheme=BLOCK.with_store(QuantStore.Native))),
    ("SHAPE_MISMATCH", dict(values=t(64, 16, size=1))),
    ("SHAPE_MISMATCH", dict(values=t(1, 64, 16, size=4))),
    ("SHAPE_MISMATCH", dict(params=t(64, 4, size=2))),
    ("SHAPE_MISMATCH", dict(params=t(64, 5, size=4))),
    ("SHAPE_MISMATCH", dict(params=t(4, size=4))),
    ("SHAPE_MISMATCH", dict(scheme=BLOCK.with_level(QuantLevel.block([48])))),
    ("SHAPE_MISMATCH", dict(scheme=BLOCK.with_level(QuantLevel.block([3, 32])))),
    ("SHAPE_MISMATCH", dict(x=t(5, 120))),
    ("SHAPE_MISMATCH", dict(x=t(5, 128, size=4))),
    ("SHAPE_MISMATCH", dict(x=t(4, 128))),
    ("SHAPE_MISMATCH", dict(x=t(128), y=t(5, 64))),
    ("SHAPE_MISMATCH", dict(y=t(5, 63))),
    ("SHAPE_MISMATCH", dict(y=t(5, 64, size=4))),
    ("SHAPE_MISMATCH", dict(epilogue=Epilogue(gated=True))),
    ("SHAPE_MISMATCH", dict(values=t(63, 16, size=4), params=t(63, 4, size=4), y=t(5, 31), epilogue=Epilogue(gated=True))),
    ("SHAPE_MISMATCH", dict(epilogue=Epilogue(bias=t(63)))),
    ("SHAPE_MISMATCH", dict(epilogue=Epilogue(bias=t(64, size=8)))),
    ("SHAPE_MISMATCH", dict(epilogue=Epilogue(bias=t(1, 64)))),
    ("SHAPE_MISMATCH", dict(epilogue=Epilogue(residual=t(5, 63)))),
    ("SHAPE_MISMATCH", dict(epilogue=Epilogue(residual=t(5, 64, size=4)))),
    ("NON_CONTIGUOUS", dict(values=t(64, 16, size=4, strides=(1, 64)))),
    ("NON_CONTIGUOUS", dict(x=t(5, 128, strides=(1, 5)))),
    ("NON_CONTIGUOUS", dict(y=t(5, 64, strides=(128, 2)))),
    ("NON_CONTIGUOUS", dict(epilogue=Epilogue(residual=t(5, 64, strides=(1, 5))))),
    ("TOO_LARGE", dict(values=t(64, 1 << 29, size=4))),
    ("TOO_LARGE", dict(values=t(1 << 32, 16, size=4))),
]


@pytest.mark.parametrize("name,changes", OTHER, ids=range(len(OTHER)))
def test_products_refuse(name, changes):
    a = {**GOOD, **changes}
    assert status(matmul.launch_ref, CLIENT, a["values"], a["params"], a["scheme"], a["x"], a["y"], a["elem"], a["y_elem"], a["epilogue"]) == getattr(_ffi, "ERR_" + name)


GROUPED = dict(values=t(3, 64, 16, size=4), params=t(3, 64, 4, size=4), scheme=BLOCK, x=t(5, 128), offsets=t(4, size=4), y=t(9, 64), rows=t(9, size=4), epilogue=Epilogue())
OTHER_GROUPED = [
    ("SHAPE_MISMATCH", dict(values=t(64, 16, size=4))),
    ("SHAPE_MISMATCH", dict(params=t(2, 64, 4, size=4))),
    ("SHAPE_MISMATCH", dict(scheme=BLOCK.with_level(QuantLevel.block([3, 1, 32])))),
    ("SHAPE_MISMATCH", dict(offsets=t(3, size=4))),
    ("SHAPE_MISMATCH", dict(offsets=t(4, size=8))),
    ("SHAPE_MISMATCH", dict(rows=t(8, size=4))),
    ("SHAPE_MISMATCH", dict(rows=None)),
    ("SHAPE_MISMATCH", dict(x=t(128))),
    ("SHAPE_MISMATCH", dict(x=t(0, 128))),
    ("SHAPE_MISMATCH", dict(epilogue=Epilogue(bias=t(64)))),
    ("NON_CONTIGUOUS", dict(offsets=t(4, size=4, strides=(2,)))),
    ("NON_CONTIGUOUS", dict(rows=t(9, size=4, strides=(2,)))),
    ("INVALID_ARGUMENT", dict(offsets=t(4, size=4, ptr=0))),
    ("INVALID_ARGUMENT", dict(rows=t(9, size=4, ptr=P + 2))),
]


@pytest.mark.parametrize("name,changes", OTHER_GROUPED, ids=range(len(OTHER_GROUPED)))
def test_grouped_products_refuse(name, changes):
    a = {**GROUPED, **changes}
    assert status(experts.launch_ref, CLIENT, a["values"], a["params"], a["scheme"], a["x"], a["offsets"], a["y"], BF16, BF16, a["rows"],
                  a["epilogue"]) == getattr(_ffi, "ERR_" + name)


ROUTE = dict(logits=t(5, 8, size=4), weights=t(5, 2, size=4), experts=t(5, 2, size=4), offsets=t(9, size=4), rows=t(10, size=4), slots=t(5, 2, size=4), elem=F32,
             score=Score.Softmax)
OTHER_ROUTE = [
    ("INVALID_ARGUMENT", dict(logits=t(5, 8, size=4, ptr=0))),
    ("INVALID_ARGUMENT", dict(score=2)),
    ("INVALID_ARGUMENT", dict(weights=t(5, 9, size=4), experts=t(5, 9, size=4), slots=t(5, 9, size=4), rows=t(45, size=4))),
    ("INVALID_ARGUMENT", dict(weights=t(5, 0, size=4), experts=t(5, 0, size=4), slots=t(5, 0, size=4), rows=t(0, size=4))),
    ("SHAPE_MISMATCH", dict(logits=t(5, 8))),
    ("SHAPE_MISMATCH", dict(experts=t(5, 3, size=4))),
    ("SHAPE_MISMATCH", dict(slots=t(4, 2, size=4))),
    ("SHAPE_MISMATCH", dict(offsets=t(8, size=4))),
    ("SHAPE_MISMATCH", dict(rows=t(9, size=4))),
    ("NON_CONTIGUOUS", dict(weights=t(5, 2, size=4, strides=(4, 1)))),
    ("TOO_LARGE", dict(logits=t(5, 1025, size=4), offsets=t(1026, size=4))),
    ("WORKSPACE_TOO_SMALL", dict(logits=t(500, 8, size=4), weights=t(500, 2, size=4), experts=t(500, 2, size=4), slots=t(500, 2, size=4), rows=t(1000, size=4))),
]


@pytest.mark.parametrize("name,changes", OTHER_ROUTE, ids=range(len(OTHER_ROUTE)))
def test_routing_refuses(name, changes):
    a = {**ROUTE, **changes}
    assert status(routing.launch_ref, CLIENT, a["logits"], a["weights"], a["experts"], a["offsets"], a["rows"], a["slots"], a["elem"], a["score"]) == getattr(_ffi, "ERR_" + name)


@pytest.mark.parametrize("name,changes", [
    ("INVALID_ARGUMENT", dict(h=t(10, 64, ptr=0))), ("SHAPE_MISMATCH", dict(h=t(10, 63))), ("SHAPE_MISMATCH", dict(slots=t(5, 3, size=4))),
    ("SHAPE_MISMATCH", dict(weights=t(4, 2, size=4))), ("SHAPE_MISMATCH", dict(weights=t(5, 2, size=2))), ("SHAPE_MISMATCH", dict(residual=t(5, 63))),
    ("NON_CONTIGUOUS", dict(slots=t(5, 2, size=4, strides=(1, 5)))), ("NON_CONTIGUOUS", dict(y=t(5, 64, strides=(1, 5))))])
def test_weighted_sum_refuses(name, changes):
    a = {**dict(h=t(10, 64), slots=t(5, 2, size=4), weights=t(5, 2, size=4), y=t(5, 64), residual=None), **changes}
    assert status(routing.combine, CLIENT, a["h"], a["slots"], a["weights"], a["y"], BF16, BF16, a["residual"]) == getattr(_ffi, "ERR_" + name)


def test_nothing_to_do_is_no_error():
    """Calls without tokens or rows succeed without a GPU: nothing is launched."""
    matmul.launch_ref(CLIENT, GOOD["values"], GOOD["params"], BLOCK, t(0, 128, ptr=0), t(0, 64, ptr=0), BF16, BF16)
    experts.launch_ref(CLIENT, GROUPED["values"], GROUPED["params"], BLOCK, t(0, 128, ptr=0), GROUPED["offsets"], t(0, 64, ptr=0), BF16, BF16)
    routing.combine(CLIENT, t(0, 64, ptr=0), t(0, 2, size=4, ptr=0), t(0, 2, size=4, ptr=0), t(0, 64, ptr=0), BF16, BF16)


def test_questions_about_sizes_need_no_gpu():
    assert matmul.workspace_bytes(GOOD["values"], BLOCK, GOOD["x"], BF16) >= 0
    assert experts.workspace_bytes(GROUPED["values"], BLOCK, GROUPED["y"], BF16) >= 0
    assert routing.workspace_bytes(16, 8, 2) == 0 and routing.workspace_bytes(10000, 128, 8) > 0 and routing.workspace_bytes(10000, 5000, 8) == 0
