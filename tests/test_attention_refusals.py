"""The calls of include/cubek_attention.h refuse what they do not take before anything touches a GPU, and header, binding and library agree."""
import ctypes
import os
import re
from dataclasses import replace

import pytest

from cubek_amd import (Cache, ComputeClient, ElemType, QuantError, QuantLevel, QuantScheme, QuantStore, QuantValue, Rotary, Scores, TensorHandleRef, _ffi,
                       attention, cache, rotary)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # never read: every call here is refused
CLIENT = ComputeClient(0)
BF16 = ElemType.BF16
BLOCK = QuantScheme.default().with_value(QuantValue.Q8S).with_store(QuantStore.Native).with_level(QuantLevel.block([32]))


def t(*shape, size=2, strides=None, ptr=P):
    if strides is None:
        strides, n = [], 1
        for s in reversed(shape):
            strides.insert(0, n)
            n *= s
    return TensorHandleRef(ptr, tuple(shape), tuple(strides), size)


def held(**other):
    return replace(Cache(t(9, 2, 16, 64, size=1), t(9, 2, 16, 64, size=1), BLOCK, t(9, 2, 16, 2, size=4), t(9, 2, 16, 2, size=4)), **other)


def plain(**other):
    return replace(Cache(t(9, 2, 16, 64), t(9, 2, 16, 64)), **other)


def words(scheme, stored):
    """A cache of the U32 store."""
    return held(scheme=scheme, keys=t(9, 2, 16, stored, size=4), values=t(9, 2, 16, stored, size=4))


def status(call, *args, **kwargs):
    with pytest.raises(QuantError) as e:
        call(*args, **kwargs)
    return e.value.status


def code(name):
    return getattr(_ffi, "ERR_" + name)


def test_header_binding_and_library_agree():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "cubek_attention.h")).read(), flags=re.S)
    assert sorted(set(re.findall(r"\b(cq_[a-z0-9_]+)\s*\(", text))) == sorted(_ffi.ATTENTION_SYMBOLS)
    lib = _ffi.attention_lib()
    assert all(getattr(lib, s) is not None for s in _ffi.ATTENTION_SYMBOLS)
    assert ctypes.sizeof(_ffi.CCache) == 40 and ctypes.sizeof(_ffi.CRotary) == 16 and ctypes.sizeof(_ffi.CScores) == 32


CACHES = [
    ("INVALID_ARGUMENT", held(keys=t(9, 2, 16, 64, size=1, ptr=0))),
    ("INVALID_ARGUMENT", held(values=t(9, 2, 16, 64, size=1, ptr=0))),
    ("INVALID_ARGUMENT", held(key_scales=None)),
    ("INVALID_ARGUMENT", held(value_scales=None)),
    ("INVALID_ARGUMENT", held(value_scales=t(9, 2, 16, 2, size=4, ptr=P + 2))),
    ("INVALID_ARGUMENT", plain(key_scales=t(9, 2, 16, 2, size=4))),
    ("INVALID_ARGUMENT", plain(keys=t(9, 2, 16, 64, ptr=P + 1))),
    ("SHAPE_MISMATCH", held(keys=t(9, 2, 16, 64))),
    ("SHAPE_MISMATCH", held(keys=t(9, 2, 16, 64, size=4))),
    ("SHAPE_MISMATCH", held(keys=t(2, 16, 64, size=1))),
    ("SHAPE_MISMATCH", held(values=t(9, 2, 16, 32, size=1))),
    ("SHAPE_MISMATCH", held(values=t(8, 2, 16, 64, size=1))),
    ("SHAPE_MISMATCH", held(values=t(9, 1, 16, 64, size=1))),
    ("SHAPE_MISMATCH", held(values=t(9, 2, 8, 64, size=1))),
    ("SHAPE_MISMATCH", held(key_scales=t(9, 2, 16, 2))),
    ("SHAPE_MISMATCH", held(key_scales=t(9, 2, 16, 3, size=4))),
    ("SHAPE_MISMATCH", held(key_scales=t(9, 2, 15, 2, size=4))),
    ("SHAPE_MISMATCH", held(value_scales=t(9, 2, 32, size=4))),
    ("SHAPE_MISMATCH", held(scheme=BLOCK.with_level(QuantLevel.block([48])))),
    ("SHAPE_MISMATCH", plain(keys=t(9, 2, 0, 64), values=t(9, 2, 0, 64))),
    ("SHAPE_MISMATCH", plain(keys=t(9, 0, 16, 64), values=t(9, 0, 16, 64))),
    ("SHAPE_MISMATCH", plain(keys=t(9, 2, 16, 64, size=4))),
    ("NON_CONTIGUOUS", held(keys=t(9, 2, 16, 64, size=1, strides=(4096, 2048, 128, 2)))),
    ("NON_CONTIGUOUS", plain(values=t(9, 2, 16, 64, strides=(2048, 1024, 1, 16)))),
    ("TOO_LARGE", plain(keys=t(9, 2, 16, 513), values=t(9, 2, 16, 513))),
    ("TOO_LARGE", plain(keys=t(1 << 27, 2, 16, 64), values=t(1 << 27, 2, 16, 64))),
    ("TOO_LARGE", plain(keys=t(1, 2, 1 << 31, 64), values=t(1, 2, 1 << 31, 64))),
    ("TOO_LARGE", plain(keys=t(9, 16384, 16, 64), values=t(9, 16384, 16, 64))),
    ("UNSUPPORTED_SCHEME", held(scheme=BLOCK.with_level(QuantLevel.Tensor))),
    ("UNSUPPORTED_SCHEME", held(scheme=BLOCK.with_level(QuantLevel.block([2, 32])))),
    ("UNSUPPORTED_SCHEME", held(scheme=BLOCK.with_value(QuantValue.Q4S))),
    ("UNSUPPORTED_SCHEME", words(BLOCK.with_store(QuantStore.U32).with_value(QuantValue.Q2S), 4)),
    ("UNSUPPORTED_SCHEME", words(BLOCK.with_store(QuantStore.U32).with_value(QuantValue.E4M3), 16)),
    ("UNSUPPORTED_SCHEME", words(BLOCK.with_store(QuantStore.U32).with_value(QuantValue.E5M2), 16)),
    ("BLOCK_NOT_DIVISIBLE", words(BLOCK.with_store(QuantStore.U32).with_value(QuantValue.Q4S).with_level(QuantLevel.block([4])), 8)),
    ("BLOCK_NOT_DIVISIBLE", held(scheme=BLOCK.with_value(QuantValue.E2M1).with_level(QuantLevel.block([1])), keys=t(9, 2, 16, 32, size=1), values=t(9, 2, 16, 32, size=1))),
]


@pytest.mark.parametrize("i", range(len(CACHES)))
def test_caches_that_are_refused(i):
    name, c = CACHES[i]
    assert status(append, cache=c) == code(name)
    assert status(attend, cache=c) == code(name)
    assert attention.workspace_bytes(c, t(5, 4, 64), t(3, 4, size=4), BF16) == 0


APPEND = dict(cache=held(), k=t(5, 2, 64), v=t(5, 2, 64), slots=t(5, size=4), elem=BF16, q=t(5, 4, 64), q_out=t(5, 4, 64), positions=t(5, size=4),
              rotary=Rotary(t(32, size=4)))


def append(**other):
    a = dict(APPEND, **other)
    cache.append(CLIENT, a.pop("cache"), a.pop("k"), a.pop("v"), a.pop("slots"), a.pop("elem"), **a)


@pytest.mark.parametrize("name,other", [
    ("INVALID_ARGUMENT", dict(elem=7)),
    ("INVALID_ARGUMENT", dict(k=t(5, 2, 64, ptr=0))),
    ("INVALID_ARGUMENT", dict(v=t(5, 2, 64, ptr=P + 1))),
    ("INVALID_ARGUMENT", dict(slots=t(5, size=4, ptr=P + 2))),
    ("INVALID_ARGUMENT", dict(q=None)),
    ("INVALID_ARGUMENT", dict(q_out=None)),
    ("INVALID_ARGUMENT", dict(positions=None)),
    ("INVALID_ARGUMENT", dict(rotary=None)),
    ("INVALID_ARGUMENT", dict(rotary=Rotary(t(32, size=4), interleaved=2))),
    ("INVALID_ARGUMENT", dict(rotary=Rotary(t(32, size=4, ptr=0)))),
    ("SHAPE_MISMATCH", dict(rotary=Rotary(t(33, size=4)))),
    ("SHAPE_MISMATCH", dict(rotary=Rotary(t(32, size=2)))),
    ("SHAPE_MISMATCH", dict(rotary=Rotary(t(1, 32, size=4)))),
    ("SHAPE_MISMATCH", dict(k=t(5, 128))),
    ("SHAPE_MISMATCH", dict(k=t(5, 3, 64))),
    ("SHAPE_MISMATCH", dict(k=t(5, 2, 32))),
    ("SHAPE_MISMATCH", dict(k=t(5, 2, 64, size=4))),
    ("SHAPE_MISMATCH", dict(v=t(4, 2, 64))),
    ("SHAPE_MISMATCH", dict(slots=t(6, size=4))),
    ("SHAPE_MISMATCH", dict(slots=t(5, size=8))),
    ("SHAPE_MISMATCH", dict(positions=t(4, size=4))),
    ("SHAPE_MISMATCH", dict(q=t(6, 4, 64))),
    ("SHAPE_MISMATCH", dict(q_out=t(5, 3, 64))),
    ("SHAPE_MISMATCH", dict(q=t(5, 256))),
    ("NON_CONTIGUOUS", dict(k=t(5, 2, 64, strides=(256, 128, 2)))),
    ("NON_CONTIGUOUS", dict(slots=t(5, size=4, strides=(2,)))),
    ("NON_CONTIGUOUS", dict(rotary=Rotary(t(32, size=4, strides=(2,))))),
    ("TOO_LARGE", dict(k=t(1 << 24, 2, 64))),
    ("TOO_LARGE", dict(q=t(5, 16384, 64))),
])
def test_appends_that_are_refused(name, other):
    assert status(append, **other) == code(name)


ATTEND = dict(cache=held(), q=t(5, 4, 64), y=t(5, 4, 64), table=t(3, 4, size=4), offsets=t(4, size=4), lengths=t(3, size=4), elem=BF16, scores=Scores())


def attend(**other):
    attention.launch_ref(CLIENT, **dict(ATTEND, **other))


@pytest.mark.parametrize("name,other", [
    ("INVALID_ARGUMENT", dict(elem=-1)),
    ("INVALID_ARGUMENT", dict(q=t(5, 4, 64, ptr=0))),
    ("INVALID_ARGUMENT", dict(y=t(5, 4, 64, ptr=P + 1))),
    ("INVALID_ARGUMENT", dict(table=t(3, 4, size=4, ptr=P + 2))),
    ("INVALID_ARGUMENT", dict(lengths=t(3, size=4, ptr=0))),
    ("INVALID_ARGUMENT", dict(scores=Scores(cap=-1.0))),
    ("INVALID_ARGUMENT", dict(scores=Scores(cap=float("nan")))),
    ("INVALID_ARGUMENT", dict(scores=Scores(cap=float("inf")))),
    ("INVALID_ARGUMENT", dict(scores=Scores(slopes=t(4, size=4, ptr=0)))),
    ("SHAPE_MISMATCH", dict(scores=Scores(slopes=t(2, size=4)))),
    ("SHAPE_MISMATCH", dict(scores=Scores(slopes=t(4, size=2)))),
    ("SHAPE_MISMATCH", dict(scores=Scores(prefix=t(5, size=4)))),
    ("NON_CONTIGUOUS", dict(scores=Scores(prefix=t(3, size=4, strides=(2,))))),
    ("SHAPE_MISMATCH", dict(q=t(5, 3, 64), y=t(5, 3, 64))),
    ("SHAPE_MISMATCH", dict(q=t(5, 4, 32))),
    ("SHAPE_MISMATCH", dict(q=t(5, 256))),
    ("SHAPE_MISMATCH", dict(q=t(5, 4, 64, size=4))),
    ("SHAPE_MISMATCH", dict(y=t(4, 4, 64))),
    ("SHAPE_MISMATCH", dict(table=t(12, size=4))),
    ("SHAPE_MISMATCH", dict(table=t(3, 4, size=8))),
    ("SHAPE_MISMATCH", dict(offsets=t(3, size=4))),
    ("SHAPE_MISMATCH", dict(lengths=t(4, size=4))),
    ("NON_CONTIGUOUS", dict(q=t(5, 4, 64, strides=(256, 1, 4)))),
    ("NON_CONTIGUOUS", dict(table=t(3, 4, size=4, strides=(1, 3)))),
    ("NON_CONTIGUOUS", dict(offsets=t(4, size=4, strides=(2,)))),
    ("TOO_LARGE", dict(q=t(1 << 24, 4, 64), y=t(1 << 24, 4, 64))),
    ("TOO_LARGE", dict(q=t(5, 16384, 64))),
    ("TOO_LARGE", dict(table=t(3, 1 << 28, size=4))),
])
def test_attentions_that_are_refused(name, other):
    assert status(attend, **other) == code(name)


def test_windows_are_numbers_of_32_bits():
    with pytest.raises(OverflowError):
        attend(scores=Scores(window=1 << 32))
    with pytest.raises(OverflowError):
        attend(scores=Scores(window=-1))


@pytest.mark.parametrize("name,tensors,pairs", [
    ("INVALID_ARGUMENT", [t(4, 8)], t(3, 2, size=4, ptr=0)),
    ("INVALID_ARGUMENT", [t(4, 8)], t(3, 2, size=4, ptr=P + 1)),
    ("INVALID_ARGUMENT", [t(4, 8), t(4, 8, ptr=0)], t(3, 2, size=4)),
    ("INVALID_ARGUMENT", [t(4, 8, size=0)], t(3, 2, size=4)),
    ("SHAPE_MISMATCH", [t(4, 8)], t(3, 3, size=4)),
    ("SHAPE_MISMATCH", [t(4, 8)], t(6, size=4)),
    ("SHAPE_MISMATCH", [t(4, 8)], t(3, 2, size=8)),
    ("NON_CONTIGUOUS", [t(4, 8)], t(3, 2, size=4, strides=(1, 3))),
    ("NON_CONTIGUOUS", [t(4, 8), t(4, 8, 2, strides=(32, 4, 1))], t(3, 2, size=4)),
    ("NON_CONTIGUOUS", [t(4, 8, 2, strides=(16, 1, 8))], t(3, 2, size=4)),
    ("TOO_LARGE", [t(4, 8)], t(1 << 24, 2, size=4)),
    ("TOO_LARGE", [t(1 << 31, 8)], t(3, 2, size=4)),
    ("TOO_LARGE", [t(4, 1 << 20, 1 << 20)], t(3, 2, size=4)),
])
def test_copies_that_are_refused(name, tensors, pairs):
    assert status(cache.copy_pages, CLIENT, tensors, pairs) == code(name)


def test_what_is_not_a_handle_is_a_type_error():
    with pytest.raises((TypeError, AttributeError)):
        cache.copy_pages(CLIENT, [3], t(3, 2, size=4))
    with pytest.raises(TypeError):
        cache.copy_pages(CLIENT, 3, t(3, 2, size=4))
    with pytest.raises(TypeError):
        attend(scores=Scores(cap="x"))


def test_nothing_to_do_is_no_error_without_a_gpu():
    append(k=t(0, 2, 64), v=t(0, 2, 64), slots=t(0, size=4), q=t(0, 4, 64), q_out=t(0, 4, 64), positions=t(0, size=4))
    attend(q=t(0, 4, 64), y=t(0, 4, 64))
    attend(table=t(0, 4, size=4), offsets=t(1, size=4), lengths=t(0, size=4))
    cache.copy_pages(CLIENT, [], t(3, 2, size=4))
    cache.copy_pages(CLIENT, [t(4, 8)], t(0, 2, size=4))


def test_frequencies():
    plain_ones = rotary.frequencies(8, 100.0)
    assert plain_ones == [1.0, 100.0 ** -0.25, 100.0 ** -0.5, 100.0 ** -0.75]
    assert rotary.frequencies(8, 100.0, 4.0) == [f / 4.0 for f in plain_ones]
    with pytest.raises(ValueError):
        rotary.frequencies(7)
    parts = rotary.frequencies_by_parts(128, 8.0, 8192)
    assert parts[0] == 1.0 and parts[-1] == rotary.frequencies(128)[-1] / 8.0 and all(a > b for a, b in zip(parts, parts[1:]))
    assert rotary.magnitude(0.5) == 1.0 and abs(rotary.magnitude(8.0) - 1.2079441541679836) < 1e-15
