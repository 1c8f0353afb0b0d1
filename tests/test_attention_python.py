"""The Python layer in front of include/cubek_attention.h: what it makes of its arguments before the library sees them; no GPU."""
import subprocess
import sys

import pytest

from cubek_amd import Cache, ComputeClient, ElemType, QuantError, TensorHandleRef, _ffi, attention, rotary


def test_a_list_of_tensors_that_changes_while_it_is_read():
    """What stands for a tensor may run code of its own (as_c), which empties the list it is read from: the call sees the tensors that it was given."""
    code = """
import ctypes
from cubek_amd import ComputeClient, TensorHandleRef, cache
class Emptying:
    def as_c(self):
        tensors.clear()
        return TensorHandleRef(1 << 20, (4, 8), (8, 1), 2).as_c()
pairs = TensorHandleRef(1 << 20, (0, 2), (2, 1), 4)
tensors = [Emptying()] + [TensorHandleRef((1 << 20) + 64 * i, (4, 8), (8, 1), 2) for i in range(50)]
cache.copy_pages(ComputeClient(0), tensors, pairs)
print("read")
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.strip() == "read", run.stderr[-300:]


@pytest.mark.parametrize("shape", [(), (5, 4, 0), (0,)])
def test_queries_without_entries_are_refused_by_the_library(shape):
    """The scale that stands for none given is worked out of the heads' size, where there is one."""
    t = lambda s, size: TensorHandleRef(1 << 20, s, tuple(1 for _ in s), size)  # noqa: E731
    held = Cache(TensorHandleRef(1 << 20, (9, 2, 16, 64), (2048, 1024, 64, 1), 2), TensorHandleRef(1 << 20, (9, 2, 16, 64), (2048, 1024, 64, 1), 2))
    with pytest.raises(QuantError) as e:
        attention.launch_ref(ComputeClient(0), held, t(shape, 2), t(shape, 2), t((3, 4), 4), t((4,), 4), t((3,), 4), ElemType.BF16)
    assert e.value.status in (_ffi.ERR_SHAPE_MISMATCH, _ffi.ERR_INVALID_ARGUMENT)


def test_a_ramp_of_frequencies_by_parts():
    """Pairs by the number of times they turn within the trained length: with base e^4 and 16 entries, pair i turns trained / (2 pi) e^(-i / 2) times; more than 32 times: as it is; less than
    once: slowed; between the indexes of both, rounded outwards, in a straight line."""
    import math

    base, trained, factor = math.exp(4.0), 600, 8.0
    plain = rotary.frequencies(16, base)
    turns = [trained * f / (2 * math.pi) for f in plain]
    low = math.floor(2 * math.log(trained / (32 * 2 * math.pi)))  # 2
    high = math.ceil(2 * math.log(trained / (2 * math.pi)))       # 10
    got = rotary.frequencies_by_parts(16, factor, trained, base)
    assert (low, high) == (2, 10)
    for i, (f, n, g) in enumerate(zip(plain, turns, got)):
        share = min(1.0, max(0.0, (i - low) / (high - low)))
        assert abs(g - f * ((1.0 - share) + share / factor)) <= 1e-15 * f
        if n > 32:
            assert g == f
    # within one length that turns every pair less than once all are slowed, and where all turn often none is
    assert rotary.frequencies_by_parts(16, factor, 4, base) == [f / factor for f in plain]
    assert rotary.frequencies_by_parts(16, factor, 10 ** 7, base) == plain
