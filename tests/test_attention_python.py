"""The Python layer in front of include/cubek_attention.h: what it makes of its arguments before the library sees them; no GPU."""
import subprocess
import sys


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
