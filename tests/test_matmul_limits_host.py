"""The limits of the products' kernels and the room they ask for, walked over random sizes without a GPU."""
import os

import pytest

from test_matmul_host import ROOT, run


@pytest.mark.parametrize("name", ["matmul_limits", "matmul_workspace"])
def test_walk(tmp_path, name):
    program = str(tmp_path / name)
    run("/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-O2", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        os.path.join(ROOT, "tests", "cpp", name + ".hip"), "-o", program)
    assert run(program).endswith("ok\n")
