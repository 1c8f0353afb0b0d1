"""The limits of the products' kernels, walked over sizes up to a card's memory without a GPU."""
import os

from test_matmul_host import ROOT, run


def test_no_size_leaves_the_matrix_cores(tmp_path):
    program = str(tmp_path / "matmul_limits")
    run("/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-O2", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        os.path.join(ROOT, "tests", "cpp", "matmul_limits.hip"), "-o", program)
    assert run(program).endswith("ok\n")
