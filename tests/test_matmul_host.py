"""What of the products needs no GPU: the header stands on its own, choices and grids hold over random shapes."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = os.path.join(ROOT, "include")


def run(*command):
    proc = subprocess.run(command, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert proc.returncode == 0, proc.stdout
    return proc.stdout


def test_header_is_c99_and_cpp(tmp_path):
    source = '#include "cubek_matmul.h"\nint main(void) { cq_epilogue e = {0, 0, 0, 0}; return (int)e.gated + CQ_ACT_IDENTITY; }\n'
    for compiler, std, suffix in (("gcc", "c99", ".c"), ("g++", "c++17", ".cpp")):
        path = tmp_path / f"tu{suffix}"
        path.write_text(source)
        run(compiler, f"-std={std}", "-fsyntax-only", "-Wall", "-Wextra", "-pedantic", "-Werror", f"-I{INCLUDE}", str(path))


def test_choices_fit_and_grids_hold_every_tile_once(tmp_path):
    program = str(tmp_path / "matmul_choices")
    run("/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-O2", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
        os.path.join(ROOT, "tests", "cpp", "matmul_choices.hip"), "-o", program)
    assert run(program).endswith("ok\n")
