"""Host-side properties of include/cubek_attention.h and its library; no GPU."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_header_is_c99_and_cpp(tmp_path):
    source = '#include "cubek_attention.h"\nint main(void) { cq_scores s = {0}; cq_rotary r = {0, 1.0f, 0}; return (int)s.window + (int)r.interleaved; }\n'
    for compiler, std, suffix in (("gcc", "c99", ".c"), ("g++", "c++17", ".cpp")):
        path = tmp_path / ("header" + suffix)
        path.write_text(source)
        subprocess.run([compiler, f"-std={std}", "-Wall", "-Wextra", "-Werror", "-Wno-missing-field-initializers", "-fsyntax-only", "-I", os.path.join(ROOT, "include"), str(path)], check=True)


def test_every_attention_object_is_built_without_packed_f32_and_contraction():
    """What a product's FMAs are is written out; packed f32 instructions are not to be made."""
    out = subprocess.run(["make", "-n", "-B", "-C", os.path.join(ROOT, "cubek_amd", "csrc")], capture_output=True, text=True, check=True).stdout
    lines = [line for line in out.splitlines() if "hipcc" in line and " -c " in line and ("attention" in line or "kernels_cache" in line or "kernels_pages" in line)]
    assert len(lines) >= 18
    for line in lines:
        assert "-packed-fp32-ops" in line and "-ffp-contract=off" in line and "--offload-arch=gfx950" in line, line
