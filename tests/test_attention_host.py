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


def test_pages_too_large_for_a_launch_are_refused_before_anything_is_copied():
    """Bytes are copied one by one where a page allows nothing else, 1024 by a workgroup, of which a launch has fewer than 2^24; by fours and sixteens there is room for the largest pages."""
    import pytest

    from cubek_amd import ComputeClient, QuantError, TensorHandleRef, _ffi, cache

    def pool(ptr, page, size=1):
        return TensorHandleRef(ptr, (2, 1 << 10, page >> 10), (page, page >> 10, 1), size)

    pairs = TensorHandleRef(1 << 20, (0, 2), (2, 1), 4)  # nothing to copy: what is taken returns without a GPU
    small, large = pool(1 << 20, 1 << 20), 1 << 34
    cache.copy_pages(ComputeClient(0), [small, pool(1 << 20, large)], pairs)
    cache.copy_pages(ComputeClient(0), [small, pool((1 << 20) + 4, large)], pairs)
    cache.copy_pages(ComputeClient(0), [small, pool((1 << 20) + 1, large - 1024)], pairs)
    for tensors in ([pool((1 << 20) + 1, large)], [small] * 40 + [pool((1 << 20) + 2, large)]):
        with pytest.raises(QuantError) as e:
            cache.copy_pages(ComputeClient(0), tensors, pairs)
        assert e.value.status == _ffi.ERR_TOO_LARGE
