"""What the compiler needs for the attention kernels: registers that spill into scratch memory cost a step more than it computes, so none is to be read there in a loop."""
import os
import re
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cubek_amd", "csrc")


def compiled(kernel, code):
    """{name: figures} of the kernels of one object, from the compiler's own remarks; flags as the Makefile has them."""
    make = subprocess.run(["make", "-n", "-B", "-C", CSRC], capture_output=True, text=True, check=True).stdout
    line = next(x for x in make.splitlines() if f"cq_kernels_attention_{kernel}_{code}.o" in x and " -c " in x)
    flags = line.split(" -o ")[0].split() + ["--cuda-device-only", "-o", os.devnull, "-Rpass-analysis=kernel-resource-usage"]
    text = subprocess.run(flags, capture_output=True, text=True, check=True, cwd=CSRC).stderr
    found = {}
    for part in text.split("Function Name: ")[1:]:
        found[part.split()[0]] = {k: int(v) for k, v in re.findall(r"remark: .*?\b(VGPRs Spill|ScratchSize \[bytes/lane\]): (\d+)", part)}
    return found


@pytest.fixture(scope="module")
def kernels():
    with ThreadPoolExecutor(4) as pool:
        jobs = {(kernel, code): pool.submit(compiled, kernel, code) for kernel in ("few", "many") for code in (0, 1, 2, 5)}  # 3 and 4 are the like of 2 and 1
        return {key: job.result() for key, job in jobs.items()}


def test_no_kernel_of_few_rows_spills(kernels):
    for (kernel, code), of in kernels.items():
        if kernel == "few":
            assert len(of) >= 8
            assert all(figures["VGPRs Spill"] == 0 for figures in of.values()), (code, of)


def test_kernels_of_many_rows_put_away_four_registers_at_most(kernels):
    """Heads of 64, in front of their loop; they take them back behind it."""
    for (kernel, code), of in kernels.items():
        if kernel == "many":
            assert len(of) >= 6
            for name, figures in of.items():
                assert figures["VGPRs Spill"] <= (4 if "ELi64E" in name else 0), (code, name, figures)
