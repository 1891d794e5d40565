"""Compile-time resources of the paged attention kernels (no GPU): no spills, and the
tcgen05 kernels, which move registers between their warps, are given exactly the count
that the split was made for (an increase waits for registers the CTA has).  Reads only
the summary that `-Xptxas -v` prints."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "rdnattention_b200" / "csrc"
NVCC = "/usr/local/cuda/bin/nvcc"

pytestmark = pytest.mark.skipif(not Path(NVCC).exists() or shutil.which("c++filt") is None,
                                reason="needs nvcc and c++filt")

SOURCE = """
#include "fa_paged_mma.cuh"
using namespace rdna::paged;
#define FEW(E, D, C) template __global__ void rdna::paged::fa_paged_kernel<E, D, C>( \\
    const __grid_constant__ CUtensorMap, const __grid_constant__ CUtensorMap, const __grid_constant__ AttnParams);
#define MANY(E, D) template __global__ void rdna::paged::fa_paged_mma_kernel<E, D>( \\
    const __grid_constant__ CUtensorMap, const __grid_constant__ CUtensorMap, const __grid_constant__ AttnParams);
FEW(F16, 64, false) FEW(F16, 64, true) FEW(F16, 128, false) FEW(F16, 128, true) FEW(F16, 256, false) FEW(F16, 256, true)
MANY(F16, 64) MANY(F16, 128) MANY(BF16, 64) MANY(BF16, 128)
template __global__ void rdna::paged::join_kernel<F16, true>(const __grid_constant__ AttnParams);
template __global__ void rdna::paged::join_kernel<F16, false>(const __grid_constant__ AttnParams);
"""


@pytest.fixture(scope="module")
def report(tmp_path_factory):
    d = tmp_path_factory.mktemp("paged")
    (d / "paged_kernels.cu").write_text(SOURCE.replace("\\\\", "\\"))
    res = subprocess.run([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-lineinfo",
                          "--expt-relaxed-constexpr", f"-I{ROOT / 'include'}", f"-I{CSRC}", "-Xptxas", "-v", "-c",
                          str(d / "paged_kernels.cu"), "-o", str(d / "k.o")], capture_output=True, text=True, check=True)
    parts = re.split(r"Compiling entry function '([^']+)' for 'sm_100a'", res.stderr)
    names = subprocess.run(["c++filt"], input="\n".join(parts[1::2]), capture_output=True, text=True,
                           check=True).stdout.splitlines()
    out = {}
    for name, body in zip(names, parts[2::2]):
        spill = re.search(r"(\d+) bytes spill stores, (\d+) bytes spill loads", body)
        out[name] = (int(re.search(r"Used (\d+) registers", body).group(1)), int(spill.group(1)), int(spill.group(2)))
    return out


def test_no_spills(report):
    assert len([n for n in report if "fa_paged" in n]) == 10
    assert not {n: r for n, r in report.items() if r[1] or r[2]}


def test_register_split(report):
    text = (CSRC / "fa_paged_mma.cuh").read_text()
    launch, softmax, other = map(int, re.search(
        r"LAUNCH_REGS = (\d+), SOFTMAX_REGS = (\d+), OTHER_REGS = (\d+)", text).groups())
    assert 8 * softmax + 4 * other <= 12 * launch <= 65536 // 32
    many = [r[0] for n, r in report.items() if "fa_paged_mma_kernel" in n]
    assert many == [launch] * 4
