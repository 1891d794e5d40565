"""Compile-time resources of the few-rows paged kernels and the join in bf16, as
test_paged_resources_cpu.py checks them in fp16 (no GPU): no spills."""
import pytest

import test_paged_resources_cpu as fp16

pytestmark = fp16.pytestmark


@pytest.fixture(scope="module")
def report(tmp_path_factory):
    text = fp16.SOURCE.replace("FEW(F16, ", "FEW(BF16, ").replace("join_kernel<F16", "join_kernel<BF16")
    text = "\n".join(line for line in text.splitlines() if not line.startswith("MANY("))
    saved, fp16.SOURCE = fp16.SOURCE, text
    try:
        return fp16.report.__wrapped__(tmp_path_factory)
    finally:
        fp16.SOURCE = saved


def test_no_spills_in_bf16(report):
    assert len([n for n in report if "fa_paged_kernel" in n and "BF16" in n]) == 6
    assert len([n for n in report if "join_kernel" in n and "BF16" in n]) == 2
    assert not {n: r for n, r in report.items() if r[1] or r[2]}
