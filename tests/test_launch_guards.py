"""Every kernel that takes tensor memory checks its launch contract before it
initialises a barrier or allocates: a wrong block or cluster size ends in a status
word, not in a wait. (Read from the source: a launch that breaks the contract is
not made.)"""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "gb300_microbench_b200" / "csrc"
SITES = [(path.name, m.start()) for path in sorted(CSRC.glob("*.cu*")) if path.name != "ptx.cuh"
         for m in re.finditer(r"\btmem_alloc<", path.read_text())]


def test_the_kernels_are_found():
    assert {name for name, _ in SITES} == {"gemm_lowp.cuh", "gemm_sm100.cu", "lowp_linear.cu", "umma_probe.cu"}


@pytest.mark.parametrize("name,at", SITES)
def test_guard_comes_first(name, at):
    text = (CSRC / name).read_text()
    start = max(m.start() for m in re.finditer(r"^(?:extern \"C\" )?(?:static )?__(?:global|device)__", text, re.M) if m.start() < at)
    body = text[start:at]
    guard = body.find("kDevBadLaunch")
    assert guard >= 0, "no launch-contract guard before the allocation"
    for op in ("mbar_init(", "barrier.cluster", "cluster_sync(", "grid_wait(", "__syncthreads("):
        assert op not in body[:guard]
