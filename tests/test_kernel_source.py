"""CPU: rules that the kernels' sources keep, for faults that no run shows reliably."""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "waminfer_b200" / "csrc"


@pytest.mark.parametrize("name", ["attention.cuh", "gemm.cuh", "kvattend_many.cuh", "pass.cuh"])
def test_the_verdict_of_a_wait_reaches_the_warp_with_its_memory(name):
    """Where one lane waits for the warp, the others read or overwrite what the wait was for.  A shuffle alone
    orders no memory, so the verdict goes through warp_verdict, which ends in a warp barrier."""
    text = (CSRC / name).read_text()
    assert not re.findall(r"__shfl_sync\(0xffffffffu, (?:int\()?\w*(?:ok|go|got)\)?, 0\)", text)
    assert text.count("warp_verdict(") >= 4
    helper = (CSRC / "ptx.cuh").read_text().split("int warp_verdict(int found) {")[1].split("\n}")[0]
    assert helper.index("__shfl_sync") < helper.index("__syncwarp();")
