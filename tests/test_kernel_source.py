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


def test_one_kernel_s_build_does_not_decide_over_the_library():
    """A kernel that a compiler gives other registers than its split needs is refused where it is launched; what
    prepares a device for every entry fails for the device and for CUDA's errors only."""
    text = (CSRC / "capi.cu").read_text()
    prepare = text.split("int prepare_device(int device, int* sm_count) {")[1].split("\n}\n")[0]
    refusals = [line for line in prepare.splitlines() if "fail(" in line]
    assert len(refusals) == 2 and "bad device" in refusals[0] and "built for sm_100a" in refusals[1]
    launch = text.split("int wamffn_cache_attention(void* stream,")[1].split("\n}\n")[0]
    assert launch.index("registers != kManyLaunchRegs") < launch.index("launch_pdl(kv_attend_many_kernel")
