"""Stages of LDS that direct loads fill again: a wavefront's own reads have to be over before the barrier that frees the
stage, and the source has to say so, not the place that a compiler finds for its waits."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pisceslx_amd", "csrc")


@pytest.mark.parametrize("name", ["yvmoe_fp8.hip", "yvmoe_swiglu.hip"])
def test_reads_of_a_stage_end_before_its_barrier(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    barriers = [m.start() for m in re.finditer(r"__builtin_amdgcn_s_barrier\(\)", text)]
    assert barriers
    for at in barriers:
        before = text[:at].split("\n")[-5:]
        line = text.count("\n", 0, at) + 1
        assert any("lgkm0()" in b or "all_done()" in b or "nothing has been read" in b for b in before), f"{name}:{line}"
