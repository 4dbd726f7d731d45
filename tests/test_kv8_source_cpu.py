"""What the 8-bit KV kernels' sources have to keep to where a run could not show it: an instruction that is
undefined when a warpgroup's warps execute it apart."""

import re
from pathlib import Path

import quail_b200

CSRC = Path(quail_b200.__file__).parent / "csrc"


def test_setmaxnreg_is_executed_by_whole_warpgroups():
    # `setmaxnreg.sync.aligned` has to be the same instruction for all four warps of a warpgroup: it stands
    # directly under a branch on whole warpgroups, one for each, and the shares add up to the launch's registers
    text = (CSRC / "attention_kv8_tc.cu").read_text()
    found = re.findall(r"\n *([^\n]*)\n *asm volatile\(\"setmaxnreg\.(dec|inc)\.sync\.aligned\.u32 (\d+);\"\);", text)
    assert text.count("setmaxnreg.") == len(found)
    assert [(branch, int(n)) for branch, _, n in found] == [
        ("if (warp < 4) {", 88), ("} else if (warp >= 12) {", 72), ("} else {", 176)]
    assert "constexpr int kThreads = 512;" in text
    assert 128 * (88 + 2 * 176 + 72) == 512 * 128
