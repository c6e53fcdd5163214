"""What holds for every kernel source, read as text."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "berth_b200", "csrc")
# instructions in which the lanes of a warp, or the threads of a block or cluster, meet
MEETING = r"redux\.sync|shfl\.sync|vote\.sync|match\.[a-z]+\.sync|elect\.sync|bar\.sync|barrier\.|griddepcontrol"


@pytest.mark.parametrize("path", sorted(glob.glob(os.path.join(CSRC, "*.cu*"))), ids=os.path.basename)
def test_inline_assembly_in_which_lanes_meet_is_volatile(path):
    """A plain asm may be moved to the only place that uses its result; behind a branch, its lanes would wait for lanes that never come."""
    with open(path) as f:
        text = f.read()
    for m in re.finditer(r"\basm\b(\s+volatile\b)?\s*\(((?:[^;\"]|\"[^\"]*\")*)\)\s*;", text):
        if re.search(MEETING, m.group(2)):
            assert m.group(1), f"{os.path.basename(path)}:{text[:m.start()].count(chr(10)) + 1}: {m.group(0)[:80]}"
