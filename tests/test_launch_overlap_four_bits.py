"""Products with 4-bit weights that start before their predecessor has ended: the weight is read behind the wait unless the caller says that it is complete.
Read from the sources (a race on the weight is not tried out on a GPU)."""
import os
import re

import pytest

from test_launch_overlap import CSRC, kernels_of

WAIT = re.compile(r"if \(!A\.early\) pdl_wait\(\);")


@pytest.mark.parametrize("file", ["linear4_mma.cu", "linear4_tc.cu"])
def test_the_weight_is_read_behind_the_wait(file):
    found = 0
    for name, _, body in kernels_of(os.path.join(CSRC, file)):
        uses = [m.start() for m in re.finditer(r"\bfetch\((?!Codes<PER>&)[^)]*\)", body)]       # (what calls the copies of the weight)
        assert uses, name
        wait = WAIT.search(body)
        assert wait and wait.end() < min(uses), f"{name} reads the weight before it has waited"
        found += 1
    assert found == 1


def test_the_general_kernel_waits_first():
    for name, _, body in kernels_of(os.path.join(CSRC, "linear4.cu")):
        assert body.index("pdl_overlap_few()") < body.index("A.weight"), name
