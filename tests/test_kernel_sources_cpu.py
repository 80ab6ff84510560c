"""What the sources of the kernels promise and a run cannot show."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "swiglu-recompute_b200", "csrc")


def _code(path):
    with open(path) as f:
        text = f.read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


EARLY = [p for p in sorted(glob.glob(os.path.join(CSRC, "*.cu*")))
         if os.path.basename(p) not in ("ptx.cuh", "host.cuh") and "wait_for_previous()" in _code(p)]


def test_the_early_kernels_are_found():
    assert {os.path.basename(p) for p in EARLY} >= {"norm.cu", "gradnorm.cu", "mxfp4.cu", "tc_mxfp4.cuh"}


@pytest.mark.parametrize("path", EARLY, ids=os.path.basename)
def test_kernels_placed_early_keep_off_the_read_only_path(path):
    """A kernel that starts while the previous one still writes its input (and
    gradient scaling, which writes what it reads) may not call the input read-only
    for its whole life: no __ldg, no ld.global.nc, no __restrict__."""
    found = re.findall(r"__ldg\w*|ld\.global\.nc|__restrict__", _code(path))
    assert not found, (os.path.basename(path), found)
