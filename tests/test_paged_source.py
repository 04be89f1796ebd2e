"""What the paged-cache kernels' order rests on, read from their source: no GPU needed.  They are resident while the
kernels before them still write (programmatic dependent launch), so a slip here shows on a GPU only by chance."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "anedvd_b200", "csrc")
FILES = ["paged.cu", "paged.cuh", "paged_attn.cu", "paged_attn_tc.cu", "paged_mass.cu", "paged_tc.cuh"]


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


@pytest.mark.parametrize("name", FILES)
def test_no_read_takes_the_read_only_path(name):
    """ld.global.nc is for data that no one writes while the kernel lives; that of an earlier grid in flight is not."""
    found = re.findall(r"__ldg\b|\bld\.global\.nc\b|__restrict__", source(name))
    assert not found
