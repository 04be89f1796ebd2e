"""Refusals of the paged-cache calls that came after the operators themselves: no GPU needed."""
import pytest

from anedvd_b200 import runtime as rt


@pytest.mark.parametrize("limit_us", [0, 1000001, 0xFFFFFFFF])
def test_the_wait_probe_is_bounded(limit_us):
    assert rt.load().cuq_paged_wait_probe(limit_us, None) == rt.EINVAL
    assert "limit" in rt.last_error()
