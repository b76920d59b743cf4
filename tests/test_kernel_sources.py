"""Headers define no kernels: every source that includes one would compile its own copy."""
import pytest

import build as B

HEADERS = sorted(B.CSRC.glob("*.h"))


@pytest.mark.parametrize("header", HEADERS, ids=lambda p: p.name)
def test_no_kernel_in_a_header(header):
    assert "__global__" not in header.read_text()
