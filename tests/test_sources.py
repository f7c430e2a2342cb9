"""What the library's sources keep out, for reasons that no result shows."""
import os

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tannic_amd", "csrc")
SOURCES = [os.path.join(at, name) for at, _, names in os.walk(CSRC) for name in names if name.endswith((".hip", ".hpp", ".cpp"))]


@pytest.mark.parametrize("source", SOURCES, ids=lambda s: os.path.relpath(s, CSRC))
def test_memory_is_cleared_by_kernels(source):
    """A recorded memset has given wrong values on replays after the first: memory that calls use is cleared by kernels, recorded or not."""
    with open(source) as f:
        assert "hipMemset" not in f.read()
