"""Argument checks of the 8-bit cache's C entry points at the ends of their ranges, no GPU."""
import pytest

from hs_guard_b200 import _lib
from test_cache8_host import L, _append  # noqa: F401


@pytest.mark.parametrize("count", [2 ** 31 - 1, 2 ** 31 - 4096, 2 ** 31 - 8192])
def test_append_refuses_lists_whose_ends_are_beyond_32_bits(L, count):
    """Threads look up to 4,096 entries past the one they stand at."""
    assert _append(L, count=count, rows=count, hq=0, q=0) == _lib.HSG_ERR_INVALID
    assert "entries" in L.hsg_last_error().decode()
