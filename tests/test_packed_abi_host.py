"""What the packed products' C entry points refuse before any CUDA call, beyond test_feedforward_host."""
import ctypes

import pytest


@pytest.mark.parametrize("per", [1 << 30, 1 << 32, (1 << 32) + 2, 1 << 62])
def test_slots_per_row_beyond_32_bits(per):
    """A count of slots per row of x that an int does not hold is refused, not cut (2^32 would stand for rows in the plan's order)."""
    from mxq import _lib
    L = _lib.lib()
    spec = _lib.MxqProductSpec(4, 3, 4, 3, 0, 0, 0, 0, 0)
    none = None
    # no rows of w: nothing would be launched
    rc = L.mxq_experts_packed(64, none, 64, 2, 64, none, 64, 2, 0, 64, none, none, 4, per, ctypes.byref(spec), none, none, none, none, 0,
                              none)
    assert rc == _lib.ERR_VALUE and b"do not serve" in L.mxq_last_error()
