"""Arguments at the edge of the C entries of the rotary and page operations."""
import ctypes

import pytest

from ops_b200 import _lib

FAKE = 0x10000
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("bad", [dict(start=MOST - 1, rot=4), dict(start=MOST, rot=64), dict(start=64, rot=MOST - 1),
                                 dict(start=65, rot=0), dict(start=1, rot=64), dict(start=-1, rot=2)])
def test_rotated_part_outside_the_head(bad):
    # start + rot may pass 31 bits
    lib = _lib.load()
    P = _lib.SfaRotaryParams(num_tensors=1, batch=1, len=4, dim=64, positions=FAKE, frequencies=FAKE)
    P.t[0].x = P.t[0].y = P.t[0].dy = P.t[0].dx = FAKE
    P.t[0].heads, P.t[0].flags = 2, _lib.SFA_ROTARY_TURN
    for n, v in bad.items():
        setattr(P, n, v)
    # a call without a device ends in an error of its own, so a refusal shows by its code
    P.len = 0
    for call in (lambda: lib.sfa_rotary_fwd(ctypes.byref(P), None), lambda: lib.sfa_rotary_bwd(ctypes.byref(P), None, 0, None)):
        assert call() == _lib.SFA_ERR_INVALID_ARGUMENT
        assert "rot" in lib.sfa_last_error_string().decode()
