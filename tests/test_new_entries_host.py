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


@pytest.mark.parametrize("bad", [dict(num_pages=MOST), dict(num_seqs=MOST), dict(num_pages=MOST - 1000), dict(num_seqs=MOST - 1000)])
@pytest.mark.parametrize("name", ["reserve", "trim", "fork", "accept", "accept_table", "compact", "copy"])
def test_state_whose_strips_would_wrap(name, bad):
    # the bookkeeping CTA cuts pages and sequences into strips of whole numbers of 32 bits
    lib = _lib.load()
    arr = (_lib.SfaCachePool * 1)()
    arr[0].base, arr[0].page_stride, arr[0].page_bytes = FAKE, 64, 64
    P = _lib.SfaCacheParams(refcounts=FAKE, block_table=FAKE, cache_seqlens=FAKE, a=FAKE, b=FAKE, out=FAKE, pools=arr,
                            bt_stride=4, a_stride=2, num_pools=1, num_seqs=2, num_pages=8, page_size=16, table_width=4, count=2)
    for n, v in bad.items():
        setattr(P, n, v)
    f = getattr(lib, "sfa_cache_" + name)
    code = f(ctypes.byref(P), None) if name in ("trim", "accept", "accept_table") else f(ctypes.byref(P), None, 0, None)
    assert code == _lib.SFA_ERR_INVALID_ARGUMENT
    assert "sizes" in lib.sfa_last_error_string().decode()
