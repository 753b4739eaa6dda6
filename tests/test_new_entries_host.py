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


@pytest.mark.parametrize("bad", [dict(num_seqs=MOST, h_q=MOST, h_kv=MOST), dict(num_seqs=2 ** 30, h_q=2 ** 30, h_kv=2 ** 30, table_width=2 ** 20),
                                 dict(num_seqs=2 ** 31 - 100, h_q=1, h_kv=1, table_width=1), dict(num_seqs=2 ** 16, h_q=2 ** 15, h_kv=2 ** 15)])
def test_tree_units_that_would_wrap(bad):
    # sequences times heads times tiles (or chunks) may pass 64 bits
    lib = _lib.load()
    P = _lib.SfaTreeParams(q=FAKE, k=FAKE, v=FAKE, block_table=FAKE, cache_seqlens=FAKE, cu_seqlens=FAKE, o=FAKE, lse=FAKE,
                           q_st=512, q_sh=64, k_st=128, k_sh=64, v_st=128, v_sh=64, o_st=512, o_sh=64, l_st=8, l_sh=1,
                           bt_stride=4, num_seqs=2, total_q=6, max_q=4, max_k=64, h_q=8, h_kv=2, d_qk=64, d_v=64, num_pages=8,
                           page_size=16, table_width=0, scale=0.125)
    for n, v in bad.items():
        setattr(P, n, v)
    assert lib.sfa_tree_attention(ctypes.byref(P), None, 0, None) == _lib.SFA_ERR_UNSUPPORTED
    assert lib.sfa_tree_workspace_bytes(ctypes.byref(P)) == 0
