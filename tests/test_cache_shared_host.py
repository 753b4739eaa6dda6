"""Acceptance in shared pages, what needs no GPU: refusals, and the oracle's own
answer for a fork of drafted rows."""
import ctypes

import pytest
import torch

import ops_b200
from ops_b200 import _lib
from oracle import cache_oracle as C


@pytest.mark.parametrize("refs,msg", [(torch.zeros(5, dtype=torch.int32), "refcounts"), (torch.zeros(6), "refcounts"),
                                      (torch.zeros(6, 1, dtype=torch.int32), "refcounts"),
                                      (torch.zeros(12, dtype=torch.int32)[::2], "contiguous"),
                                      (torch.zeros(6, dtype=torch.int32), "CUDA"), (None, "CUDA")])
def test_refusals(refs, msg):
    i = dict(dtype=torch.int32)
    with pytest.raises(ValueError, match=msg):
        ops_b200.paged_cache_accept([torch.zeros(6, 8, 2)], torch.zeros(3, 4, **i), torch.zeros(3, **i), torch.zeros(3, 2, **i),
                                    torch.zeros(3, **i), refcounts=refs)


def test_c_abi_refusals():
    lib, fake = _lib.load(), 0x10000
    arr = (_lib.SfaCachePool * 1)()
    arr[0].base, arr[0].page_stride, arr[0].page_bytes = fake, 4096, 4096

    def params(**kw):
        P = _lib.SfaCacheParams(refcounts=fake, block_table=fake, cache_seqlens=fake, a=fake, b=fake, out=fake, pools=arr,
                                bt_stride=4, a_stride=2, num_pools=1, num_seqs=2, num_pages=8, page_size=16, table_width=4, count=2)
        for n, v in kw.items():
            setattr(P, n, v)
        return P

    for bad, msg in ((dict(num_pages=-1), "sizes"), (dict(page_size=0), "page_size"), (dict(block_table=None), "block_table"),
                     (dict(cache_seqlens=None), "cache_seqlens"), (dict(refcounts=None), "refcounts"), (dict(a=None), "arrays"),
                     (dict(b=None), "arrays"), (dict(out=None), "arrays"), (dict(pools=None), "pools")):
        assert lib.sfa_cache_accept_table(ctypes.byref(params(**bad)), None) == _lib.SFA_ERR_INVALID_ARGUMENT, bad
        assert msg in lib.sfa_last_error_string().decode(), bad
    assert lib.sfa_cache_accept_table(None, None) == _lib.SFA_ERR_INVALID_ARGUMENT
    assert lib.sfa_cache_accept_table(ctypes.byref(params(num_seqs=0, refcounts=None, num_pages=0)), None) == _lib.SFA_OK


def test_oracle_leaves_shared_pages_alone():
    pool = torch.arange(6 * 4).view(6, 4, 1)
    table, lens, refs = [[0, 1, -1], [-1] * 3], [8, 0], [1, 1, 0, 0, 0, 0]
    assert C.fork(refs, table, lens, [0], [1], [pool]) == [1] and refs[:2] == [2, 2]
    before = pool.clone()
    assert C.accept([pool], table, lens, [[1, 3], [0, 2]], [6, 6]) == [-1, -1]
    assert C.accept([pool], table, lens, [[0, 1], [-1, -1]], [6, 6], refs) == [4, 2]
    assert torch.equal(pool, before)
    C.trim(refs, table, lens, [-1, 0], 4)
    assert C.accept([pool], table, lens, [[1, 3], [-1, -1]], [6, 0]) == [4, 0]
    assert pool[0, 2:, 0].tolist() == [3, 5]
