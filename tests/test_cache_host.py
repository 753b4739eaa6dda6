"""Page operations, what needs no GPU: struct layouts, and the refusals of the
Python surface and of the C ABI."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

import ops_b200
from ops_b200 import _lib

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "sfa_b200.h")


@pytest.mark.parametrize("struct", ["SfaCachePool", "SfaCacheParams"])
def test_struct_layout_matches_header(struct):
    cls = getattr(_lib, struct)
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){",
             f'printf("%zu\\n", sizeof({struct}));']
    lines += [f'printf("%zu\\n", offsetof({struct}, {f[0]}));' for f in cls._fields_] + ["return 0;}"]
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "t.c"), "w").write("\n".join(lines))
        subprocess.run(["gcc", os.path.join(d, "t.c"), "-o", os.path.join(d, "t")], check=True)
        out = [int(x) for x in subprocess.run([os.path.join(d, "t")], capture_output=True, text=True, check=True).stdout.split()]
    assert out == [ctypes.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]


def ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def pool(*shape):
    return torch.zeros(*shape)


GOOD = dict(refs=ints(6), table=ints(3, 4), lens=ints(3), rows=ints(3), pools=[pool(6, 8, 2), pool(6, 8, 5)], pairs=ints(2))

CALLS = {
    "reserve": lambda a: ops_b200.paged_cache_reserve(a["refs"], a["table"], a["lens"], a["rows"], 8),
    "trim": lambda a: ops_b200.paged_cache_trim(a["refs"], a["table"], a["lens"], a["rows"], 8),
    "fork": lambda a: ops_b200.paged_cache_fork(a["refs"], a["table"], a["lens"], a["pairs"], a["pairs"], a["pools"]),
    "accept": lambda a: ops_b200.paged_cache_accept(a["pools"], a["table"], a["lens"], a.get("acc", ints(3, 2)), a["rows"]),
    "compact": lambda a: ops_b200.paged_cache_compact(a["refs"], a["table"], a["pools"]),
    "copy": lambda a: ops_b200.paged_cache_copy(a["pools"], a["pairs"], a["pairs"]),
}


@pytest.mark.parametrize("op", CALLS)
@pytest.mark.parametrize("bad,msg,ops", [
    (dict(), "CUDA", None),
    (dict(refs=torch.zeros(6)), "refcounts", ("reserve", "trim", "fork", "compact")),
    (dict(refs=ints(12)[::2]), "contiguous", ("reserve", "trim", "fork", "compact")),
    (dict(refs=ints(7)), "same pages", ("fork", "compact")),
    (dict(table=ints(3, 4).long()), "block_table", ("reserve", "trim", "fork", "accept", "compact")),
    (dict(table=ints(3, 8)[:, ::2]), "contiguous", ("reserve", "trim", "fork", "accept", "compact")),
    (dict(lens=ints(2)), "cache_seqlens", ("reserve", "trim", "fork", "accept")),
    (dict(rows=ints(4)), "entries", ("reserve", "trim", "accept")),
    (dict(acc=ints(3)), "accepted", ("accept",)),
    (dict(pairs=torch.zeros(2)), "src", ("fork", "copy")),
    (dict(pools=[]), "at least one", ("fork", "accept", "compact", "copy")),
    (dict(pools=[pool(6, 8, 2), pool(6, 4, 5)]), "same pages", ("fork", "accept", "compact", "copy")),
    (dict(pools=[pool(6, 2, 8).transpose(1, 2)]), "contiguous", ("fork", "accept", "compact", "copy")),
    (dict(pools=[pool(1, 8, 2).expand(6, 8, 2)]), "overlap", ("fork", "accept", "compact", "copy")),
    (dict(pools=[pool(6)]), "every pool", ("fork", "accept", "compact", "copy")),
])
def test_refusals(op, bad, msg, ops):
    if ops is not None and op not in ops:
        return
    with pytest.raises(ValueError, match=msg):
        CALLS[op]({**GOOD, **bad})


def test_what_would_be_moved_twice_is_refused():
    one = pool(6, 8, 2)
    for op in ("fork", "accept", "compact", "copy"):
        with pytest.raises(ValueError, match="twice"):
            CALLS[op]({**GOOD, "pools": [one, pool(6, 8, 5), one]})
        with pytest.raises(ValueError, match="CUDA"):                      # nothing in them: nothing moves
            CALLS[op]({**GOOD, "pools": [pool(6, 8, 0), pool(6, 8, 0)]})
    for op in ("reserve", "trim", "fork", "compact"):
        with pytest.raises(ValueError, match="overlap"):
            CALLS[op]({**GOOD, "table": ints(1, 4).expand(3, 4)})


def test_page_size_is_checked():
    for f in (ops_b200.paged_cache_reserve, ops_b200.paged_cache_trim):
        with pytest.raises(ValueError, match="page_size"):
            f(GOOD["refs"], GOOD["table"], GOOD["lens"], GOOD["rows"], 0)


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

    def code(name, P):
        f = getattr(lib, "sfa_cache_" + name)
        return f(ctypes.byref(P), None) if name in ("trim", "accept") else f(ctypes.byref(P), None, 0, None)

    for bad, msg, names in (
            (dict(num_pages=-1), "sizes", ("reserve", "trim", "fork", "accept", "compact", "copy")),
            (dict(page_size=0), "page_size", ("reserve", "trim", "fork", "accept", "compact", "copy")),
            (dict(refcounts=None), "refcounts", ("reserve", "trim", "fork")),
            (dict(block_table=None), "block_table", ("reserve", "trim", "fork", "accept", "compact")),
            (dict(a=None), "arrays", ("reserve", "trim", "fork", "accept", "copy")),
            (dict(b=None), "arrays", ("fork", "accept", "copy")), (dict(out=None), "output", ("reserve", "compact", "copy")),
            (dict(pools=None), "pools", ("fork", "accept", "compact", "copy"))):
        for name in names:
            assert code(name, params(**bad)) == _lib.SFA_ERR_INVALID_ARGUMENT, (name, bad)
            assert msg in lib.sfa_last_error_string().decode(), (name, bad)
    for field, value, msg in (("page_bytes", 4090, "multiple"), ("page_stride", 100, "page_stride"), ("base", None, "base")):
        keep = getattr(arr[0], field)
        setattr(arr[0], field, value)
        assert code("copy", params()) == _lib.SFA_ERR_INVALID_ARGUMENT
        assert msg in lib.sfa_last_error_string().decode()
        setattr(arr[0], field, keep)
    need = lib.sfa_cache_workspace_bytes(ctypes.byref(params()))
    assert need > 0
    for name in ("reserve", "fork", "compact", "copy"):
        f = getattr(lib, "sfa_cache_" + name)
        assert f(ctypes.byref(params()), 0x10000, need - 1, None) == _lib.SFA_ERR_WORKSPACE
        assert f(ctypes.byref(params()), 0x10001, need, None) == _lib.SFA_ERR_WORKSPACE
