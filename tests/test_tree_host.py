"""Tree attention, what needs no GPU: the struct layout, the refusals of the
Python surface and of the C ABI, and the oracle against a dense restatement."""
import ctypes
import math
import os
import subprocess
import tempfile

import pytest
import torch

import ops_b200
from ops_b200 import _lib
from oracle import tree_oracle as O

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "sfa_b200.h")


def test_struct_layout_matches_header():
    cls = _lib.SfaTreeParams
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void){",
             'printf("%zu\\n", sizeof(SfaTreeParams));']
    lines += [f'printf("%zu\\n", offsetof(SfaTreeParams, {f[0]}));' for f in cls._fields_] + ["return 0;}"]
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "t.c"), "w").write("\n".join(lines))
        subprocess.run(["gcc", os.path.join(d, "t.c"), "-o", os.path.join(d, "t")], check=True)
        out = [int(x) for x in subprocess.run([os.path.join(d, "t")], capture_output=True, text=True, check=True).stdout.split()]
    assert out == [ctypes.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]


def args():
    bf = torch.bfloat16
    return dict(q=torch.zeros(6, 8, 64, dtype=bf), k_cache=torch.zeros(5, 16, 2, 64, dtype=bf),
                v_cache=torch.zeros(5, 16, 2, 64, dtype=bf), block_table=torch.zeros(2, 3, dtype=torch.int32),
                cache_seqlens=torch.full((2,), 9, dtype=torch.int32), parents=torch.full((6,), -1, dtype=torch.int32),
                cu_seqlens=torch.tensor([0, 2, 6], dtype=torch.int32))


@pytest.mark.parametrize("bad,msg", [
    (dict(), "CUDA"), (dict(q=torch.zeros(6, 8, 64)), "bfloat16 or float16"), (dict(q=torch.zeros(6, 512, dtype=torch.bfloat16)), "total"),
    (dict(k_cache=torch.zeros(5, 16, 2, 64).half()), "q's type"), (dict(k_cache=torch.zeros(5, 16, 2, 32, dtype=torch.bfloat16)), "head size"),
    (dict(v_cache=torch.zeros(5, 8, 2, 64, dtype=torch.bfloat16)), "same pages"), (dict(v_cache=torch.zeros(5, 16, 128, dtype=torch.bfloat16)), "page pool"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), "int32"), (dict(cache_seqlens=torch.zeros(3, dtype=torch.int32)), "same number"),
    (dict(cu_seqlens=None), "one row"), (dict(cu_seqlens=torch.zeros(2, dtype=torch.int32)), "cu_seqlens"),
    (dict(parents=torch.zeros(5, dtype=torch.int32)), "parents"), (dict(parents=torch.zeros(6)), "parents"),
    (dict(attn_sink=torch.zeros(2)), "attn_sink"),
])
def test_refusals(bad, msg):
    with pytest.raises(ValueError, match=msg):
        ops_b200.tree_attention_paged(**{**args(), **bad})


def params(**kw):
    fake = 0x10000
    P = _lib.SfaTreeParams(q=fake, k=fake, v=fake, block_table=fake, cache_seqlens=fake, cu_seqlens=fake, o=fake, lse=fake,
                           q_st=512, q_sh=64, k_st=128, k_sh=64, v_st=128, v_sh=64, o_st=512, o_sh=64, l_st=8, l_sh=1,
                           bt_stride=4, num_seqs=2, total_q=6, max_q=4, max_k=64, h_q=8, h_kv=2, d_qk=64, d_v=64, num_pages=8,
                           page_size=16, table_width=4, scale=0.125)
    for n, v in kw.items():
        setattr(P, n, v)
    return P


@pytest.mark.parametrize("bad,code,msg", [
    (dict(h_kv=3), "INVALID_ARGUMENT", "multiple"), (dict(page_size=0), "INVALID_ARGUMENT", "page_size"),
    (dict(d_qk=60), "UNSUPPORTED", "head dims"), (dict(d_v=264), "UNSUPPORTED", "head dims"),
    (dict(dtype=2), "UNSUPPORTED", "bf16"), (dict(scale=0.0), "INVALID_ARGUMENT", "scale"),
    (dict(scale=float("nan")), "INVALID_ARGUMENT", "scale"), (dict(scale=float("inf")), "INVALID_ARGUMENT", "scale"),
    (dict(parents=0x10000, max_q=257), "INVALID_ARGUMENT", "256"), (dict(q=None), "INVALID_ARGUMENT", "non-NULL"),
    (dict(block_table=None), "INVALID_ARGUMENT", "block_table"), (dict(k_st=124), "INVALID_ARGUMENT", "strides"),
    (dict(q_sh=0), "INVALID_ARGUMENT", "strides"), (dict(v=0x10008), "INVALID_ARGUMENT", "aligned"),
    (dict(num_pages=2 ** 30, page_size=2), "UNSUPPORTED", "rows"), (dict(table_width=2 ** 30, page_size=64), "UNSUPPORTED", "table"),
    (dict(max_q=32 * 65535 + 1), "UNSUPPORTED", "too many drafted rows"),
    (dict(num_seqs=2 ** 15, max_q=32 * 40000, table_width=1), "UNSUPPORTED", "too many drafted rows"),
    (dict(num_seqs=-1), "INVALID_ARGUMENT", "sizes"), (dict(cu_seqlens=None, total_q=1), "INVALID_ARGUMENT", "one row"),
])
def test_c_abi_refusals(bad, code, msg):
    lib = _lib.load()
    P = params(**bad)
    assert lib.sfa_tree_attention(ctypes.byref(P), None, 0, None) == getattr(_lib, "SFA_ERR_" + code)
    assert msg in lib.sfa_last_error_string().decode()
    assert lib.sfa_tree_workspace_bytes(ctypes.byref(P)) == 0


def test_workspace_is_asked_for():
    lib = _lib.load()
    P = params()
    need = lib.sfa_tree_workspace_bytes(ctypes.byref(P))
    assert need > 0
    for ws, size in ((None, need), (0x10000, need - 1), (0x10010, need)):
        assert lib.sfa_tree_attention(ctypes.byref(P), ws, size, None) == _lib.SFA_ERR_WORKSPACE
    P = params(total_q=0, num_seqs=0)
    assert lib.sfa_tree_attention(ctypes.byref(P), None, 0, None) == _lib.SFA_OK


def test_oracle_against_a_dense_mask():
    g = torch.Generator().manual_seed(0)
    kc, vc = torch.randn(4, 4, 1, 8, generator=g), torch.randn(4, 4, 1, 8, generator=g)
    table, lens = torch.tensor([[2, 0, 3]]), torch.tensor([10])
    q, par = torch.randn(4, 2, 8, generator=g), torch.tensor([-1, 0, 0, 2])
    o, lse, _, _ = O.tree_attention(q, kc, vc, table, lens, par, cu_seqlens=torch.tensor([0, 4]))
    k, v = (c[table[0]].flatten(0, 1)[:10, 0].double() for c in (kc, vc))
    mask = torch.zeros(4, 10, dtype=torch.bool)
    mask[:, :6] = True
    for j, seen in enumerate(([0], [0, 1], [0, 2], [0, 2, 3])):
        for i in seen:
            mask[j, 6 + i] = True
    sc = (torch.einsum("nhd,kd->nhk", q.double(), k) / math.sqrt(8)).masked_fill(~mask[:, None], -math.inf)
    assert torch.allclose(lse, sc.logsumexp(-1)) and torch.allclose(o, sc.softmax(-1) @ v)
