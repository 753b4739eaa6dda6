"""Norm and rotary positions, what needs no GPU: the frequencies, the refusals
of the Python surface and of the C ABI, the struct layouts, and the oracle's
gradient against autograd of its forward."""
import ctypes
import math
import os
import subprocess
import tempfile

import pytest
import torch

import ops_b200
from ops_b200 import _lib
from oracle import rotary_oracle as R

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "sfa_b200.h")


@pytest.mark.parametrize("struct", ["SfaRotaryTensor", "SfaRotaryParams"])
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


def test_frequencies():
    f, a = ops_b200.rotary_frequencies(8, base=10000.0)
    assert a == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    assert torch.equal(ops_b200.rotary_frequencies(8, scaling="linear", factor=4.0)[0], f / 4)
    n, _ = ops_b200.rotary_frequencies(8, scaling="ntk", factor=4.0)
    assert float(n[0]) == 1.0 and math.isclose(float(n[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    y, a = ops_b200.rotary_frequencies(64, scaling="yarn", factor=8.0, original_length=4096)
    p, _ = ops_b200.rotary_frequencies(64)
    turns = 4096 * p / (2 * math.pi)
    assert math.isclose(a, 0.1 * math.log(8) + 1)
    assert torch.equal(y[turns >= 32], p[turns >= 32]) and torch.allclose(y[turns <= 1], p[turns <= 1] / 8, rtol=1e-15)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (y[mid] < p[mid]).all() and (y[mid] > p[mid] / 8).all()
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, factor=-1.0),
                dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, scaling="yarn", beta_fast=1.0)):
        with pytest.raises(ValueError):
            ops_b200.rotary_frequencies(**bad)


def test_oracle_gradient_is_the_derivative():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 3, 20, generator=g, dtype=torch.float64, requires_grad=True)
    w = torch.randn(20, generator=g, dtype=torch.float64, requires_grad=True)
    dy, pos = torch.randn(5, 3, 20, generator=g, dtype=torch.float64), torch.arange(5) * 1000
    f, _ = ops_b200.rotary_frequencies(12)
    kw = dict(eps=1e-3, start=6, interleaved=True, amplitude=1.3)
    dx, dw, _, _ = R.backward(x.detach(), w.detach(), dy, pos, f, **kw)
    ax, aw = torch.autograd.grad(R.forward(x, w, pos, f, **kw), [x, w], dy)
    assert torch.allclose(dx, ax, rtol=1e-12, atol=1e-13) and torch.allclose(dw, aw, rtol=1e-12, atol=1e-13)


def good():
    q, k = torch.zeros(2, 6, 4, 64), torch.zeros(2, 6, 2, 64)
    return dict(q=q, k=k, positions=torch.arange(6), frequencies=ops_b200.rotary_frequencies(32)[0],
                q_weight=torch.ones(64), k_weight=torch.ones(64))


@pytest.mark.parametrize("bad,msg", [
    (dict(), "CUDA"), (dict(q=torch.zeros(2, 6, 4, 64, dtype=torch.float64)), "bfloat16"),
    (dict(q=torch.zeros(6, 64)), "must be"), (dict(q=torch.zeros(2, 6, 0, 64)), "at least one"),
    (dict(k=torch.zeros(2, 6, 2, 64, dtype=torch.bfloat16)), "q's type"), (dict(k=torch.zeros(2, 5, 2, 64)), "tokens"),
    (dict(k=torch.zeros(2, 6, 2, 32)), "head size"), (dict(positions=None), "go together"),
    (dict(positions=torch.arange(5)), "broadcast"), (dict(positions=torch.zeros(6)), "int32"),
    (dict(frequencies=torch.zeros(16)), "float64"), (dict(start=33), "within the head"), (dict(start=-1), "within the head"),
    (dict(q_weight=torch.ones(32)), "q_weight"), (dict(k_weight=torch.ones(64, dtype=torch.int64)), "k_weight"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(frequencies=torch.zeros(16, dtype=torch.float64, requires_grad=True)), "no gradient"),
])
def test_refusals(bad, msg):
    with pytest.raises(ValueError, match=msg):
        ops_b200.qk_norm_rotary(**{**good(), **bad})


ONE_POOL = torch.zeros(5, 8, 2, 64)


def append_args():
    f = torch.float32
    return dict(q=torch.zeros(3, 4, 64), k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), positions=torch.arange(3),
                frequencies=ops_b200.rotary_frequencies(64)[0], k_cache=torch.zeros(5, 8, 2, 64, dtype=f),
                v_cache=torch.zeros(5, 8, 2, 64, dtype=f), block_table=torch.zeros(3, 2, dtype=torch.int32),
                cache_seqlens=torch.ones(3, dtype=torch.int32))


@pytest.mark.parametrize("bad,msg", [
    (dict(), "CUDA"), (dict(v=torch.zeros(2, 2, 64)), "v must be"), (dict(v=torch.zeros(3, 1, 64)), "k's heads"),
    (dict(k_cache=torch.zeros(5, 8, 2, 64).half()), "k_cache"), (dict(v_cache=torch.zeros(5, 8, 2, 32)), "v_cache"),
    (dict(v_cache=torch.zeros(4, 8, 2, 64)), "same pages"), (dict(k_cache=ONE_POOL, v_cache=ONE_POOL), "same memory"),
    (dict(v_cache=torch.zeros(5, 8, 1, 64).expand(5, 8, 2, 64)), "overlap"),
    (dict(k_cache=torch.zeros(1, 1, 2, 64).expand(5, 8, 2, 64)), "overlap"),
    (dict(k_cache=torch.zeros(5, 2, 8, 64).transpose(1, 2)), "row ranges"),
    (dict(block_table=torch.zeros(3, 2)), "int32"), (dict(cache_seqlens=torch.ones(2, dtype=torch.int32)), "same number"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int32), cache_seqlens=torch.ones(2, dtype=torch.int32)), "one row"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), "cu_seqlens"),
])
def test_append_refusals(bad, msg):
    with pytest.raises(ValueError, match=msg):
        ops_b200.qk_norm_rotary_append(**{**append_args(), **bad})


def test_c_abi_refusals():
    lib = _lib.load()
    fake = 0x10000

    def params(**kw):
        P = _lib.SfaRotaryParams(num_tensors=1, batch=1, len=4, dim=64, rot=64, positions=fake, frequencies=fake)
        P.t[0].x = P.t[0].y = P.t[0].dy = P.t[0].dx = fake
        P.t[0].heads, P.t[0].flags = 2, _lib.SFA_ROTARY_TURN
        for n, v in kw.items():
            setattr(P.t[0] if n in ("x", "y", "dx", "heads", "flags", "dweight") else P, n, v)
        return P

    for bad, msg in ((dict(num_tensors=4), "num_tensors"), (dict(dim=1025), "dim"), (dict(rot=7), "rot"),
                     (dict(start=8), "rot"), (dict(dtype=3), "dtype"), (dict(heads=0), "heads"), (dict(x=None), "non-NULL"),
                     (dict(y=None), "non-NULL"), (dict(positions=None), "positions"), (dict(len=-1), "len")):
        P = params(**bad)
        assert lib.sfa_rotary_fwd(ctypes.byref(P), None) == _lib.SFA_ERR_INVALID_ARGUMENT, bad
        assert msg in lib.sfa_last_error_string().decode()
    paged = dict(flags=_lib.SFA_ROTARY_TURN | _lib.SFA_ROTARY_PAGED, page_size=16, num_pages=4, table_width=1, num_seqs=1,
                 block_table=fake, cache_seqlens=fake)
    for bad, msg in ((dict(batch=2), "batch 1"), (dict(page_size=0), "page_size"), (dict(block_table=None), "block_table")):
        P = params(**{**paged, **bad})
        assert lib.sfa_rotary_fwd(ctypes.byref(P), None) == _lib.SFA_ERR_INVALID_ARGUMENT
        assert msg in lib.sfa_last_error_string().decode()
    P = params(**paged)
    assert lib.sfa_rotary_bwd(ctypes.byref(P), None, 0, None) == _lib.SFA_ERR_UNSUPPORTED
    P = params(dweight=fake)
    assert lib.sfa_rotary_bwd(ctypes.byref(P), None, 0, None) == _lib.SFA_ERR_INVALID_ARGUMENT   # no weight
    assert lib.sfa_rotary_bwd_workspace_bytes(ctypes.byref(P)) == 0
    P.t[0].weight = fake
    assert lib.sfa_rotary_bwd_workspace_bytes(ctypes.byref(P)) > 0
    assert lib.sfa_rotary_bwd(ctypes.byref(P), None, 0, None) == _lib.SFA_ERR_WORKSPACE
