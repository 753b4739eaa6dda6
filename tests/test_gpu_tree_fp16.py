"""GPU: fp16 probabilities of tree attention under one dominant key.

Tolerance.  u = 2^-11 is half a step of fp16.  The result is rounded once
(u |o|) and so is every probability that is a normal number (u sum p |v|).  The
scores are exact.  exp2 and the row sum stay below 2^-16 of the terms, and the
product sum takes a step of 2^-23 at most for every 16 keys.  A probability is held against a
reference 2^8 below the largest one, so what is below fp16's normal numbers
loses at most 2^-25 2^-8 of the largest probability, twice where the reference
was raised inside a chunk; the row sum is at least the largest."""
import pytest
import torch

import ops_b200

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dv", [64, 192])
@pytest.mark.parametrize("gap", [13, 15, 17, 19])
@pytest.mark.parametrize("at", ["first", "last", "raised"])
def test_one_dominant_key_over_a_long_cache(dv, gap, at):
    # the first dim of k is the score, and q's first dim is 1.  max_seqlen_k 1 leaves the whole cache to one
    # CTA, so that the dominant key and the others meet one reference
    keys, page, hq, d = 16384, 64, 4, 64
    top = {"first": {0: gap}, "last": {keys - 1: gap}, "raised": {40: gap - 8, 100: gap}}[at]
    kc = torch.zeros(keys // page, page, 1, d, dtype=torch.float16)
    vc = torch.ones(keys // page, page, 1, dv, dtype=torch.float16)
    vc[..., 1::2] = 0.25
    flat_k, flat_v = kc.view(keys, d), vc.view(keys, dv)
    flat_k[::2, 0] = -1.0                       # every other key e times less
    for t, score in top.items():
        flat_k[t, 0], flat_v[t] = score, 0.0
    q = torch.zeros(1, hq, d, dtype=torch.float16)
    q[..., 0] = 1.0
    q[:, 1:, 0] = 0.5                           # and heads with half the gap
    o, lse = ops_b200.tree_attention_paged(q.cuda(), kc.cuda(), vc.cuda(),
                                           torch.arange(keys // page, dtype=torch.int32, device="cuda")[None],
                                           torch.tensor([keys], dtype=torch.int32, device="cuda"), scale=1.0, max_seqlen_k=1)
    s = q[0, :, :1].double() * flat_k[:, 0].double()[None]
    ref_l = torch.logsumexp(s, 1)
    ref = torch.exp(s - ref_l[:, None]) @ flat_v.double()
    u, e = 2.0 ** -11, 2.0 ** -16 + keys / 16 * 2.0 ** -23
    tol = u * ref + (u + e) * ref * (1 + u) + 2 * keys * 2.0 ** -33 * float(flat_v.max()) + 2.0 ** -25
    off = ((o[0].double().cpu() - ref).abs() / tol).max()
    assert float(off) <= 1.0, f"{float(off):.3f} of the tolerance"
    # a chain of one addition for 64 keys
    assert ((lse[0].double().cpu() - ref_l).abs() <= 2.0 ** -16 + keys / 64 * 2.0 ** -24 + 2.0 ** -20 * ref_l.abs()).all()
