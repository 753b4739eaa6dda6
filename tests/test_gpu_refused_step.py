"""GPU: a step of speculative decoding in which a sequence gets no room.  Its
rows, its length and its pages stay as they were, its queries see nothing, and
the other sequences' results are those of a step without it."""
import pytest
import torch

import ops_b200

pytestmark = pytest.mark.gpu

N, M, HQ, HK, D, PAGE = 4, 6, 8, 2, 64, 16


def state(pages):
    """Four sequences of 20, 31, 16 and 9 rows; the pool has `pages` pages."""
    i32 = dict(dtype=torch.int32, device="cuda")
    refs, table, lens = torch.zeros(pages, **i32), torch.full((N, 4), -1, **i32), torch.zeros(N, **i32)
    assert ops_b200.paged_cache_reserve(refs, table, lens, torch.tensor([20, 31, 16, 9], **i32), PAGE).tolist() == [1] * N
    g = torch.Generator().manual_seed(1)
    kc, vc = (torch.randn(30, PAGE, HK, D, generator=g).bfloat16()[:pages].cuda() for _ in range(2))
    return refs, table, lens, kc, vc


def inputs():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(N * M, h, D, generator=g).bfloat16().cuda() for h in (HQ, HK, HK))
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(q=q, k=k, v=v, cu=torch.arange(N + 1, **i32) * M, drafted=torch.full((N,), M, **i32),
                parents=torch.tensor([-1, 0, 0, 1, 2, 4], **i32).repeat(N),
                accepted=torch.tensor([[0, 2, 4, 5, -1, -1]] * N, **i32), pos=torch.arange(N * M, **i32),
                freq=ops_b200.rotary_frequencies(D, device="cuda")[0])


def step(st, x):
    refs, table, lens, kc, vc = st
    granted = ops_b200.paged_cache_reserve(refs, table, lens, x["drafted"], PAGE)
    now, drafted = lens * granted, x["drafted"] * granted     # a refused sequence has no rows in this step
    q = ops_b200.qk_norm_rotary_append(x["q"], x["k"], x["v"], x["pos"], x["freq"], kc, vc, table, now, cu_seqlens=x["cu"])
    o, lse = ops_b200.tree_attention_paged(q, kc, vc, table, now, x["parents"], cu_seqlens=x["cu"], max_seqlen_q=M)
    keep = ops_b200.paged_cache_accept([kc, vc], table, lens, x["accepted"], drafted, refcounts=refs)
    ops_b200.paged_cache_trim(refs, table, lens, keep, PAGE)
    return granted, o, lse


def rows(st, s):
    _, table, lens, kc, vc = st
    at = [(int(table[s, t // PAGE]), t % PAGE) for t in range(int(lens[s]))]
    return [torch.stack([c[p, r] for p, r in at]) for c in (kc, vc)]


@pytest.mark.parametrize("captured", [False, True])
def test_a_refused_sequence_is_left_as_it_is(captured):
    # 6 pages are held; sequences 1 (rows 31 .. 36) and 2 (16 .. 21) need one more each, and there is one
    x, free, short = inputs(), state(30), state(6 + 1)
    before = [rows(short, s) for s in range(N)]
    want = step(free, x)
    assert want[0].tolist() == [1] * N
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(short, x)
        graph.replay()
        torch.cuda.synchronize()
    else:
        got = step(short, x)
    assert got[0].tolist() == [1, 1, 0, 1]
    assert short[2].tolist() == [24, 35, 16, 13] and free[2].tolist() == [24, 35, 20, 13]
    for s in range(N):
        mine = slice(s * M, (s + 1) * M)
        if s == 2:
            assert not got[1][mine].any() and torch.isinf(got[2][mine]).all()
            for a, b in zip(rows(short, s), before[s]):
                assert torch.equal(a, b)
        else:
            assert torch.equal(got[1][mine], want[1][mine]) and torch.equal(got[2][mine], want[2][mine])
            for a, b in zip(rows(short, s), rows(free, s)):
                assert torch.equal(a, b)
    assert int((short[0] > 0).sum()) == 2 + 3 + 1 + 1
