"""GPU: the page operations of a kv cache against plain Python, exactly: whole
numbers and copied bytes."""
import random

import pytest
import torch

import ops_b200
from oracle import cache_oracle as C
from oracle import tree_oracle as T

pytestmark = pytest.mark.gpu


class Both:
    """The same cache on the GPU and in plain Python."""

    def __init__(self, n, width, pages, shapes, seed):
        g = torch.Generator().manual_seed(seed)
        self.page = shapes[0][0][0]
        self.pools = [torch.randint(-100, 100, (pages, *shape), generator=g).to(dtype) for shape, dtype in shapes]
        self.refs, self.table, self.lens = [0] * pages, [[-1] * width for _ in range(n)], [0] * n
        self.up()

    def up(self):
        i32 = dict(dtype=torch.int32, device="cuda")
        self.g_refs, self.g_lens = torch.tensor(self.refs, **i32), torch.tensor(self.lens, **i32)
        self.g_table = torch.tensor(self.table, **i32).view(len(self.table), -1)
        self.g_pools = [p.cuda() for p in self.pools]

    def same(self, what=""):
        assert self.g_refs.tolist() == self.refs, what
        assert self.g_lens.tolist() == self.lens, what
        assert self.g_table.tolist() == self.table, what
        for a, b in zip(self.g_pools, self.pools):
            assert torch.equal(a.cpu(), b), what

    def reserve(self, add):
        got = ops_b200.paged_cache_reserve(self.g_refs, self.g_table, self.g_lens, ints(add), self.page)
        assert got.tolist() == C.reserve(self.refs, self.table, self.lens, add, self.page)

    def trim(self, keep):
        ops_b200.paged_cache_trim(self.g_refs, self.g_table, self.g_lens, ints(keep), self.page)
        C.trim(self.refs, self.table, self.lens, keep, self.page)

    def fork(self, src, dst):
        got = ops_b200.paged_cache_fork(self.g_refs, self.g_table, self.g_lens, ints(src), ints(dst), self.g_pools)
        assert got.tolist() == C.fork(self.refs, self.table, self.lens, src, dst, self.pools)

    def accept(self, acc, drafted):
        got = ops_b200.paged_cache_accept(self.g_pools, self.g_table, self.g_lens, ints(acc).view(len(drafted), -1), ints(drafted))
        keep = C.accept(self.pools, self.table, self.lens, acc, drafted)
        assert got.tolist() == keep
        return keep

    def compact(self):
        got = ops_b200.paged_cache_compact(self.g_refs, self.g_table, self.g_pools)
        assert got.tolist() == [C.compact(self.refs, self.table, self.pools)]

    def copy(self, src, dst):
        got = ops_b200.paged_cache_copy(self.g_pools, ints(src), ints(dst))
        assert got.tolist() == C.copy(self.pools, src, dst)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


SHAPES = [
    [((16, 2, 64), torch.bfloat16), ((16, 2, 64), torch.bfloat16)],          # pages of 16-byte units
    [((7, 3, 5), torch.uint8), ((7, 2), torch.float32), ((7, 1, 6), torch.float16)],   # bytes, words, odd sizes
    [((64, 8, 128), torch.bfloat16)],                                        # pages of several steps
]


@pytest.mark.parametrize("shapes", SHAPES, ids=["vectors", "bytes", "large"])
@pytest.mark.parametrize("n,width,pages,seed", [(9, 6, 23, 1), (40, 4, 200, 2), (3, 12, 9, 3)])
def test_random_histories(shapes, n, width, pages, seed):
    r, c = random.Random(seed), Both(n, width, pages, shapes, seed)
    for step in range(24):
        op = r.choice(["reserve", "reserve", "trim", "fork", "accept", "compact", "copy"])
        if op == "reserve":
            c.reserve([r.choice([0, 1, r.randint(0, 3 * c.page), -1]) for _ in range(n)])
        elif op == "trim":
            c.trim([r.choice([-1, 0, r.randint(0, width * c.page)]) if r.random() < 0.5 else -1 for _ in range(n)])
        elif op == "fork":
            f = r.randint(0, n)
            c.fork([r.randint(-1, n) for _ in range(f)], [r.randint(-1, n) for _ in range(f)])
        elif op == "accept":
            drafted = [r.randint(0, min(length, 9)) if r.random() < 0.9 else length + 1 for length in c.lens]
            drafted = [0 if any(c.refs[p] > 1 for p in c.table[s] if p >= 0) else d for s, d in enumerate(drafted)]
            acc = [sorted(r.sample(range(d), r.randint(0, d)))[:8] if 0 < d <= length else [] for d, length in zip(drafted, c.lens)]
            c.trim(c.accept([a + [-1] * (8 - len(a)) for a in acc], drafted))
        elif op == "compact":
            c.compact()
        else:
            m = r.randint(0, 6)
            free = [i for i in range(pages) if c.refs[i] == 0] + [-1, pages]
            c.copy([r.randint(-1, pages) for _ in range(m)], [r.choice(free) for _ in range(m)])
        c.same(f"step {step}: {op}")


def test_reserve_refuses_what_does_not_fit():
    c = Both(6, 4, 6, SHAPES[0], 4)
    c.reserve([20, 16, 0, 65, 1, 40])          # 2 + 1 pages; a table of 64 rows; then 1 page; 3 more than are left
    c.same()
    assert c.lens == [20, 16, 0, 0, 1, 0]
    c.reserve([0, 2 ** 31 - 1, -5, 0, 2 ** 30, 16])
    c.same()
    c.fork([1, 0], [2, 3])                     # row 1's page is shared whole; row 0's last page is copied
    c.same()
    c.trim([-1, 10, -1, -1, -1, -1])           # row 1 now ends inside the page that row 2 shares
    c.same()
    c.reserve([0, 1, 1, 0, 0, 0])              # row 1 must not write there; row 2 is full and out of pages or not
    c.same()
    assert c.lens[1] == 10


def test_many_rows_and_pages():
    n, pages = 3000, 9000                      # more rows and pages than threads
    c = Both(n, 4, pages, [((4, 2), torch.int32)], 5)
    r = random.Random(7)
    c.reserve([r.randint(0, 9) for _ in range(n)])
    c.same()
    c.trim([r.choice([-1, 0, 3]) for _ in range(n)])
    c.same()
    dst = [s for s in range(n) if c.lens[s] == 0][:700]
    src = [r.choice([s for s in range(n) if c.lens[s]][:50]) for _ in dst]
    c.fork(src + src[:9], dst + dst[:9])       # the last nine name targets again
    c.same()
    c.compact()
    c.same()
    c.reserve([16 - length for length in c.lens])   # more than the pool holds: the first rows get theirs
    c.same()


def test_accept_moves_long_paths_and_many_pools():
    n, m = 3, 150                              # more accepted rows than one list, pools than one launch
    shapes = [((32, 8), torch.int16)] * 130
    c = Both(n, 10, 40, shapes, 6)
    c.reserve([m + 5, m + 40, m])
    r = random.Random(1)
    acc = [sorted(r.sample(range(m), k)) for k in (149, 70, 0)]
    acc = [a + [-1] * (m - len(a)) for a in acc]
    acc[1][10] = acc[1][9]                     # not ascending: the path ends there
    keep = c.accept(acc, [m, m, m])
    assert keep == [5 + 149, 40 + 10, 0]
    c.same()
    c.trim(keep)
    c.same()
    c.accept([[] for _ in range(n)], [0, 1, 2])  # no columns at all
    c.fork([0], [2])
    c.compact()
    c.same()


def test_strided_pools_and_state():
    # K and V as two halves of one tensor of pages; the table a slice of a wider one
    both = torch.randint(-9, 9, (12, 2, 8, 4), dtype=torch.int32)
    want = both.clone()
    g = both.cuda()
    pools = [g[:, 0], g[:, 1]]
    copied = ops_b200.paged_cache_copy(pools, ints([3, 3, 5, 9, 2]), ints([4, 6, 4, 9, 3]))
    # 2 -> 3 writes the source of the first two
    assert copied.tolist() == [0, 0, 0, 1, 1]
    want[3] = both[2]
    assert torch.equal(g.cpu(), want)
    wide = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    refs, lens = torch.zeros(12, dtype=torch.int32, device="cuda"), ints([0, 0, 0])
    view = wide[:, 5:9]
    assert ops_b200.paged_cache_reserve(refs, view, lens, ints([9, 1, 40]), 8).tolist() == [1, 1, 0]
    assert view.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1], [-1] * 4] and int((wide >= 0).sum()) == 3


def test_empty_calls():
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    refs, pool = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, 8, 2, device="cuda")
    table = none.view(0, 3)
    assert ops_b200.paged_cache_reserve(refs, table, none, none, 8).numel() == 0
    ops_b200.paged_cache_trim(refs, table, none, none, 8)
    assert ops_b200.paged_cache_fork(refs, table, none, none, none, [pool]).numel() == 0
    assert ops_b200.paged_cache_accept([pool], table, none, none.view(0, 2), none).numel() == 0
    assert ops_b200.paged_cache_compact(refs, table, [pool]).tolist() == [0]
    assert ops_b200.paged_cache_copy([pool], none, none).numel() == 0


def serving_step(state, q, k, v, parents, accepted, cu, m, freq):
    """Room, rows into the pages, attention over them, the accepted path kept."""
    refs, table, lens, kc, vc, page, depth = state
    before = lens.clone()
    granted = ops_b200.paged_cache_reserve(refs, table, lens, torch.full_like(lens, m), page)
    pos = (before[:, None] + depth).view(-1)
    qr = ops_b200.qk_norm_rotary_append(q, k, v, pos, freq, kc, vc, table, lens, cu_seqlens=cu)
    o, lse = ops_b200.tree_attention_paged(qr, kc, vc, table, lens, parents, cu_seqlens=cu, max_seqlen_q=m)
    keep = ops_b200.paged_cache_accept([kc, vc], table, lens, accepted, torch.full_like(lens, m))
    ops_b200.paged_cache_trim(refs, table, lens, keep, page)
    return granted, o, lse


@pytest.mark.parametrize("captured", [False, True])
def test_steps_of_speculative_decoding(captured):
    # three steps of drafted trees; each step's attention against the rows that were accepted, kept apart
    from oracle import rotary_oracle as R
    n, m, hq, hk, d, page = 5, 7, 8, 2, 64, 16
    g = torch.Generator().manual_seed(0)
    freq, _ = ops_b200.rotary_frequencies(d)
    refs, table = torch.zeros(40, dtype=torch.int32, device="cuda"), torch.full((n, 8), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(n, dtype=torch.int32, device="cuda")
    kc, vc = (torch.full((40, page, hk, d), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    par = torch.tensor([-1, 0, 0, 1, 1, 2, 4], dtype=torch.int32)
    depth = torch.tensor([0, 1, 1, 2, 2, 2, 3], dtype=torch.int32)
    paths = [[0, 1, 4, 6], [0, 2], [0, 1, 3], [0], [0, 2, 5]]
    acc = torch.tensor([p + [-1] * (m - len(p)) for p in paths], dtype=torch.int32).cuda()
    cu = (torch.arange(n + 1, dtype=torch.int32) * m).cuda()
    parents = par.repeat(n).cuda()
    state = (refs, table, lens, kc, vc, page, depth.cuda())
    q, k, v = (torch.empty(n * m, h, d, dtype=torch.bfloat16, device="cuda") for h in (hq, hk, hk))
    kept = [([], []) for _ in range(n)]
    args = (state, q, k, v, parents, acc, cu, m, freq.cuda())
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = serving_step(*args)
    for _ in range(3):
        qn, kn, vn = (torch.randn(t.shape, generator=g).bfloat16() for t in (q, k, v))
        q.copy_(qn)
        k.copy_(kn)
        v.copy_(vn)
        before = lens.tolist()
        if captured:
            graph.replay()
        else:
            out = serving_step(*args)
        granted, o, lse = out
        assert granted.tolist() == [1] * n
        assert lens.tolist() == [b + len(p) for b, p in zip(before, paths)]
        pos = (torch.tensor(before)[:, None] + depth).view(-1)
        # bf16 rows as the kernel stores them, up to the roundings of a step: checked to 2^-7 below
        kr, qr = (R.forward(t, None, pos, freq).bfloat16() for t in (kn, qn))
        for s in range(n):
            ks, vs = kept[s]
            pool_k = torch.cat([torch.stack(ks) if ks else kr[:0], kr[s * m:(s + 1) * m]])[None]
            pool_v = torch.cat([torch.stack(vs) if vs else vn[:0], vn[s * m:(s + 1) * m]])[None]
            ro, rl, size, reach = T.tree_attention(qr[s * m:(s + 1) * m], pool_k, pool_v, torch.zeros(1, 1, dtype=torch.int32),
                                                   torch.tensor([pool_k.shape[1]]), par, cu_seqlens=torch.tensor([0, m]))
            # a score moves by at most 2 * 2^-8 of sum |q k| scale where a row was rounded the other way
            e = 4 * 2.0 ** -8 * reach
            rows = slice(s * m, (s + 1) * m)
            assert ((lse[rows].double().cpu() - rl).abs() <= e).all()
            assert ((o[rows].double().cpu() - ro).abs() <= 2.0 ** -8 * ro.abs() + (2.0 ** -7 + 2 * e[..., None]) * size).all()
            for a in paths[s]:
                ks.append(kr[s * m + a])
                vs.append(vn[s * m + a])
    # what is left of the cache: the accepted rows, in order
    for s in range(n):
        rows = [(int(table[s, t // page]), t % page) for t in range(int(lens[s]))]
        got_v = torch.stack([vc[p, r] for p, r in rows]).cpu()
        assert torch.equal(got_v, torch.stack(kept[s][1]))
        got_k = torch.stack([kc[p, r] for p, r in rows]).cpu().double()
        ref_k = torch.stack(kept[s][0]).double()
        assert ((got_k - ref_k).abs() <= 2.0 ** -7 * ref_k.abs()).all()
    assert int((refs > 0).sum()) == sum((int(x) + page - 1) // page for x in lens)


def test_training_step_through_the_op():
    # norm and rotation before the sparse op: the gradient of the whole against the formulas of both
    from oracle import rotary_oracle as R
    from oracle import sfa_oracle as O
    from sfa_check import assert_close
    g = torch.Generator().manual_seed(0)
    b, t, hq, hk, d, bs, sel = 1, 256, 16, 2, 64, 64, 3
    q, k, v = (torch.randn(b, t, h, d, generator=g).bfloat16() for h in (hq, hk, hk))
    wq, wk = 1 + 0.2 * torch.randn(d, generator=g), 1 + 0.2 * torch.randn(d, generator=g)
    do = torch.randn(b, t, hq, d, generator=g).bfloat16()
    idx = torch.stack([torch.randperm(4, generator=g)[:sel] for _ in range(b * t * hk)]).view(b, t, hk, sel).to(torch.int32)
    freq, _ = ops_b200.rotary_frequencies(d)
    pos = torch.arange(t)
    leaves = [x.cuda().requires_grad_() for x in (q, k, v, wq, wk)]
    qr, kr = ops_b200.qk_norm_rotary(leaves[0], leaves[1], pos.cuda(), freq.cuda(), leaves[3], leaves[4])
    o, _ = ops_b200.sparse_flash_attention(qr, kr, leaves[2], idx.cuda(), bs)
    grads = torch.autograd.grad(o, leaves, do.cuda())
    rq, rk = (x.detach().cpu().float() for x in (qr, kr))
    ro, rl = O.sfa_forward(rq, rk, v.float(), idx, bs)
    assert_close("o", o, ro)
    dqr, dkr, dv, _ = O.sfa_backward(rq, rk, v.float(), idx, o.detach().cpu().float(), rl, do.float(), bs)
    dq, dwq, _, _ = R.backward(q, wq, dqr, pos.expand(b, t), freq)
    dk, dwk, _, _ = R.backward(k, wk, dkr, pos.expand(b, t), freq)
    for name, got, ref in zip(("dq", "dk", "dv", "dwq", "dwk"), grads, (dq, dk, dv, dwq, dwk)):
        assert_close(name, got, ref)           # the op's own tolerance: its gradients are inputs of the norm's
