"""GPU: attention of drafted rows over a paged cache against the 64-bit
definition, at the sizes and masks where it can go wrong.

Tolerances.  With u half a step of the type (eps / 2): the result is rounded
once (u |o|) and so is every probability (u sum p |v|).  The scores are summed
in fp32 over D products, so a probability carries a relative error of twice
D 2^-24 times the largest sum |q k| scale of its row, and exp2, the row sum and
the product sum together stay below 2^-16.  fp16 probabilities below 2^-14 of
the reference maximum lose at most 2^-25 each.  lse is a sum of the same errors
without the roundings to the type."""
import math

import pytest
import torch

import ops_b200
from oracle import tree_oracle as O

pytestmark = pytest.mark.gpu


def check(got, ref, q, v_cache, keys):
    o, lse = got
    ro, rl, size, reach = ref
    u = torch.finfo(o.dtype).eps / 2
    e = 2 * q.shape[-1] * 2.0 ** -24 * reach + 2.0 ** -16
    go, gl = o.double().cpu(), lse.double().cpu()
    fin = torch.isfinite(rl)
    assert torch.equal(gl[~fin], rl[~fin]), "lse of rows that see nothing"
    assert torch.equal(torch.isnan(go), torch.isnan(ro))
    inf = torch.isinf(ro)
    assert torch.equal(go[inf], ro[inf])
    off_l = ((gl - rl).abs() / (e + 2.0 ** -20 * rl.abs()))[fin]
    assert off_l.numel() == 0 or float(off_l.max()) <= 1.0, f"lse {float(off_l.max()):.3f} of the tolerance"
    ok = torch.isfinite(ro)
    tol = u * ro.abs() + (u + e[..., None]) * size * (1 + u) + 2.0 ** -126
    if o.dtype == torch.float16:
        vmax = v_cache.double().nan_to_num(0, 0, 0).abs().max()
        tol = tol + keys * 2.0 ** -25 * vmax + 2.0 ** -25
    off = ((go - ro).abs() / tol)[ok]
    assert off.numel() == 0 or float(off.max()) <= 1.0, f"o {float(off.max()):.3f} of the tolerance"


def problem(counts, prefixes, hq, hk, dqk, dv, page, dtype, seed, shape="tree", behind=0, fill=float("nan")):
    """Inputs on the CPU; cache rows that no sequence holds are `fill`."""
    g = torch.Generator().manual_seed(seed)
    n = len(counts)
    lens = torch.tensor([c + p for c, p in zip(counts, prefixes)], dtype=torch.int32)
    width = max(1, (int(lens.max()) + page - 1) // page) + 1
    pages = sum((int(l) + page - 1) // page for l in lens) + 3
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((n, width), -1, dtype=torch.int32)
    kc = torch.full((pages, page, hk, dqk), fill, dtype=dtype)
    vc = torch.full((pages, page, hk, dv), fill, dtype=dtype)
    at = 0
    for s in range(n):
        for i in range((int(lens[s]) + page - 1) // page):
            pg = int(perm[at])
            at += 1
            table[s, i] = pg
            r = min(page, int(lens[s]) - i * page)
            kc[pg, :r] = torch.randn(r, hk, dqk, generator=g).to(dtype)
            vc[pg, :r] = torch.randn(r, hk, dv, generator=g).to(dtype)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), torch.tensor(counts).cumsum(0)]).to(torch.int32)
    q = torch.randn(int(cu[-1]) + behind, hq, dqk, generator=g).to(dtype)
    par = None
    if shape == "tree":
        par = torch.full((q.shape[0],), -1, dtype=torch.int32)
        for s in range(n):
            for j in range(1, counts[s]):
                par[int(cu[s]) + j] = int(torch.randint(-1, j, (1,), generator=g))
    return q, kc, vc, table, lens, par, cu


def run(q, kc, vc, table, lens, par, cu, **kw):
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    return ops_b200.tree_attention_paged(q.cuda(), dev(kc), dev(vc), dev(table), dev(lens), dev(par), cu_seqlens=dev(cu), **kw)


CASES = [
    # counts, prefixes, hq, hk, dqk, dv, page, dtype, shape
    ([1], [0], 8, 1, 64, 64, 16, torch.bfloat16, "chain"),                       # one key, its own
    ([1, 1, 1], [63, 64, 65], 16, 2, 128, 128, 64, torch.bfloat16, "chain"),     # around a chunk's end
    ([1] * 9, [0, 1, 127, 200, 333, 64, 5, 1000, 12], 64, 8, 128, 128, 64, torch.bfloat16, "chain"),
    ([7, 1, 16, 3], [100, 0, 513, 60], 12, 4, 96, 80, 24, torch.float16, "tree"),
    ([5, 0, 2, 0], [40, 17, 0, 0], 6, 2, 72, 8, 7, torch.bfloat16, "tree"),      # pages of seven rows, empty sequences
    ([64], [1000], 64, 8, 128, 128, 64, torch.bfloat16, "tree"),                 # several row tiles
    ([33, 90], [70, 3], 5, 5, 64, 64, 16, torch.bfloat16, "chain"),              # one head a kv head, long chains
    ([256], [130], 4, 1, 64, 128, 32, torch.float16, "tree"),                    # the largest tree
    ([300, 2], [20, 700], 8, 2, 64, 64, 128, torch.bfloat16, "chain"),           # a chunk of a prompt
    ([3, 2], [150, 90], 160, 1, 128, 64, 48, torch.bfloat16, "tree"),            # more heads than a tile
    ([2, 4], [200, 64], 256, 2, 64, 64, 1, torch.bfloat16, "tree"),              # pages of one row
    ([9], [777], 8, 2, 256, 256, 64, torch.bfloat16, "tree"),                    # wide heads: one CTA per SM
    ([4, 11], [300, 20], 16, 4, 192, 136, 40, torch.float16, "tree"),
    ([2], [120], 3, 3, 8, 16, 8, torch.bfloat16, "tree"),
    ([1], [9000], 8, 1, 128, 128, 64, torch.bfloat16, "chain"),                  # one unit over many ranges
    ([6, 3], [6000, 2500], 16, 2, 64, 64, 256, torch.float16, "tree"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c[0][:4]}-{c[1][:4]}-h{c[2]}/{c[3]}-d{c[4]}/{c[5]}-p{c[6]}-{c[8]}")
@pytest.mark.parametrize("sink", [False, True])
def test_matches_the_definition(case, sink):
    counts, prefixes, hq, hk, dqk, dv, page, dtype, shape = case
    args = problem(counts, prefixes, hq, hk, dqk, dv, page, dtype, seed=len(counts) + page, shape=shape)
    s = torch.randn(hq, generator=torch.Generator().manual_seed(7)) if sink else None
    got = run(*args, attn_sink=None if s is None else s.cuda())
    q, kc, vc, table, lens, par, cu = args
    ref = O.tree_attention(q, kc, vc, table, lens, par, cu_seqlens=cu, attn_sink=s)
    check(got, ref, q, vc, int(lens.max()))


def test_defaults_scale_and_strides():
    # one row per sequence without cu_seqlens; k and v two halves of one pool; q a slice of a wider projection
    n, hq, hk, d, page = 5, 8, 2, 64, 32
    q, kc, vc, table, lens, _, _ = problem([1] * n, [10, 100, 64, 31, 200], hq, hk, d, d, page, torch.bfloat16, 3)
    both = torch.stack([kc, vc], 3).cuda()                          # [pages, page, hk, 2, d]
    wide = torch.zeros(n, hq + 4, d + 8, dtype=torch.bfloat16)
    wide[:, 2:-2, 4:-4] = q                                         # an unaligned slice: taken through a copy
    ref = O.tree_attention(q, kc, vc, table, lens, scale=0.3)
    got = ops_b200.tree_attention_paged(wide.cuda()[:, 2:-2, 4:-4], both[:, :, :, 0], both[:, :, :, 1], table.cuda(), lens.cuda(), scale=0.3)
    check(got, ref, q, vc, 201)
    aligned = torch.zeros(n, hq + 4, d + 8, dtype=torch.bfloat16)
    aligned[:, 2:-2, 8:] = q
    got = ops_b200.tree_attention_paged(aligned.cuda()[:, 2:-2, 8:], both[:, :, :, 0], both[:, :, :, 1], table.cuda(), lens.cuda(), scale=0.3,
                                        max_seqlen_k=1)             # a poor estimate changes only the split
    check(got, ref, q, vc, 201)
    wide_table = torch.full((n, 2 * table.shape[1]), 0, dtype=torch.int32)
    wide_table[:, ::2] = table
    got = ops_b200.tree_attention_paged(q.cuda(), both[:, :, :, 0], both[:, :, :, 1], wide_table.cuda()[:, ::2], lens.cuda(), scale=0.3)
    check(got, ref, q, vc, 201)


KINDS = pytest.mark.parametrize("hq,dqk,dv", [(8, 64, 72), (64, 64, 72), (8, 128, 200), (64, 256, 136)],
                                ids=["one tile", "several tiles", "wide", "wide, several tiles"])


@KINDS
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("where", ["first chunk", "later chunk"])
def test_what_a_row_does_not_see_does_not_matter(dtype, where, hq, dqk, dv):
    # a drafted row's NaN and infinite keys and values reach its descendants and nobody else
    prefix = 3 if where == "first chunk" else 150
    q, kc, vc, table, lens, par, cu = problem([9, 4], [prefix, 40], hq, 2, dqk, dv, 16, dtype, 5)
    par[:9] = torch.tensor([-1, 0, 0, 1, 1, 2, 4, 5, -1])

    def place(j):
        t = prefix + j
        return int(table[0, t // 16]), t % 16

    kc[place(3)] = float("nan")                 # node 3 has no descendants
    vc[place(3)] = float("inf")
    vc[(*place(2), 0, 5)] = float("inf")        # node 2: itself, 5 and 7
    vc[(*place(5), 1, 6)] = -float("inf")       # node 5: itself and 7
    vc[(*place(7), 0, 5)] = -float("inf")       # meets node 2's +inf: NaN
    vc[(*place(8), 1, 0)] = float("nan")
    got = run(q, kc, vc, table, lens, par, cu)
    ref = O.tree_attention(q, kc, vc, table, lens, par, cu_seqlens=cu)
    nan_row = 3
    assert torch.isnan(got[0][nan_row]).all() and torch.isnan(got[1][nan_row]).all()
    keep = [i for i in range(13) if i != nan_row]
    check((got[0][keep], got[1][keep]), [r[keep] for r in ref], q, vc, int(lens.max()))
    assert torch.isfinite(got[0].cpu()[[0, 1, 4, 6, 9, 10, 11, 12]]).all()


@pytest.mark.parametrize("dv", [64, 176])
def test_missing_pages_short_caches_and_rows_behind(dv):
    # entries outside the pool, a table shorter than the cache, a cache shorter than its drafted rows, no cache,
    # rows behind the last sequence
    q, kc, vc, table, lens, par, cu = problem([3, 2, 4, 2, 1], [90, 70, 0, 30, 50], 8, 2, 64, dv, 16, torch.bfloat16, 9, behind=5)
    table[0, 1], table[0, 4], table[1, 2] = -7, kc.shape[0], 2 ** 31 - 1
    table[4, :] = -1                                       # every page of a sequence missing
    lens[2], lens[3] = 2, 0                                # four rows in a cache of two; no cache at all
    short = table[:, :4]                                   # positions from 64 on are behind the table
    for t, sink in ((table, None), (short, None), (table, torch.randn(8, generator=torch.Generator().manual_seed(1)))):
        got = run(q, kc, vc, t.contiguous(), lens, par, cu, attn_sink=None if sink is None else sink.cuda())
        ref = O.tree_attention(q, kc, vc, t, lens, par, cu_seqlens=cu, attn_sink=sink)
        check(got, ref, q, vc, 120)
        assert not got[0][-5:].any() and torch.equal(got[1][-5:].cpu(), ref[1][-5:].float())
    # a pool and a table of nothing
    none = ops_b200.tree_attention_paged(q.cuda()[:2], kc.cuda()[:0], vc.cuda()[:0], table.cuda()[:2, :0], lens.cuda()[:2])
    assert not none[0].any() and torch.isinf(none[1]).all()
    empty = ops_b200.tree_attention_paged(q.cuda()[:0], kc.cuda(), vc.cuda(), table.cuda()[:0], lens.cuda()[:0])
    assert empty[0].shape == (0, 8, dv)


def test_rows_before_the_first_sequence_and_bad_offsets():
    q, kc, vc, table, lens, par, cu = problem([3, 70, 2], [90, 130, 40], 8, 2, 64, 64, 16, torch.bfloat16, 21, behind=4)
    want = run(q, kc, vc, table, lens, par, cu)
    front = 3
    q2, par2 = torch.cat([q[:front], q]), torch.cat([par[:front], par])
    got = run(q2, kc, vc, table, lens, par2, cu + front, max_seqlen_q=70, max_seqlen_k=2 ** 40)
    assert not got[0][:front].any() and torch.isinf(got[1][:front]).all()
    assert torch.equal(got[0][front:], want[0]) and torch.equal(got[1][front:], want[1])
    # offsets in front of the tensor name no rows; the other sequences are untouched by them
    odd = cu.clone()
    odd[0] = -5
    got = run(q, kc, vc, table, lens, par, odd, max_seqlen_q=70)
    assert torch.equal(got[0][3:], want[0][3:]) and torch.equal(got[1][3:], want[1][3:])


def test_pools_past_32_bit_offsets():
    # the pages of a small case at the end of pools of more than 2^31 elements
    q, kc, vc, table, lens, par, cu = problem([5, 1, 12], [300, 77, 40], 16, 8, 128, 128, 64, torch.bfloat16, 17, fill=0.0)
    want = run(q, kc, vc, table, lens, par, cu)
    pages = 2 ** 31 // (64 * 8 * 128) + 2 + kc.shape[0]
    big = []
    for c in (kc, vc):
        big.append(torch.zeros(pages, 64, 8, 128, dtype=torch.bfloat16, device="cuda"))
        big[-1][-kc.shape[0]:] = c.cuda()
        assert big[-1].numel() > 2 ** 31
    far = torch.where(table >= 0, table + pages - kc.shape[0], table)
    got = run(q, big[0], big[1], far, lens, par, cu)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a non-finite element of a drafted value row, which is read from the pool again
    last = int(lens[0]) - 1
    for v, t in ((vc, table), (big[1], far)):
        v[int(t[0, last // 64]), last % 64] = float("inf")
    want = run(q, kc, vc, table, lens, par, cu)
    got = run(q, big[0], big[1], far, lens, par, cu)
    assert torch.isinf(want[0]).any()
    assert torch.equal(got[0].nan_to_num(nan=7.0), want[0].nan_to_num(nan=7.0)) and torch.equal(got[1], want[1])


@KINDS
def test_extreme_scores(hq, dqk, dv):
    # scores that rise by far more than a rescale allows from chunk to chunk, and fall; one key that takes all
    q, kc, vc, table, lens, par, cu = problem([14, 1], [700, 300], hq, 2, dqk, dv, 64, torch.bfloat16, 4, fill=0.0)
    for t in range(int(lens[0])):
        kc[int(table[0, t // 64]), t % 64] *= (t // 64 + 1) * 2.0
    for t in range(int(lens[1])):
        kc[int(table[1, t // 64]), t % 64] *= 12.0 / (t // 64 + 1)
    check(run(q, kc, vc, table, lens, par, cu), O.tree_attention(q, kc, vc, table, lens, par, cu_seqlens=cu), q, vc, 714)


@pytest.mark.parametrize("dv", [128, 192])
def test_streams_graphs_and_repeats(dv):
    a = problem([16, 3, 1], [900, 10, 64], 16, 2, 128, dv, 64, torch.bfloat16, 2)
    b = problem([2] * 6, [50] * 6, 16, 2, 128, dv, 64, torch.bfloat16, 6)
    dev = [[None if t is None else t.cuda() for t in x] for x in (a, b)]

    def call(x):
        return ops_b200.tree_attention_paged(*x[:6], cu_seqlens=x[6], max_seqlen_q=16)

    ref = [call(x) for x in dev]
    for r, x in zip(ref, dev):                               # bit for bit, again
        again = call(x)
        assert torch.equal(r[0], again[0]) and torch.equal(r[1], again[1])
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):                            # both at once
        other = call(dev[1])
    here = call(dev[0])
    torch.cuda.synchronize()
    assert torch.equal(other[0], ref[1][0]) and torch.equal(here[0], ref[0][0])
    pool = torch.cuda.graph_pool_handle()
    graphs = []
    for x in dev:                                            # two graphs of one memory pool
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            out = call(x)
        graphs.append((graph, out))
    for i in (0, 1, 0):
        graphs[i][0].replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[i][1][0], ref[i][0]) and torch.equal(graphs[i][1][1], ref[i][1])
    dev[0][4].sub_(70)                                       # another length in the same graph
    graphs[0][0].replay()
    now = call(dev[0])
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][0], now[0]) and torch.equal(graphs[0][1][1], now[1])


def test_single_tokens_match_the_sparse_surface():
    # the same cache through the op that attends to selected blocks, all of them selected
    q, kc, vc, table, lens, _, _ = problem([1] * 4, [100, 63, 300, 511], 16, 2, 128, 128, 64, torch.bfloat16, 8, fill=0.0)
    blocks = 8
    idx = torch.arange(blocks, dtype=torch.int32).expand(4, 2, blocks).contiguous()
    o, lse = ops_b200.sparse_flash_attention_paged(q.cuda(), kc.cuda(), vc.cuda(), idx.cuda(), table.cuda(), lens.cuda(), 64,
                                                   max_seqlen_k=512)
    o2, lse2 = ops_b200.tree_attention_paged(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), lens.cuda())
    # both carry the tolerance of the tests above
    assert float((lse - lse2).abs().max()) < 1e-3 and float((o.float() - o2.float()).abs().max()) < 2e-2


def test_status_word_stays_clear():
    import ctypes
    from ops_b200 import _lib
    status = ctypes.c_int32(-1)
    _lib.check(_lib.load().sfa_device_status(torch.cuda.current_stream().cuda_stream, ctypes.byref(status)), "status")
    assert status.value == 0
