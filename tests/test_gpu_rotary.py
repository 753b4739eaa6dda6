"""GPU: norm and rotary positions (forward, backward, and stored into pages)
against the 64-bit definition.

Tolerances.  Every output is computed in fp32 and rounded once, so an element
is off by at most half a step of its type, ``eps / 2 * |value|``, plus the fp32
error.  In units of 2^-24: the sum of squares adds at most 8 * 4 terms per lane
and 5 lane exchanges (a relative error of 40, halved by the square root), the
reciprocal root and three products add 5, the angle is off by pi / 2 (its
rounding to a float of at most one half turn), sine and cosine by 4, each turned
element joins two products: below 64 of the pair's size, at most twice the
row's largest element.  Backward doubles the number of products and subtracts
two terms, whose sizes the oracle returns; a weight gradient adds a chain of at
most 128 terms per lane, warp and CTA, each off by the forward's error."""
import pytest
import torch

import ops_b200
from oracle import rotary_oracle as R

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def check(name, got, ref, size, units):
    half_step = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps    # one subnormal step
    g = got.detach().double().cpu()
    assert g.shape == ref.shape and torch.isfinite(g).all(), name
    tol = half_step * (ref.abs() + units * U * size) + units * U * size + tiny
    off = ((g - ref).abs() / tol).max() if g.numel() else 0.0
    assert off <= 1.0, f"{name}: {float(off):.3f} of the tolerance"


def row_size(ref):
    return 2 * ref.abs().amax(-1, keepdim=True)


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(shape, generator=g)).to(dtype)


# (tokens shape, Hq, Hk, D, rot, start, interleaved, dtype, positions from, weights)
SHAPES = [
    ((2, 37), 8, 2, 128, 128, 0, False, torch.bfloat16, 0, True),
    ((2, 37), 8, 2, 128, 128, 0, True, torch.bfloat16, 5, True),
    ((1, 301), 10, 2, 96, 48, 48, True, torch.float16, 120000, True),
    ((61,), 5, 1, 64, 32, 0, False, torch.float32, 1 << 20, True),
    ((1,), 64, 8, 128, 128, 0, False, torch.bfloat16, 131071, True),
    ((3, 5), 3, 3, 256, 64, 192, False, torch.bfloat16, 0, True),
    ((7,), 16, 1, 576, 64, 512, True, torch.bfloat16, 32000, True),     # latent kv: the last 64 dims turn
    ((9,), 2, 1, 1024, 1024, 0, False, torch.float16, 0, True),
    ((33,), 4, 2, 8, 8, 0, True, torch.float32, 0, True),
    ((33,), 4, 2, 24, 16, 8, False, torch.float16, 0, True),
    ((11,), 3, 2, 50, 18, 7, False, torch.bfloat16, 9, True),           # no vector form: odd offsets
    ((11,), 3, 2, 37, 36, 1, True, torch.float32, 9, True),
    ((2, 130), 6, 2, 80, 80, 0, False, torch.bfloat16, 0, False),       # rotation alone
    ((2, 13), 6, 2, 80, 0, 0, False, torch.bfloat16, 0, True),          # norm alone
    ((4, 1100), 24, 8, 64, 64, 0, False, torch.bfloat16, 0, True),      # several items per warp
]


def inputs(case, seed=0):
    lead, hq, hk, D, rot, start, inter, dtype, first, weights = case
    q, k = make((*lead, hq, D), dtype, seed), make((*lead, hk, D), dtype, seed + 1)
    w = [(1 + 0.2 * make((D,), torch.float32, seed + 2 + i)) if weights else None for i in range(2)]
    pos = (first + torch.arange(lead[-1])).to(torch.int64 if first % 2 else torch.int32).expand(lead).contiguous()
    f = ops_b200.rotary_frequencies(rot, scaling="yarn", factor=4.0)[0] if rot else None
    return q, k, w, (pos if rot else None), f, dict(eps=1e-6, start=start, interleaved=inter, amplitude=1.14 if rot else 1.0)


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


@pytest.mark.parametrize("case", SHAPES, ids=lambda c: "x".join(str(v).replace("torch.", "") for v in c))
def test_forward_and_gradients(case):
    q, k, w, pos, f, kw = inputs(case)
    gq, gk, gwq, gwk, gpos, gf = cuda(q, k, w[0], w[1], pos, f)
    leaves = [t.requires_grad_() for t in (gq, gk, gwq, gwk) if t is not None]
    oq, ok = ops_b200.qk_norm_rotary(gq, gk, gpos, gf, gwq, gwk, **kw)
    dq, dk = make(q.shape, q.dtype, 11), make(k.shape, k.dtype, 12)
    grads = torch.autograd.grad([oq, ok], leaves, cuda(dq, dk))
    for i, (x, wi, o, dy) in enumerate(((q, w[0], oq, dq), (k, w[1], ok, dk))):
        ref = R.forward(x, wi, pos, f, **kw)
        check("forward", o, ref, row_size(ref), 64)
        dx, dw, size, dsize = R.backward(x, wi, dy, pos, f, **kw)
        check("dx", grads[i], dx, size, 256)
        if wi is not None:
            check("dweight", grads[2 + i], dw, dsize, 256)


def test_gradient_against_differences():
    # central differences of the kernel's own fp32 forward, step 2^-7: the truncation is the third derivative
    # times 2^-14 / 6, the rounding 2^-17 of the loss's terms
    case = ((3,), 2, 1, 16, 16, 0, False, torch.float32, 3, True)
    q, k, w, pos, f, kw = inputs(case)
    gq, gk, wq, wk, gpos, gf = cuda(q, k, w[0], w[1], pos, f)
    cq, ck = cuda(make(q.shape, q.dtype, 21), make(k.shape, k.dtype, 22))

    def loss(a, b):
        oq, ok = ops_b200.qk_norm_rotary(a, gk, gpos, gf, b, wk, **kw)
        return (oq.double() * cq.double()).sum() + (ok.double() * ck.double()).sum()

    gq.requires_grad_()
    wq.requires_grad_()
    dq, dw = torch.autograd.grad(loss(gq, wq), [gq, wq])
    h = 2.0 ** -7
    for t, d in ((gq, dq), (wq, dw)):
        flat = t.detach().clone().view(-1)
        for i in range(0, flat.numel(), 5):
            vals = []
            for s in (h, -h):
                moved = flat.clone()
                moved[i] += s
                moved = moved.view(t.shape)
                vals.append(float(loss(moved if t is gq else gq.detach(), moved if t is wq else wq.detach())))
            # the terms of the loss are below 4 and at most 96 of them; third derivatives of x / |x| below 32
            assert abs((vals[0] - vals[1]) / (2 * h) - float(d.view(-1)[i])) < 32 * h * h / 6 + 96 * 4 * 2.0 ** -23 / h


def test_strides_orders_and_broadcast_gradients():
    # SBHD tensors, a slice of a wider projection, batch-broadcast positions, expanded output gradients
    S, B, D = 29, 3, 64
    wide = make((S, B, 10, D + 8), torch.bfloat16, 1).cuda()
    q, k = wide[:, :, :8, :D].permute(1, 0, 2, 3), wide[:, :, 8:, 8:].permute(1, 0, 2, 3)
    pos = torch.arange(S, device="cuda")
    f, _ = ops_b200.rotary_frequencies(D, device="cuda")
    wide.requires_grad_()
    q, k = wide[:, :, :8, :D].permute(1, 0, 2, 3), wide[:, :, 8:, 8:].permute(1, 0, 2, 3)
    oq, ok = ops_b200.qk_norm_rotary(q, k, pos, f)
    (oq.sum() + 2 * ok.float().sum()).backward()
    for x, o in ((q, oq), (k, ok)):
        ref = R.forward(x.detach().cpu(), None, pos.cpu().expand(B, S), f.cpu())
        check("forward", o, ref, row_size(ref), 64)
    ref = torch.zeros(wide.shape, dtype=torch.float64)
    one = torch.ones(B, S, 8, D, dtype=torch.float64)
    ref[:, :, :8, :D] += R.backward(one, None, one, pos.cpu().expand(B, S), f.cpu())[0].permute(1, 0, 2, 3)
    two = 2 * one[:, :, :2]
    ref[:, :, 8:, 8:] += R.backward(two, None, two, pos.cpu().expand(B, S), f.cpu())[0].permute(1, 0, 2, 3)
    # one more rounding: autograd adds slices of the wide gradient (zeros elsewhere)
    check("wide gradient", wide.grad, ref, torch.full_like(ref[..., :1], 4.0), 64)


@pytest.mark.parametrize("inter,D,rot,start", [(False, 128, 64, 64), (True, 30, 10, 3)])
def test_rotary_embedding_alone(inter, D, rot, start):
    x, pos = make((2, 17, 3, D), torch.float32, 4), torch.randint(-50, 1 << 30, (17,), generator=torch.Generator().manual_seed(1))
    f, a = ops_b200.rotary_frequencies(rot, base=500000.0, scaling="linear", factor=8.0)
    gx = x.cuda().requires_grad_()
    y = ops_b200.rotary_embedding(gx, pos.cuda(), f.cuda(), interleaved=inter, start=start, amplitude=a)
    # the 64-bit angle itself carries 2^-53 of up to 2^30 positions: 2^-23 of a radian, two units
    ref = R.forward(x, None, pos.expand(2, 17), f, start=start, interleaved=inter, amplitude=a)
    check("forward", y, ref, row_size(ref), 68)
    dy = make(x.shape, x.dtype, 5)
    dx, _, size, _ = R.backward(x, None, dy, pos.expand(2, 17), f, start=start, interleaved=inter, amplitude=a)
    check("dx", torch.autograd.grad(y, gx, dy.cuda())[0], dx, 2 * size, 68)


def test_empty_batches_and_partial_needs():
    f, _ = ops_b200.rotary_frequencies(64, device="cuda")
    w = torch.ones(64, device="cuda", requires_grad=True)
    q = torch.empty(0, 4, 64, device="cuda", requires_grad=True)
    oq, ok = ops_b200.qk_norm_rotary(q, q[:, :1], torch.empty(0, dtype=torch.int32, device="cuda"), f, w, w)
    (oq.sum() + ok.sum()).backward()
    assert q.grad.shape == q.shape and torch.equal(w.grad, torch.zeros_like(w))
    # gradients of the weights alone, of bf16 weights in bf16, and of one tensor alone
    q, k = make((9, 4, 64), torch.bfloat16, 1).cuda(), make((9, 2, 64), torch.bfloat16, 2).cuda().requires_grad_()
    wb = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    pos = torch.arange(9, device="cuda", dtype=torch.int32)
    oq, ok = ops_b200.qk_norm_rotary(q, k, pos, f, wb, None)
    dq, dk = make((9, 4, 64), torch.bfloat16, 3).cuda(), make((9, 2, 64), torch.bfloat16, 4).cuda()
    gw, gk = torch.autograd.grad([oq, ok], [wb, k], [dq, dk])
    _, dw, _, dsize = R.backward(q.cpu(), wb.detach().cpu(), dq.cpu(), pos.cpu(), f.cpu())
    check("bf16 dweight", gw, dw, dsize, 256)
    dx, _, size, _ = R.backward(k.detach().cpu(), None, dk.cpu(), pos.cpu(), f.cpu())
    check("dk", gk, dx, 2 * size, 64)


def test_repeats_bit_for_bit():
    q, k, w, pos, f, kw = inputs(((4, 700), 16, 4, 128, 128, 0, False, torch.bfloat16, 0, True))
    args = cuda(q, k, pos, f, w[0], w[1])
    leaves = [args[i].requires_grad_() for i in (0, 1, 4, 5)]
    dy = cuda(make(q.shape, q.dtype, 1), make(k.shape, k.dtype, 2))

    def step():
        out = ops_b200.qk_norm_rotary(*args, **kw)
        return [*out, *torch.autograd.grad(out, leaves, dy)]

    first = step()
    for a, b in zip(first, step()):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ append
def pool_case(n, counts, hq, hk, D, Dv, page, dtype, seed, prefix_to=200):
    g = torch.Generator().manual_seed(seed)
    counts = torch.tensor(counts)
    prefix = torch.randint(0, prefix_to, (n,), generator=g)
    lens = (prefix + counts).to(torch.int32)
    width = int((lens.max() + page - 1) // page) + 1
    pages = n * width + 2
    table = torch.randperm(pages, generator=g)[: n * width].to(torch.int32).view(n, width)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)]).to(torch.int32)
    rows = int(cu[-1])
    q, k, v = make((rows, hq, D), dtype, seed), make((rows, hk, D), dtype, seed + 1), make((rows, hk, Dv), dtype, seed + 2)
    kc, vc = make((pages, page, hk, D), dtype, seed + 3), make((pages, page, hk, Dv), dtype, seed + 4)
    return q, k, v, kc, vc, table, lens, cu, prefix


@pytest.mark.parametrize("counts,hq,hk,D,Dv,page,dtype", [
    ([1], 64, 8, 128, 128, 64, torch.bfloat16),
    ([1] * 40, 8, 2, 64, 64, 16, torch.float16),
    ([3, 0, 16, 1, 0, 0, 7, 2], 6, 2, 96, 80, 24, torch.bfloat16),
    ([5, 9], 3, 1, 36, 36, 7, torch.float32),
    (list(range(70)), 4, 1, 64, 64, 32, torch.bfloat16),
])
def test_append_stores_exactly_its_rows(counts, hq, hk, D, Dv, page, dtype):
    n = len(counts)
    q, k, v, kc, vc, table, lens, cu, prefix = pool_case(n, counts, hq, hk, D, Dv, page, dtype, 3)
    g = torch.Generator().manual_seed(8)
    pos = torch.randint(0, 100000, (q.shape[0],), generator=g)
    f, _ = ops_b200.rotary_frequencies(D // 4 * 2)
    w = 1 + 0.1 * make((D,), torch.float32, 9)
    gk, gv = kc.cuda(), vc.cuda()
    out = ops_b200.qk_norm_rotary_append(*cuda(q, k, v, pos, f), gk, gv, *cuda(table, lens),
                                         cu_seqlens=None if counts == [1] * n else cu.cuda(),
                                         q_weight=w.cuda(), k_weight=w.cuda())
    ref = R.forward(q, w, pos, f)
    check("q", out, ref, row_size(ref), 64)
    kr = R.forward(k, w, pos, f)
    touched = torch.zeros(kc.shape[:2], dtype=torch.bool)
    got_k, got_v = gk.cpu(), gv.cpu()
    i = 0
    for s, c in enumerate(counts):
        for j in range(c):
            at = int(prefix[s]) + j
            p, r = int(table[s, at // page]), at % page
            touched[p, r] = True
            check("k", got_k[p, r], kr[i], row_size(kr[i]), 64)
            assert torch.equal(got_v[p, r], v[i])
            i += 1
    assert torch.equal(got_k[~touched], kc[~touched]) and torch.equal(got_v[~touched], vc[~touched])


def test_append_leaves_out_what_has_no_place():
    # a page of -1, a page id past the pool, a position behind the table, a length below its rows,
    # and rows behind the last sequence: q is still returned for all of them
    hk, D, page = 2, 64, 4
    cu = torch.tensor([0, 2, 4, 6, 9, 10], dtype=torch.int32)
    rows = 13
    q, k, v = make((rows, 4, D), torch.bfloat16, 1), make((rows, hk, D), torch.bfloat16, 2), make((rows, hk, D), torch.bfloat16, 3)
    kc = make((6, page, hk, D), torch.bfloat16, 4)
    table = torch.tensor([[0, -1], [1, 6], [2, 3], [4, -1], [-2000000000, 5]], dtype=torch.int32)
    lens = torch.tensor([5, 6, 9, 1, 8], dtype=torch.int32)
    # stored: seq 0 row 0 (page 0, row 3); seq 1 none (page 6 is outside); seq 2 row 0 (position 7: page 3, row 3);
    # seq 3 row 2 (position 0: page 4); seq 4 row 0 (position 7: page 5, row 3)
    gk, gv = kc.cuda(), kc.cuda()
    out = ops_b200.qk_norm_rotary_append(*cuda(q, k, v), None, None, gk, gv, *cuda(table, lens), cu_seqlens=cu.cuda())
    assert torch.equal(out.cpu(), q)
    want_k, want_v = kc.clone(), kc.clone()
    for row, p, r in ((0, 0, 3), (4, 3, 3), (8, 4, 0), (9, 5, 3)):
        want_k[p, r], want_v[p, r] = k[row], v[row]
    assert torch.equal(gk.cpu(), want_k) and torch.equal(gv.cpu(), want_v)


def test_append_past_32_bit_offsets():
    q, k, v, kc, vc, table, lens, cu, _ = pool_case(3, [2, 1, 5], 8, 8, 128, 128, 64, torch.bfloat16, 15)
    f, _ = ops_b200.rotary_frequencies(128, device="cuda")
    pos = torch.arange(8, dtype=torch.int32).cuda()
    rest = cuda(lens)
    small = [kc.cuda(), vc.cuda()]
    want = ops_b200.qk_norm_rotary_append(*cuda(q, k, v), pos, f, *small, table.cuda(), *rest, cu_seqlens=cu.cuda())
    pages = 2 ** 31 // (64 * 8 * 128) + 2 + kc.shape[0]
    big = []
    for c in (kc, vc):
        big.append(torch.zeros(pages, 64, 8, 128, dtype=torch.bfloat16, device="cuda"))
        big[-1][-kc.shape[0]:] = c.cuda()
    got = ops_b200.qk_norm_rotary_append(*cuda(q, k, v), pos, f, *big, (table + pages - kc.shape[0]).cuda(), *rest,
                                         cu_seqlens=cu.cuda())
    assert torch.equal(got, want)
    for b, c in zip(big, small):
        assert torch.equal(b[-kc.shape[0]:], c) and not b[:-kc.shape[0]].any()


def test_rows_past_32_bit_offsets():
    T = 2 ** 31 // (64 * 128) + 70
    f, _ = ops_b200.rotary_frequencies(128, device="cuda")
    pos = torch.arange(T, dtype=torch.int32, device="cuda")
    w = torch.rand(128, device="cuda")
    x = torch.zeros(T, 64, 128, dtype=torch.bfloat16, device="cuda")
    x[-64:] = make((64, 64, 128), torch.bfloat16, 4).cuda()
    x[-64:].mul_(2)
    x.requires_grad_()
    y, _ = ops_b200.qk_norm_rotary(x, x[:, :1], pos, f, w)
    tail = x.detach()[-64:].clone().requires_grad_()
    want, _ = ops_b200.qk_norm_rotary(tail, tail[:, :1], pos[-64:], f, w)
    assert torch.equal(y[-64:], want) and not y[:-64].any()
    dy = torch.zeros_like(y)
    dy[-64:] = make((64, 64, 128), torch.bfloat16, 5).cuda()
    dx, = torch.autograd.grad(y, x, dy)
    want, = torch.autograd.grad(want, tail, dy[-64:])
    assert torch.equal(dx[-64:], want) and not dx[:-64].any()


def test_append_on_another_stream_and_in_a_graph():
    q, k, v, kc, vc, table, lens, cu, _ = pool_case(6, [4] * 6, 8, 2, 64, 64, 16, torch.bfloat16, 5)
    f, _ = ops_b200.rotary_frequencies(64, device="cuda")
    pos = torch.arange(24, dtype=torch.int32).cuda()
    args = cuda(q, k, v)
    tb = cuda(table, lens)
    ref_k, ref_v = kc.cuda(), vc.cuda()
    ref = ops_b200.qk_norm_rotary_append(*args, pos, f, ref_k, ref_v, *tb, cu_seqlens=cu.cuda())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    gk, gv, gcu = kc.cuda(), vc.cuda(), cu.cuda()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        o = ops_b200.qk_norm_rotary_append(*args, pos, f, gk, gv, *tb, cu_seqlens=gcu)
    side.synchronize()
    assert torch.equal(o, ref) and torch.equal(gk, ref_k) and torch.equal(gv, ref_v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = ops_b200.qk_norm_rotary_append(*args, pos, f, gk, gv, *tb, cu_seqlens=gcu)
    args[1].mul_(2)                       # new rows for the replay (norm off: k doubles)
    graph.replay()
    ops_b200.qk_norm_rotary_append(*args, pos, f, ref_k, ref_v, *tb, cu_seqlens=gcu)
    torch.cuda.synchronize()
    assert torch.equal(o, ref) and torch.equal(gk, ref_k) and torch.equal(gv, ref_v)


def test_training_step_in_a_graph():
    q, k, w, pos, f, kw = inputs(((2, 64), 8, 2, 64, 64, 0, False, torch.bfloat16, 0, True))
    gq, gk, wq, wk, gpos, gf = cuda(q, k, w[0], w[1], pos, f)
    leaves = [t.requires_grad_() for t in (gq, gk, wq, wk)]
    dy = cuda(make(q.shape, q.dtype, 1), make(k.shape, k.dtype, 2))

    def step():
        out = ops_b200.qk_norm_rotary(gq, gk, gpos, gf, wq, wk, **kw)
        return torch.autograd.grad(out, leaves, dy)

    ref = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        graphs.append((graph, got))
    for graph, got in graphs + graphs[:1]:
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(ref, got):
            assert torch.equal(a, b)
