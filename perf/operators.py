"""Cases, plain forms and 64-bit answers for the serving-step operators around the paged kv cache: norm and
rotary positions of queries and keys (with their gradients), the same step written straight into a paged
cache, attention of a tree of drafted tokens over that cache, and the page operations between steps.

``run`` computes an operator either in elementary torch operations (``own`` false) or through ``ops_b200``
(``own`` true); both take what ``prepare`` made.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # training step of the 8192-token GQA configuration: whole-head rotation in the half layout
        dict(name="rotary_train", op="rotary", batch=4, length=8192, hq=64, hk=4, dim=128, rot=128, start=0,
             interleaved=False, dtype="bf16", base=10000.0, factor=1.0, first=0),
        # packed training batch of odd length, rotation of the second half of the head, interleaved pairs,
        # positions far into a context stretched eightfold
        dict(name="rotary_odd", op="rotary", batch=1, length=5003, hq=10, hk=2, dim=96, rot=48, start=48,
             interleaved=True, dtype="fp16", base=500000.0, factor=8.0, first=120000),
        # one new token of one sequence: the smallest call of a decode loop
        dict(name="append_one", op="append", seqs=1, nodes=1, kv_min=1000, kv_max=1000, hq=64, hk=8, dim=128,
             rot=128, start=0, interleaved=False, dtype="bf16", page=64, base=10000.0, factor=1.0),
        # drafted trees of a served batch, lengths ragged, pages of an odd size
        dict(name="append_tree", op="append", seqs=37, nodes=16, kv_min=200, kv_max=1900, hq=64, hk=8, dim=128,
             rot=64, start=0, interleaved=True, dtype="bf16", page=48, base=10000.0, factor=4.0),
        # one token over a short cache: latency
        dict(name="tree_small", op="tree", seqs=1, nodes=1, kv_min=700, kv_max=700, hq=16, hk=1, dim=64, dim_v=64,
             page=16, dtype="bf16", shape="chain"),
        # small heads in odd numbers, fp16, pages that end inside a tile, chains of drafts
        dict(name="tree_odd", op="tree", seqs=5, nodes=13, kv_min=300, kv_max=4100, hq=12, hk=4, dim=96, dim_v=80,
             page=24, dtype="fp16", shape="chain"),
        # plain decoding of a served batch: one token a sequence, long ragged caches
        dict(name="tree_decode", op="tree", seqs=16, nodes=1, kv_min=4096, kv_max=32768, hq=64, hk=8, dim=128,
             dim_v=128, page=64, dtype="bf16", shape="chain"),
        # verification of 64-node trees
        dict(name="tree_64", op="tree", seqs=8, nodes=64, kv_min=4096, kv_max=16384, hq=64, hk=8, dim=128,
             dim_v=128, page=64, dtype="bf16", shape="tree"),
        # one very long context, a small tree
        dict(name="tree_long", op="tree", seqs=1, nodes=16, kv_min=131072, kv_max=131072, hq=64, hk=8, dim=128,
             dim_v=128, page=128, dtype="bf16", shape="tree"),
        # a beam step: losing beams freed, winning ones forked, room made for the next token
        dict(name="pages_beam", op="beam", seqs=64, kv_min=500, kv_max=1500, hk=8, dim=128, page=64, layers=8),
        # after verification: the accepted path of every tree moved together, the rest of the rows given back
        dict(name="pages_accept", op="accept", seqs=128, nodes=32, kv_min=100, kv_max=600, hk=8, dim=128, page=32,
             layers=16),
        # a fragmented pool compacted into its first pages
        dict(name="pages_compact", op="compact", seqs=96, kv_min=200, kv_max=3000, hk=8, dim=128, page=64, layers=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "append", "append", "tree", "tree", "tree", "beam", "accept", "compact"])
    hk = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"] if op in ("rotary", "append") else ["bf16", "bf16", "fp16"])
    dim = rng.choice([64, 80, 96, 112, 128, 128, 192, 256])
    if op in ("rotary", "append"):
        rot = rng.choice([dim, dim // 2 // 8 * 8, 16])
        c = dict(op=op, hq=hk * group, hk=hk, dim=dim, rot=rot, start=rng.choice([0, dim - rot]),
                 interleaved=rng.random() < 0.5, dtype=dtype, base=rng.choice([10000.0, 500000.0]),
                 factor=rng.choice([1.0, 2.0, 8.0]))
        if op == "rotary":
            return dict(c, batch=rng.randint(1, 4), length=_log(rng, 1, 6000), first=rng.choice([0, 0, 100000]))
        lo = _log(rng, 20, 2000)
        return dict(c, seqs=_log(rng, 1, 64), nodes=_log(rng, 1, 20), kv_min=lo, kv_max=lo + _log(rng, 1, 500),
                    page=rng.choice([16, 32, 48, 64, 128]))
    if op == "tree":
        nodes, seqs = _log(rng, 1, 64), _log(rng, 1, 16)
        most = min(32768, 400_000 // seqs, 4_000_000 // (seqs * nodes))
        hi = _log(rng, 80, most)
        return dict(op=op, seqs=seqs, nodes=nodes, kv_min=max(nodes, hi // rng.choice([1, 2, 8])), kv_max=max(nodes, hi),
                    hq=hk * group, hk=hk, dim=dim, dim_v=rng.choice([dim, 64, 128]),
                    page=rng.choice([8, 16, 24, 32, 64, 128]), dtype=dtype, shape=rng.choice(["tree", "chain"]))
    c = dict(op=op, seqs=_log(rng, 2, 96), hk=hk, dim=dim, page=rng.choice([16, 24, 32, 64, 128]),
             layers=rng.randint(1, 8), kv_min=_log(rng, 20, 200), kv_max=_log(rng, 200, 1200))
    return dict(c, nodes=rng.randint(2, 32)) if op == "accept" else c


# ------------------------------------------------------------------------------------------------ inputs
def _frequencies(case, device):
    """Radians a position for each rotated pair; a stretched context turns its slow pairs `factor` times slower
    (pairs that turn more than 32 times in the first 8192 positions stay as they are)."""
    rot = case["rot"]
    f = torch.pow(torch.tensor(case["base"], dtype=torch.float64),
                  -torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if case["factor"] != 1.0:
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0, 1)
        f = f * keep + f / case["factor"] * (1 - keep)
    return f.to(device)


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype) if dtype != torch.bfloat16 \
        else torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _lens(case, g):
    return torch.randint(case["kv_min"], case["kv_max"] + 1, (case["seqs"],), generator=g, device="cuda").to(torch.int32)


def _table(lens, page, width, g, spare):
    """Block table over a shuffled pool: sequence s holds ceil(lens / page) pages; -1 behind them."""
    n = lens.numel()
    pages = (lens.to(torch.int64) + page - 1) // page
    held = torch.arange(width, device="cuda")[None, :] < pages[:, None]
    total = n * width + spare
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32)[: n * width].view(n, width)
    return torch.where(held, perm, torch.full_like(perm, -1)), total


def _prepare_rotary(case, g):
    B, T, D, dt = case["batch"], case["length"], case["dim"], DTYPES[case["dtype"]]
    s = dict(q=_normal(g, (B, T, case["hq"], D), dt), k=_normal(g, (B, T, case["hk"], D), dt))
    s["gq"], s["gk"] = _normal(g, s["q"].shape, dt), _normal(g, s["k"].shape, dt)
    s["wq"] = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    s["wk"] = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    s["positions"] = (case["first"] + torch.arange(T, device="cuda", dtype=torch.int32)).expand(B, T).contiguous()
    for x in ("q", "k", "wq", "wk"):
        s[x].requires_grad_(True)
    return s


def _prepare_append(case, g):
    n, m, D, dt, page = case["seqs"], case["nodes"], case["dim"], DTYPES[case["dtype"]], case["page"]
    rows = n * m
    lens = _lens(case, g) + m                                   # with the new rows
    width = (case["kv_max"] + m + page - 1) // page
    table, total = _table(lens, page, width, g, 3)
    s = dict(q=_normal(g, (rows, case["hq"], D), dt), k=_normal(g, (rows, case["hk"], D), dt),
             v=_normal(g, (rows, case["hk"], D), dt), table=table, lens=lens)
    s["k_cache"] = _normal(g, (total, page, case["hk"], D), dt)
    s["v_cache"] = _normal(g, (total, page, case["hk"], D), dt)
    s["wq"] = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    s["wk"] = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    s["cu"] = torch.arange(n + 1, device="cuda", dtype=torch.int32) * m
    # a node's position is its prefix plus its depth in the tree
    depth = (torch.rand(n, m, generator=g, device="cuda") * torch.arange(1, m + 1, device="cuda")).long()
    s["positions"] = ((lens - m)[:, None] + depth).to(torch.int32).view(-1)
    return s


def _prepare_tree(case, g):
    n, m, dt, page, hk = case["seqs"], case["nodes"], DTYPES[case["dtype"]], case["page"], case["hk"]
    lens = _lens(case, g)
    width = (case["kv_max"] + page - 1) // page
    table, total = _table(lens, page, width, g, 3)
    s = dict(q=_normal(g, (n * m, case["hq"], case["dim"]), dt), table=table, lens=lens, max_k=case["kv_max"], max_q=m)
    s["k_cache"] = _normal(g, (total, page, hk, case["dim"]), dt)
    s["v_cache"] = _normal(g, (total, page, hk, case["dim_v"]), dt)
    s["cu"] = torch.arange(n + 1, device="cuda", dtype=torch.int32) * m
    # node j hangs on a node before it (or on the prefix): the trees of a drafting model
    up = (torch.rand(n, m, generator=g, device="cuda") * torch.arange(0, m, device="cuda")).long()
    s["parents"] = (up - (torch.arange(m, device="cuda") == 0).long()).to(torch.int32).view(-1) \
        if case["shape"] == "tree" else None
    return s


def _pools(case, g, total):
    return [_normal(g, (total, case["page"], case["hk"], case["dim"]), torch.bfloat16) for _ in range(2 * case["layers"])]


def _refcounts(table, total):
    held = table[table >= 0].long()
    return torch.zeros(total, dtype=torch.int32, device="cuda").index_add_(0, held, torch.ones_like(held, dtype=torch.int32))


def _prepare_pages(case, g):
    n, page, op = case["seqs"], case["page"], case["op"]
    lens = _lens(case, g)
    extra = case.get("nodes", 1)
    width = (case["kv_max"] + extra + page - 1) // page
    if op == "accept":
        lens = lens + case["nodes"]
    table, total = _table(lens, page, width, g, 5)
    s = dict(table=table, lens=lens, pools=_pools(case, g, total), refcounts=_refcounts(table, total))
    if op == "beam":
        lost = torch.randperm(n, generator=g, device="cuda")[: n // 2]
        won = torch.ones(n, dtype=torch.bool, device="cuda")
        won[lost] = False
        winners = won.nonzero()[:, 0]
        s["dst"] = lost.to(torch.int32)
        s["src"] = winners[torch.randint(0, winners.numel(), (lost.numel(),), generator=g, device="cuda")].to(torch.int32)
        s["keep"] = torch.where(won, lens, torch.zeros_like(lens))      # what each row keeps: losers nothing
        s["one"] = torch.ones_like(lens)
    elif op == "accept":
        m = case["nodes"]
        # a root-to-leaf path of each tree: ascending node numbers, -1 behind
        take = torch.rand(n, m, generator=g, device="cuda") < 4.0 / m
        node = torch.where(take, torch.arange(m, device="cuda").expand(n, m), torch.full((n, m), m, device="cuda"))
        node = node.sort(1)[0]
        s["accepted"] = torch.where(node < m, node, torch.full_like(node, -1)).to(torch.int32)
        s["drafted"] = torch.full((n,), m, dtype=torch.int32, device="cuda")
        s["lens0"], s["table0"], s["refcounts0"] = lens.clone(), table.clone(), s["refcounts"].clone()
    else:
        s["table0"], s["refcounts0"] = table.clone(), s["refcounts"].clone()
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    make = {"rotary": _prepare_rotary, "append": _prepare_append, "tree": _prepare_tree}.get(case["op"], _prepare_pages)
    s = make(case, g)
    s["case"] = dict(case)
    if "rot" in case:
        s["frequencies"] = _frequencies(case, "cuda")
        s["amplitude"] = 1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _pairs(x, case):
    """The rotated part of x [..., D] as its two members of each pair [..., rot / 2]."""
    part = x[..., case["start"]: case["start"] + case["rot"]]
    if case["interleaved"]:
        return part[..., 0::2], part[..., 1::2]
    return part[..., : case["rot"] // 2], part[..., case["rot"] // 2:]


def _joined(x, a, b, case):
    part = torch.stack([a, b], -1).flatten(-2) if case["interleaved"] else torch.cat([a, b], -1)
    return torch.cat([x[..., : case["start"]], part, x[..., case["start"] + case["rot"]:]], -1)


def _turned(x, cos, sin, case, sign):
    a, b = _pairs(x, case)
    return _joined(x, a * cos - sign * b * sin, b * cos + sign * a * sin, case)


def _cos_sin(s):
    angle = s["positions"].double()[..., None] * s["frequencies"]
    return [(f(angle) * s["amplitude"]).float()[..., None, :] for f in (torch.cos, torch.sin)]


EPS = 1e-6


def _norm_rotary(x, w, cos, sin, case):
    x = x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return _turned(x * r * w, cos, sin, case, 1.0)


def _norm_rotary_grad(x, w, g, cos, sin, case):
    dt, x = x.dtype, x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    h = _turned(g.float(), cos, sin, case, -1.0)
    n = x * r
    dw = (h * n).flatten(0, -2).sum(0, dtype=torch.float64).float()
    h = h * w
    return (r * (h - n * (h * n).mean(-1, keepdim=True))).to(dt), dw


def _plain_rotary(s):
    case, dt = s["case"], s["q"].dtype
    cos, sin = _cos_sin(s)
    q, k, wq, wk = (s[x].detach() for x in ("q", "k", "wq", "wk"))
    oq, ok = (_norm_rotary(x, w, cos, sin, case).to(dt) for x, w in ((q, wq), (k, wk)))
    (dq, dwq), (dk, dwk) = (_norm_rotary_grad(x, w, g, cos, sin, case) for x, w, g in ((q, wq, s["gq"]), (k, wk, s["gk"])))
    return [oq, ok, dq, dk, dwq, dwk]


def _slots(s, m, page):
    """(page, row) of each new cache row: the last m rows of every sequence."""
    at = (s["lens"].long() - m)[:, None] + torch.arange(m, device="cuda")
    return s["table"].long().gather(1, at // page).view(-1), (at % page).view(-1)


def _plain_append(s):
    case, dt = s["case"], s["q"].dtype
    cos, sin = _cos_sin(s)
    pg, row = _slots(s, case["nodes"], case["page"])
    s["k_cache"][pg, row] = _norm_rotary(s["k"], s["wk"], cos, sin, case).to(dt)
    s["v_cache"][pg, row] = s["v"]
    return [_norm_rotary(s["q"], s["wq"], cos, sin, case).to(dt), s["k_cache"], s["v_cache"]]


def _gathered(cache, table, most):
    return cache[table.long().clamp(min=0)].flatten(1, 2)[:, :most].float()


def _seen(s, n, m, most):
    """[n, m, most]: which cache rows each drafted node sees: the prefix, its ancestors and itself."""
    node = torch.arange(most, device="cuda")[None, :] - (s["lens"].long() - m)[:, None]
    if s["parents"] is None:
        up = torch.tril(torch.ones(m, m, device="cuda", dtype=torch.bool)).expand(n, m, m)
    else:
        p = s["parents"].view(n, m, 1).long()
        reach = (p == torch.arange(m, device="cuda")).float() + torch.eye(m, device="cuda")
        for _ in range(max(1, (m - 1).bit_length())):
            reach = (reach @ reach).clamp(max=1.0)
        up = reach > 0
    inside = up.gather(2, node.clamp(0, m - 1)[:, None, :].expand(n, m, most))
    return torch.where((node < 0)[:, None, :], True, inside & (node < m)[:, None, :])


def _plain_tree(s):
    case, dt = s["case"], s["q"].dtype
    n, m, hk, most = case["seqs"], case["nodes"], case["hk"], s["max_k"]
    group = case["hq"] // hk
    k, v = _gathered(s["k_cache"], s["table"], most), _gathered(s["v_cache"], s["table"], most)
    q = s["q"].float().view(n, m, hk, group, -1).permute(0, 2, 1, 3, 4).reshape(n, hk, m * group, -1)
    score = q @ k.permute(0, 2, 3, 1) / math.sqrt(case["dim"])
    seen = _seen(s, n, m, most)[:, None, :, None, :]
    score = torch.where(seen, score.view(n, hk, m, group, most), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    o = (p / total).view(n, hk, m * group, most) @ v.permute(0, 2, 1, 3)
    o = o.view(n, hk, m, group, -1).permute(0, 2, 1, 3, 4).reshape(n * m, case["hq"], -1).to(dt)
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 2, 1, 3).reshape(n * m, case["hq"])
    return [o, lse]


def _plain_trim(s, keep, page):
    table, lens = s["table"], s["lens"]
    left = torch.minimum(lens, keep)
    col = torch.arange(table.shape[1], device="cuda")[None, :]
    gone = (col >= ((left + page - 1) // page)[:, None]) & (table >= 0)
    s["refcounts"].index_add_(0, torch.where(gone, table, 0).long().view(-1), -gone.to(torch.int32).view(-1))
    table.copy_(torch.where(gone, -1, table))
    lens.copy_(left)


def _free_pages(s):
    """Free page numbers in ascending order."""
    return torch.sort((s["refcounts"] > 0).to(torch.int8), stable=True)[1].to(torch.int32)


def _plain_beam(s):
    case, page = s["case"], s["case"]["page"]
    table, lens, refs = s["table"], s["lens"], s["refcounts"]
    _plain_trim(s, s["keep"], page)
    src, dst = s["src"].long(), s["dst"].long()
    # fork: whole pages are shared, a partly filled last page is copied to the lowest free pages in order
    length = lens[src]
    last, part = (length // page).long(), length % page > 0
    new = _free_pages(s)[(torch.cumsum(part.int(), 0) - 1).clamp(min=0)]
    row = table[src]
    old = row.gather(1, last.clamp(max=table.shape[1] - 1)[:, None])[:, 0]
    here = (torch.arange(table.shape[1], device="cuda")[None, :] == last[:, None]) & part[:, None]
    row = torch.where(here, new[:, None], row)
    refs.index_add_(0, row.clamp(min=0).long().view(-1), (row >= 0).to(torch.int32).view(-1))
    table[dst] = row
    lens[dst] = length
    for pool in s["pools"]:
        pool[new[part].long()] = pool[old[part].long()]
    # room for one more row a sequence: a new page where the last one is full
    need = lens % page == 0
    fresh = _free_pages(s)[(torch.cumsum(need.int(), 0) - 1).clamp(min=0)]
    here = (torch.arange(table.shape[1], device="cuda")[None, :] == (lens // page)[:, None]) & need[:, None]
    table.copy_(torch.where(here, fresh[:, None], table))
    refs.index_add_(0, fresh.long(), need.to(torch.int32))
    lens.add_(1)
    done = torch.ones_like(s["src"])
    return [refs, table, lens, done, torch.ones_like(lens)] + s["pools"]


def _restored(s):
    """The state as before the step, so that every pass does the whole step."""
    s["table"].copy_(s["table0"])
    s["refcounts"].copy_(s["refcounts0"])
    if "lens0" in s:
        s["lens"].copy_(s["lens0"])


def _plain_accept(s):
    case, page = s["case"], s["case"]["page"]
    _restored(s)
    acc, table = s["accepted"].long(), s["table"].long()
    prefix = (s["lens"] - s["drafted"]).long()[:, None]
    count = (acc >= 0).sum(1)
    ok = torch.arange(acc.shape[1], device="cuda")[None, :] < count[:, None]
    here, there = prefix + acc.clamp(min=0), prefix + torch.arange(acc.shape[1], device="cuda")
    there = torch.where(ok, there, prefix)
    a = (table.gather(1, here // page)[ok], (here % page)[ok])
    b = (table.gather(1, there // page)[ok], (there % page)[ok])
    for pool in s["pools"]:
        pool[b] = pool[a]
    keep = (prefix[:, 0] + count).to(torch.int32)
    _plain_trim(s, keep, page)
    return [keep, s["refcounts"], s["table"], s["lens"]] + s["pools"]


def _plain_compact(s):
    _restored(s)
    refs, table = s["refcounts"], s["table"]
    used = refs > 0
    live = used.sum()
    num = torch.arange(refs.numel(), device="cuda")
    movers, holes = (used & (num >= live)).nonzero()[:, 0], (~used & (num < live)).nonzero()[:, 0]
    to = num.clone()
    to[movers] = holes
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), -1))
    refs[holes] = refs[movers]
    refs[movers] = 0
    for pool in s["pools"]:
        pool[holes] = pool[movers]
    return [refs, table, live.to(torch.int32).view(1)] + s["pools"]


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own_rotary(s):
    import ops_b200
    case = s["case"]
    oq, ok = ops_b200.qk_norm_rotary(s["q"], s["k"], s["positions"], s["frequencies"], s["wq"], s["wk"], eps=EPS,
                                     interleaved=case["interleaved"], start=case["start"], amplitude=s["amplitude"])
    grads = torch.autograd.grad([oq, ok], [s["q"], s["k"], s["wq"], s["wk"]], [s["gq"], s["gk"]])
    return [oq.detach(), ok.detach(), *grads]


def _own_append(s):
    import ops_b200
    case = s["case"]
    q = ops_b200.qk_norm_rotary_append(s["q"], s["k"], s["v"], s["positions"], s["frequencies"], s["k_cache"],
                                       s["v_cache"], s["table"], s["lens"], cu_seqlens=s["cu"], q_weight=s["wq"],
                                       k_weight=s["wk"], eps=EPS, interleaved=case["interleaved"],
                                       start=case["start"], amplitude=s["amplitude"])
    return [q, s["k_cache"], s["v_cache"]]


def _own_tree(s):
    import ops_b200
    o, lse = ops_b200.tree_attention_paged(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                           parents=s["parents"], cu_seqlens=s["cu"], max_seqlen_q=s["max_q"],
                                           max_seqlen_k=s["max_k"])
    return [o, lse]


def _own_beam(s):
    import ops_b200
    page = s["case"]["page"]
    ops_b200.paged_cache_trim(s["refcounts"], s["table"], s["lens"], s["keep"], page)
    forked = ops_b200.paged_cache_fork(s["refcounts"], s["table"], s["lens"], s["src"], s["dst"], s["pools"])
    granted = ops_b200.paged_cache_reserve(s["refcounts"], s["table"], s["lens"], s["one"], page)
    return [s["refcounts"], s["table"], s["lens"], forked, granted] + s["pools"]


def _own_accept(s):
    import ops_b200
    _restored(s)
    keep = ops_b200.paged_cache_accept(s["pools"], s["table"], s["lens"], s["accepted"], s["drafted"])
    ops_b200.paged_cache_trim(s["refcounts"], s["table"], s["lens"], keep, s["case"]["page"])
    return [keep, s["refcounts"], s["table"], s["lens"]] + s["pools"]


def _own_compact(s):
    import ops_b200
    _restored(s)
    live = ops_b200.paged_cache_compact(s["refcounts"], s["table"], s["pools"])
    return [s["refcounts"], s["table"], live] + s["pools"]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "append": _own_append, "tree": _own_tree, "beam": _own_beam,
                "accept": _own_accept, "compact": _own_compact}[op](state)
    return {"rotary": _plain_rotary, "append": _plain_append, "tree": _plain_tree, "beam": _plain_beam,
            "accept": _plain_accept, "compact": _plain_compact}[op](state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    op, size = case["op"], {"bf16": 2, "fp16": 2, "fp32": 4}[case.get("dtype", "bf16")]
    if op == "rotary":
        n = case["batch"] * case["length"] * (case["hq"] + case["hk"]) * case["dim"]
        return {"bytes": 4 * n * size + 4 * case["batch"] * case["length"], "flops": 30 * n}
    if op == "append":
        rows, hq, hk, d = case["seqs"] * case["nodes"], case["hq"], case["hk"], case["dim"]
        return {"bytes": rows * (2 * hq + 4 * hk) * d * size + 8 * rows, "flops": 10 * rows * (hq + hk) * d}
    mean = (case["kv_min"] + case["kv_max"]) / 2
    if op == "tree":
        n, m, hq, d = case["seqs"], case["nodes"], case["hq"], case["dim"] + case["dim_v"]
        return {"bytes": n * mean * case["hk"] * d * size + n * m * hq * d * size, "flops": 2 * n * m * hq * mean * d}
    row = case["hk"] * case["dim"] * 2 * 2 * case["layers"]             # K and V of every layer, bf16
    n, page = case["seqs"], case["page"]
    if op == "beam":                                                    # the partly filled last pages, read and written
        return {"bytes": 2 * (n // 2) * page * row + 8 * n * mean / page, "flops": 0}
    if op == "accept":                                                  # about four rows a tree
        return {"bytes": 2 * 4 * n * row + 8 * n * mean / page, "flops": 0}
    pages = n * (mean + page / 2) / page                                # live pages above the live count move
    width = (case["kv_max"] + 1 + page - 1) // page
    return {"bytes": 2 * pages * max(0.0, 1 - pages / (n * width)) * page * row + 8 * n * width, "flops": 0}


# ------------------------------------------------------------------------------------------------ 64-bit answers
def _exact_rows(x, w, angle, case, amplitude):
    """Norm, then each pair turned by its angle as a complex number."""
    x = x.detach().double()
    y = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w.detach().double()
    i = torch.arange(case["rot"] // 2, device=x.device)
    first = case["start"] + (2 * i if case["interleaved"] else i)
    second = first + (1 if case["interleaved"] else case["rot"] // 2)
    z = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.full_like(angle, amplitude), angle)[..., None, :]
    out = y.clone()
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_rotary(s, case):
    angle = s["positions"].double()[..., None] * s["frequencies"]
    out = []
    for x, w, g in (("q", "wq", "gq"), ("k", "wk", "gk")):
        dx, dw, y = [], 0, []
        for b in range(case["batch"]):                                  # the gradients by differentiating the formula
            xi = s[x][b].detach().double().requires_grad_(True)
            wi = s[w].detach().double().requires_grad_(True)
            r = xi / torch.sqrt((xi ** 2).sum(-1, keepdim=True) / xi.shape[-1] + EPS) * wi
            i = torch.arange(case["rot"] // 2, device="cuda")
            first = case["start"] + (2 * i if case["interleaved"] else i)
            second = first + (1 if case["interleaved"] else case["rot"] // 2)
            z = torch.complex(r[..., first], r[..., second]) * torch.polar(
                torch.full_like(angle[b], s["amplitude"]), angle[b])[:, None, :]
            o = r.index_copy(-1, first, z.real).index_copy(-1, second, z.imag)
            gx, gw = torch.autograd.grad(o, [xi, wi], s[g][b].double())
            y.append(o.detach())
            dx.append(gx)
            dw = dw + gw
        out.append((torch.stack(y), torch.stack(dx), dw))
    (oq, dq, dwq), (ok, dk, dwk) = out
    return [oq, ok, dq, dk, dwq, dwk]


def _exact_append(s, case):
    angle = s["positions"].double()[:, None] * s["frequencies"]
    k = _exact_rows(s["k"], s["wk"], angle, case, s["amplitude"])
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    m, page, table, lens = case["nodes"], case["page"], s["table"].tolist(), s["lens"].tolist()
    for i in range(case["seqs"]):
        for j in range(m):
            at = lens[i] - m + j
            kc[table[i][at // page], at % page] = k[i * m + j]
            vc[table[i][at // page], at % page] = s["v"][i * m + j].double()
    return [_exact_rows(s["q"], s["wq"], angle, case, s["amplitude"]), kc, vc]


def _exact_tree(s, case):
    m, hk, page = case["nodes"], case["hk"], case["page"]
    group, lens = case["hq"] // hk, s["lens"].tolist()
    par = None if s["parents"] is None else s["parents"].tolist()
    o = torch.empty(case["seqs"] * m, case["hq"], case["dim_v"], dtype=torch.float64, device="cuda")
    lse = torch.empty(case["seqs"] * m, case["hq"], dtype=torch.float64, device="cuda")
    for i in range(case["seqs"]):
        L = lens[i]
        ids = s["table"][i, : (L + page - 1) // page].long()
        k, v = (s[c][ids].flatten(0, 1)[:L].double() for c in ("k_cache", "v_cache"))
        mask = torch.zeros(m, L, dtype=torch.bool)
        mask[:, : L - m] = True
        for j in range(m):
            a = j
            while a >= 0:
                mask[j, L - m + a] = True
                a = a - 1 if par is None else par[i * m + a]
        mask = mask.cuda()
        for h in range(case["hq"]):
            t = (s["q"][i * m:(i + 1) * m, h].double() @ k[:, h // group].T) * case["dim"] ** -0.5
            t = t.masked_fill(~mask, -math.inf)
            lse[i * m:(i + 1) * m, h] = torch.logsumexp(t, 1)
            o[i * m:(i + 1) * m, h] = torch.softmax(t, 1) @ v[:, h // group]
    return [o, lse]


def exact(case, seed):
    if case["op"] not in ("rotary", "append", "tree"):
        return None                                                     # whole numbers and copied rows
    s = prepare(case, seed)
    with torch.enable_grad():
        return {"rotary": _exact_rotary, "append": _exact_append, "tree": _exact_tree}[case["op"]](s, case)
