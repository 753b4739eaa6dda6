"""Attention of drafted rows over a paged cache in 64 bits, row by row from the
definition (test infrastructure; no reference counterpart)."""
import math

import torch


def visible(table, length, rows, j, parents, page_size, num_pages):
    """Cache positions that drafted row j of a sequence sees, as (page, row) pairs."""
    prefix = length - rows
    nodes, a = {j}, j
    while True:
        up = a - 1 if parents is None else int(parents[a])
        if not 0 <= up < a:
            break
        nodes.add(up)
        a = up
    seen = list(range(min(prefix, length))) + sorted(prefix + i for i in nodes)
    out = []
    for t in seen:
        if 0 <= t < min(length, len(table) * page_size):
            pg = int(table[t // page_size])
            if 0 <= pg < num_pages:
                out.append((pg, t % page_size))
    return out


def tree_attention(q, k_cache, v_cache, block_table, cache_seqlens, parents=None, scale=None, cu_seqlens=None,
                   attn_sink=None):
    """(o, lse, size, reach): sum p |v| and the largest sum |q k| scale of each row, which bound the
    rounding of a computation in fewer bits."""
    total, hq, d = q.shape
    num_pages, page, hk, dv = v_cache.shape
    n, scale = block_table.shape[0], scale if scale is not None else 1 / math.sqrt(d)
    cu = list(range(n + 1)) if cu_seqlens is None else cu_seqlens.tolist()
    o, size = torch.zeros(total, hq, dv, dtype=torch.float64), torch.zeros(total, hq, dv, dtype=torch.float64)
    lse, reach = torch.full((total, hq), -math.inf, dtype=torch.float64), torch.zeros(total, hq, dtype=torch.float64)
    if attn_sink is not None:
        lse = attn_sink.double().expand(total, hq).clone()
    heads = torch.arange(hq) // (hq // hk)
    for s in range(n):
        rows = cu[s + 1] - cu[s]
        for j in range(rows):
            par = None if parents is None else parents[cu[s]:cu[s + 1]]
            seen = visible(block_table[s].tolist(), int(cache_seqlens[s]), rows, j, par, page, num_pages)
            if not seen:
                continue
            pg, row = (torch.tensor(x) for x in zip(*seen))
            k, v = (c[pg, row].double()[:, heads] for c in (k_cache, v_cache))          # [keys, hq, d]
            qr = q[cu[s] + j].double()
            sc = scale * torch.einsum("hd,khd->hk", qr, k)
            reach[cu[s] + j] = (scale * torch.einsum("hd,khd->hk", qr.abs(), k.abs())).amax(1)
            full = sc if attn_sink is None else torch.cat([sc, attn_sink.double()[:, None]], 1)
            lse[cu[s] + j] = torch.logsumexp(full, 1)
            p = torch.exp(sc - lse[cu[s] + j][:, None])
            o[cu[s] + j] = torch.einsum("hk,khd->hd", p, v)
            size[cu[s] + j] = torch.einsum("hk,khd->hd", p, v.abs())
    return o, lse, size, reach
