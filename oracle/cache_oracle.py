"""Pages of a kv cache, one sequence and one page after another in plain Python
(test infrastructure; no reference counterpart).  State: ``refs`` (list),
``table`` (list of lists, -1 behind the pages), ``lens`` (list), ``pools``
(CPU tensors [num_pages, page_size, ...]); everything is changed in place."""


def pages_of(rows, page):
    return (rows + page - 1) // page if rows > 0 else 0


def free_pages(refs):
    return [i for i, r in enumerate(refs) if r <= 0]


def reserve(refs, table, lens, add, page):
    width, out, needs = len(table[0]) if table else 0, [], []
    for s, n in enumerate(add):
        need = pages_of(lens[s] + n, page) - pages_of(lens[s], page) if n >= 0 else -1
        if n < 0 or pages_of(lens[s] + n, page) > width or need > len(refs):
            need = -1
        elif n > 0 and lens[s] % page:
            pg = table[s][lens[s] // page]
            if not 0 <= pg < len(refs) or refs[pg] > 1:
                need = -1
        needs.append(need)
    free, asked = free_pages(refs), 0
    for s, need in enumerate(needs):
        ok = need >= 0 and (need == 0 or asked + need <= len(free))
        if ok:
            held = pages_of(lens[s], page)
            for j in range(need):
                table[s][held + j] = free[asked + j]
                refs[free[asked + j]] = 1
            lens[s] += add[s]
        asked += max(need, 0)
        out.append(int(ok))
    return out


def trim(refs, table, lens, keep, page):
    for s, n in enumerate(keep):
        if n < 0:
            continue
        lens[s] = min(lens[s], n)
        for c in range(pages_of(lens[s], page), len(table[s])):
            if 0 <= table[s][c] < len(refs):
                refs[table[s][c]] -= 1
            if table[s][c] >= 0:
                table[s][c] = -1


def fork(refs, table, lens, src, dst, pools):
    page = pools[0].shape[1]
    rows, before, old = [list(r) for r in table], list(lens), [p.clone() for p in pools]
    free, asked, out, named = free_pages(refs), 0, [], set()
    for s, d in zip(src, dst):
        ok = 0 <= s < len(lens) and 0 <= d < len(lens)
        first = d not in named
        named.add(d)
        if not ok or s == d or not first or before[d] != 0:
            out.append(0)
            continue
        whole, part = before[s] // page, before[s] % page
        pg = rows[s][whole] if part else -1
        if part and not 0 <= pg < len(refs):
            out.append(0)
            continue
        if part:
            asked += 1
            if asked > len(free):
                out.append(0)
                continue
        table[d] = [rows[s][c] if c < whole else -1 for c in range(len(rows[s]))]
        for c in range(whole):
            if 0 <= rows[s][c] < len(refs):
                refs[rows[s][c]] += 1
        if part:
            new = free[asked - 1]
            table[d][whole] = new
            refs[new] = 1
            for p, o in zip(pools, old):
                p[new] = o[pg]
        lens[d] = before[s]
        out.append(1)
    return out


def count(table, lens, page, num):
    """Entries of the table that hold each page."""
    out = [0] * num
    for row, length in zip(table, lens):
        for pg in row[:pages_of(length, page)]:
            if 0 <= pg < num:
                out[pg] += 1
    return out


def accept(pools, table, lens, accepted, drafted, refs=None):
    page, num = pools[0].shape[1], pools[0].shape[0]
    refs = count(table, lens, page, num) if refs is None else refs
    keep = []
    for s, row in enumerate(accepted):
        if not 0 <= drafted[s] <= lens[s]:
            keep.append(-1)
            continue
        prefix, last, taken = lens[s] - drafted[s], -1, []
        for a in row:
            if not last < a < drafted[s]:
                break
            taken.append(a)
            last = a
        moves = []
        for i, a in enumerate(taken):
            x, y = prefix + a, prefix + i
            if max(x, y) // page >= len(table[s]):
                continue
            px, py = table[s][x // page], table[s][y // page]
            if a != i and 0 <= px < num and 0 <= py < num:
                moves.append((px, x % page, py, y % page))
        if any(refs[py] > 1 for _, _, py, _ in moves):
            keep.append(-1)
            continue
        for px, x, py, y in moves:
            for p in pools:
                p[py, y] = p[px, x].clone()
        keep.append(prefix + len(taken))
    return keep


def compact(refs, table, pools):
    live = sum(r > 0 for r in refs)
    movers = [i for i in range(live, len(refs)) if refs[i] > 0]
    holes = [i for i in range(live) if refs[i] <= 0]
    to = dict(zip(movers, holes))
    for a, b in to.items():
        refs[b], refs[a] = refs[a], 0
        for p in pools:
            p[b] = p[a]
    for row in table:
        for c, pg in enumerate(row):
            row[c] = to.get(pg, pg)
    return live


def copy(pools, src, dst):
    num, old = pools[0].shape[0], [p.clone() for p in pools]
    inside = [0 <= s < num and 0 <= d < num for s, d in zip(src, dst)]
    first = {}
    for i, d in enumerate(dst):
        if inside[i]:
            first.setdefault(d, i)
    out = []
    for i, (s, d) in enumerate(zip(src, dst)):
        ok = inside[i] and first[d] == i and (s == d or s not in first)
        if ok:
            for p, o in zip(pools, old):
                p[d] = o[s]
        out.append(int(ok))
    return out
