"""Page bookkeeping one page at a time on the host: what kv_fork, kv_free, kv_compact and kv_copy_pages are
checked against. Plain Python on CPU tensors; everything is exact."""
from __future__ import annotations

import torch


def fork(table, lens, parents, counts, bs):
    table, lens, parents, rc = table.tolist(), lens.tolist(), parents.tolist(), counts.tolist()
    width = len(table[0]) if table else 0
    nb = len(rc)
    for p in parents:  # what is copied from counts as held
        if 0 <= p < len(table):
            full, rest = divmod(min(max(lens[p], 0), width * bs), bs)
            if rest and 0 <= table[p][full] < nb:
                rc[table[p][full]] = max(rc[table[p][full]], 1)
    free = iter([p for p in range(nb) if rc[p] == 0])
    child, src, dst, rows, shared = [], [], [], [], []
    for p in parents:
        row, s, d, r = [-1] * width, -1, -1, 0
        if 0 <= p < len(table):
            n = min(max(lens[p], 0), width * bs)
            full, rest = divmod(n, bs)
            row = table[p][:full] + [-1] * (width - full)
            ok = True
            if rest:
                page = table[p][full]
                if 0 <= page < nb:
                    s, r = page, rest
                    d = next(free, -1)
                    ok = d >= 0
                    row[full] = d
                else:
                    row[full] = page
            if ok:
                if d >= 0:
                    rc[d] = 1
                shared += [page for page in table[p][:full] if 0 <= page < nb]
            else:
                row = [-1] * width
        child.append(row); src.append(s); dst.append(d); rows.append(r)
    for page in shared:  # on top of what was handed out
        rc[page] += 1
    return (torch.tensor(child, dtype=torch.int64).reshape(len(parents), width), torch.tensor(src, dtype=torch.int64),
            torch.tensor(dst, dtype=torch.int64), torch.tensor(rows, dtype=torch.int32), torch.tensor(rc, dtype=torch.int32))


def free(table, rows, counts):
    table, rc = table.clone(), counts.tolist()
    for r in rows.tolist():
        if not 0 <= r < table.shape[0]:
            continue
        for page in table[r].tolist():
            if 0 <= page < len(rc):
                rc[page] = max(0, rc[page] - 1)
        table[r] = -1
    return table, torch.tensor(rc, dtype=torch.int32)


def compact(table, counts):
    rc = counts.tolist()
    nb = len(rc)
    live = sum(c > 0 for c in rc)
    page_map = [p if c > 0 else -1 for p, c in enumerate(rc)]
    moving = [p for p in reversed(range(live, nb)) if rc[p] > 0]
    holes = [p for p in range(live) if rc[p] == 0]
    assert len(moving) == len(holes)
    for s, d in zip(moving, holes):
        page_map[s], rc[d], rc[s] = d, rc[s], 0
    remap = lambda e: page_map[e] if 0 <= e < nb else e  # noqa: E731
    new = [[remap(e) for e in row] for row in table.tolist()]
    return (torch.tensor(page_map, dtype=torch.int64), torch.tensor(new, dtype=torch.int64).reshape(table.shape),
            torch.tensor(rc, dtype=torch.int32), moving, holes)


def copy(cache, src, dst, rows=None):
    out = cache.clone()
    nb, bs = cache.shape[0], cache.shape[2]
    for i, (s, d) in enumerate(zip(list(src), list(dst))):
        if 0 <= s < nb and 0 <= d < nb:
            n = bs if rows is None else min(max(int(rows[i]), 0), bs)
            out[d, :, :n] = cache[s, :, :n]
    return out
