"""What a fork promises where every page that a row names within its length is counted: none of them is handed out."""
from __future__ import annotations

import pytest
import torch

import page_oracle
from kernels.kv_cache import kv_copy_pages, kv_fork

pytestmark = [pytest.mark.gpu]
DEV = "cuda"


@pytest.mark.parametrize("B,width,bs,n,nb", [(1, 3, 4, 5, 12), (9, 12, 16, 40, 500), (6, 40, 8, 700, 4000), (9, 300, 16, 1500, 20000)])
def test_no_page_of_a_row_is_handed_out(native, B, width, bs, n, nb):
    g = torch.Generator().manual_seed(n)
    table = torch.randint(0, nb // 3, (B, width), generator=g)  # rows share pages with one another
    lens = torch.randint(0, width * bs + 1, (B,), generator=g, dtype=torch.int32)
    parents = torch.randint(0, B, (n,), generator=g, dtype=torch.int32)
    counts = torch.zeros(nb, dtype=torch.int32)
    named = set()
    for b in range(B):
        named |= set(table[b, :(int(lens[b]) + bs - 1) // bs].tolist())
    counts[list(named)] = 1
    want = page_oracle.fork(table, lens, parents, counts, bs)
    rc = counts.to(DEV)
    child, moves = kv_fork(table.to(DEV), lens.to(DEV), parents.to(DEV), rc, bs)
    for got, exp in zip((child, moves.src, moves.dst, moves.rows, rc), want):
        assert torch.equal(got.cpu(), exp)
    taken = [p for p in moves.dst.tolist() if p >= 0]
    assert len(set(taken)) == len(taken) and not set(taken) & named
    # the keys that the children see are their parents'
    k = torch.arange(nb * bs, dtype=torch.float32, device=DEV).view(nb, 1, bs, 1).expand(nb, 1, bs, 4).contiguous()
    v, was = k.clone(), k.cpu()
    kv_copy_pages(k, v, moves)
    now, rows = k.cpu()[:, 0, :, 0], child.cpu()
    for i in list(range(min(n, 60))) + [n - 1]:
        p, length = int(parents[i]), int(lens[int(parents[i])])
        if int(moves.src[i]) >= 0 and int(moves.dst[i]) < 0:
            continue  # no page was left
        pages = (length + bs - 1) // bs
        assert torch.equal(now[rows[i, :pages]].reshape(-1)[:length], was[table[p, :pages], 0, :, 0].reshape(-1)[:length])
