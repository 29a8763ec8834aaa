"""The serving-step operators at the ends of their ranges and side by side: the largest vocabulary, very many small
rows, more tokens than one grid dimension of small blocks, 64-bit indexes out of range, and two calls at once on
two streams."""
from __future__ import annotations

import pytest
import torch

import page_oracle
import sample_oracle
from kernels.attention import qk_norm_rope_append
from kernels.kv_cache import PageMoves, kv_compact, kv_copy_pages, kv_fork, kv_free
from kernels.rope import qk_norm_rope
from kernels.softmax import sample_tokens

pytestmark = [pytest.mark.gpu]
DEV = "cuda"


def test_largest_vocabulary(native):
    V = 1 << 24
    g = torch.Generator().manual_seed(0)
    x = (3 * torch.randn(1, V, generator=g)).to(torch.float16)
    u = torch.tensor([0.37])
    gx, gu = x.to(DEV), u.to(DEV)
    for kw in (dict(top_k=50, top_p=0.9), dict(top_p=0.5), dict(temperature=0.0)):
        assert sample_tokens(gx, gu, **kw).tolist() == sample_oracle.tokens(x, u, **kw)
    with pytest.raises(ValueError, match="2\\^24"):
        sample_tokens(torch.zeros(1, V + 1, dtype=torch.float16, device=DEV), gu)


def test_many_small_rows(native):
    B, V = 30000, 5
    g = torch.Generator().manual_seed(1)
    x, u = torch.randn(B, V, generator=g), torch.rand(B, generator=g)
    kw = dict(temperature=0.7, top_k=3, top_p=0.9)
    assert sample_tokens(x.to(DEV), u.to(DEV), **kw).tolist() == sample_oracle.tokens(x, u, **kw)


def test_settings_of_other_types(native):
    B, V = 6, 500
    g = torch.Generator().manual_seed(2)
    x, u = torch.randn(B, V, generator=g), torch.rand(B, generator=g)
    k = torch.tensor([0, 3, 1 << 40, -(1 << 40), 10, 499])  # far outside 32 bits: all, and off
    t = torch.tensor([1.0, 0.5, 2.0, 1.0, 0.0, 1.0], dtype=torch.float64)
    want = sample_oracle.tokens(x, u, temperature=t, top_k=k.clamp(-1, V))
    assert sample_tokens(x.to(DEV), u.double().to(DEV), temperature=t.to(DEV), top_k=k.to(DEV)).tolist() == want


def test_indexes_outside_32_bits(native):
    table = torch.arange(6).view(2, 3).to(DEV)
    counts = torch.ones(9, dtype=torch.int32, device=DEV)
    far = torch.tensor([1 << 32, 1, -(1 << 33)], device=DEV)  # would wrap to 0
    child, moves = kv_fork(table, torch.tensor([4, 8], device=DEV), far, counts, 4)
    assert child.tolist() == [[-1] * 3, [3, 4, -1], [-1] * 3]
    kv_free(table, torch.tensor([1 << 32], device=DEV), counts)
    assert table[0].tolist() == [0, 1, 2]
    q = torch.randn(2, 1, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    cos = torch.ones(4, 64, device=DEV)
    out, _ = qk_norm_rope(q, q, w, w, cos, torch.zeros_like(cos), positions=torch.tensor([1 << 32, 2], device=DEV))
    assert not out[0].any() and out[1].any()


def test_many_tokens(native):
    """300001 tokens of one head: the same values as the tokens give in pieces."""
    n, D = 300001, 64
    g = torch.Generator(device=DEV).manual_seed(3)
    q = torch.randn(n, 1, D, generator=g, device=DEV).to(torch.bfloat16)
    k = torch.randn(n, 1, D, generator=g, device=DEV).to(torch.bfloat16)
    w = torch.rand(D, generator=g, device=DEV).to(torch.bfloat16)
    ang = torch.rand(1000, D // 2, generator=g, device=DEV)
    cos, sin = torch.cat([ang.cos()] * 2, 1), torch.cat([ang.sin()] * 2, 1)
    pos = torch.randint(0, 1000, (n,), generator=g, device=DEV, dtype=torch.int32)
    a, b = qk_norm_rope(q, k, w, w, cos, sin, positions=pos)
    for lo, hi in ((0, 1), (1, 40), (150000, 150321), (n - 5, n)):
        c, d = qk_norm_rope(q[lo:hi], k[lo:hi], w, w, cos, sin, positions=pos[lo:hi])
        assert torch.equal(a[lo:hi], c) and torch.equal(b[lo:hi], d)


def test_two_streams_at_once(native):
    """The same calls on two streams over inputs of their own, interleaved without a wait, give what they give alone."""
    def work(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        logits = 4 * torch.randn(40, 30000, generator=g, device=DEV)
        u = torch.rand(40, generator=g, device=DEV)
        q = torch.randn(200, 8, 128, generator=g, device=DEV).to(torch.bfloat16)
        k, v = (torch.randn(200, 2, 128, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
        w = torch.rand(128, generator=g, device=DEV).to(torch.bfloat16)
        cos = torch.rand(200, 128, generator=g, device=DEV)
        kc, vc = (torch.randn(400, 2, 16, 128, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
        slots = torch.randperm(800, generator=g, device=DEV)[:200]
        pos = torch.arange(200, device=DEV, dtype=torch.int32)
        counts = torch.randint(0, 2, (400,), generator=g, device=DEV, dtype=torch.int32)
        table = torch.randint(0, 400, (12, 20), generator=g, device=DEV)
        counts[table.flatten()] = 1
        counts[:50] = 0
        lens = torch.randint(1, 320, (12,), generator=g, device=DEV, dtype=torch.int32)
        parents = torch.randint(0, 12, (30,), generator=g, device=DEV, dtype=torch.int32)

        def run():
            rc, t, a, b = counts.clone(), table.clone(), kc.clone(), vc.clone()
            out = [sample_tokens(logits, u, top_p=0.9), sample_tokens(logits, u, top_k=40),
                   qk_norm_rope_append(q, k, v, a, b, slots, pos, cos, cos, w, w)]
            child, moves = kv_fork(t, lens, parents, rc, 16)
            kv_copy_pages(a, b, moves)
            kv_free(t, parents[:3], rc)
            page_map, moves2 = kv_compact(child, rc)
            return out + [child, moves.src, moves.dst, t, rc, page_map, a, b]
        return run

    runs = [work(s) for s in (1, 2)]
    want = [[t.clone() for t in r()] for r in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    got = [[], []]
    for _ in range(20):
        for i, (r, s) in enumerate(zip(runs, streams)):
            with torch.cuda.stream(s):
                got[i].append(r())
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(x, y) for x, y in zip(out, want[i]))


def test_fork_of_a_page_that_two_children_copy(native):
    """One part-filled page copied to several children in one call, the parent left as it was."""
    bs, nb = 16, 12
    k = torch.randn(nb, 2, bs, 32, device=DEV)
    v = torch.randn_like(k)
    table = torch.tensor([[3, 5]], device=DEV)
    counts = torch.zeros(nb, dtype=torch.int32, device=DEV)
    counts[[3, 5]] = 1
    was = k.cpu().clone()
    child, moves = kv_fork(table, torch.tensor([21], device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV), counts, bs)
    kv_copy_pages(k, v, moves)
    assert child.tolist() == [[3, 0], [3, 1], [3, 2]] and counts[:6].tolist() == [1, 1, 1, 4, 0, 1]
    assert torch.equal(k.cpu(), page_oracle.copy(was, [5, 5, 5], [0, 1, 2], [5, 5, 5]))
    # and a PageMoves of one's own, pairs outside the pool left out
    kv_copy_pages(k, v, PageMoves(torch.tensor([1 << 40, 3], device=DEV), torch.tensor([7, 8], device=DEV)))
    assert torch.equal(k[8], k[3]) and torch.equal(k[7].cpu(), was[7])


def test_fork_from_pages_that_nobody_holds(native):
    """A table over pages whose counts are 0: sources are not handed out, so that the copies of one fork never meet."""
    g = torch.Generator().manual_seed(5)
    for n in (7, 1500):
        counts = torch.zeros(4000, dtype=torch.int32)
        table = torch.randint(0, 60, (9, 12), generator=g)
        lens = torch.randint(0, 12 * 16, (9,), generator=g, dtype=torch.int32)
        parents = torch.randint(0, 9, (n,), generator=g, dtype=torch.int32)
        want = page_oracle.fork(table, lens, parents, counts, 16)
        rc = counts.to(DEV)
        child, moves = kv_fork(table.to(DEV), lens.to(DEV), parents.to(DEV), rc, 16)
        for got, exp in zip((child, moves.src, moves.dst, moves.rows, rc), want):
            assert torch.equal(got.cpu(), exp)
        assert not set(moves.src.tolist()) & set(moves.dst.tolist()) - {-1}
