"""Forking, freeing, compacting and copying pages against a one-page-at-a-time oracle; all of it exact."""
from __future__ import annotations

import pytest
import torch

import page_oracle
from kernels.attention import int8_pool
from kernels.kv_cache import PageMoves, kv_compact, kv_copy_pages, kv_fork, kv_free

pytestmark = [pytest.mark.gpu]
DEV = "cuda"


def _pool(seed, B, bs, nb, max_len, width=None, bad=False):
    """Tables of B requests over a pool with random holes; some pages with two owners."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, max_len + 1, (B,), generator=g)
    pages = (lens + bs - 1) // bs
    width = width or int(pages.max()) + 2
    perm = torch.randperm(nb, generator=g)
    assert int(pages.sum()) <= nb
    table = torch.full((B, width), -1, dtype=torch.int64)
    counts = torch.zeros(nb, dtype=torch.int32)
    at = 0
    for b in range(B):
        n = int(pages[b])
        table[b, :n] = perm[at:at + n]
        at += n
    counts[perm[:at]] = torch.randint(1, 3, (at,), generator=g, dtype=torch.int32)
    if bad and B > 1:
        table[0, 0], table[1, min(1, width - 1)] = nb + 5, -9
    return table, lens.to(torch.int32), counts


FORKS = [(1, 16, 8, 40, 1), (4, 16, 200, 300, 9), (3, 1, 64, 20, 7), (8, 5, 500, 150, 40), (30, 16, 9000, 2000, 200),
         (7, 64, 70000, 3000, 1300), (2, 16, 5, 32, 6)]


@pytest.mark.parametrize("bad", [False, True])
@pytest.mark.parametrize("B,bs,nb,max_len,n", FORKS)
def test_fork(native, B, bs, nb, max_len, n, bad):
    table, lens, counts = _pool(B + n, B, bs, nb, max_len, bad=bad)
    parents = torch.randint(-1 if bad else 0, B + (1 if bad else 0), (n,), generator=torch.Generator().manual_seed(n), dtype=torch.int32)
    want = page_oracle.fork(table, lens, parents, counts, bs)
    t, rc = table.to(DEV), counts.to(DEV)
    child, moves = kv_fork(t, lens.to(DEV), parents.to(DEV), rc, bs)
    for got, exp in zip((child, moves.src, moves.dst, moves.rows, rc, t), (*want, table)):
        assert torch.equal(got.cpu(), exp)


def test_fork_runs_out_of_pages(native):
    bs, nb = 4, 6
    table = torch.tensor([[0, 1, 2]])
    for taken in range(nb - 3 + 1):
        counts = torch.ones(nb, dtype=torch.int32)
        counts[nb - taken:] = 0
        for length in (0, 1, 4, 5, 12, 11, 99, -3):
            lens, parents = torch.tensor([length], dtype=torch.int32), torch.zeros(5, dtype=torch.int32)
            want = page_oracle.fork(table, lens, parents, counts, bs)
            rc = counts.to(DEV)
            child, moves = kv_fork(table.to(DEV), lens.to(DEV), parents.to(DEV), rc, bs)
            for got, exp in zip((child, moves.src, moves.dst, moves.rows, rc), want):
                assert torch.equal(got.cpu(), exp)


def test_fork_groups_without_need(native):
    """More children than one group, the first 1500 of them ending on a page's border."""
    bs = 4
    table = torch.arange(6).view(2, 3)
    lens = torch.tensor([8, 7], dtype=torch.int32)
    counts = torch.zeros(3000, dtype=torch.int32)
    counts[:6] = 1
    parents = torch.cat([torch.zeros(1500, dtype=torch.int32), torch.ones(1100, dtype=torch.int32)])
    want = page_oracle.fork(table, lens, parents, counts, bs)
    rc = counts.to(DEV)
    child, moves = kv_fork(table.to(DEV), lens.to(DEV), parents.to(DEV), rc, bs)
    for got, exp in zip((child, moves.src, moves.dst, moves.rows, rc), want):
        assert torch.equal(got.cpu(), exp)


def test_fork_odd_alignment_and_types(native):
    """ref_counts that start off a 16-byte boundary, a strided table, 64-bit lengths and parents."""
    table, lens, counts = _pool(3, 6, 16, 700, 900, width=64)
    parents = torch.tensor([0, 5, 5, 2, 1])
    want = page_oracle.fork(table, lens, parents, counts, 16)
    rc = torch.empty(701, dtype=torch.int32, device=DEV)[1:]
    rc.copy_(counts)
    wide = torch.full((6, 100), -1, dtype=torch.int64, device=DEV)
    wide[:, 10:74] = table.to(DEV)
    child, moves = kv_fork(wide[:, 10:74], lens.long().to(DEV), parents.to(DEV), rc, 16)
    for got, exp in zip((child, moves.src, moves.dst, moves.rows, rc), want):
        assert torch.equal(got.cpu(), exp)


@pytest.mark.parametrize("B,nb,width", [(1, 4, 1), (12, 900, 50), (5, 3000, 700)])
def test_free(native, B, nb, width):
    g = torch.Generator().manual_seed(B)
    table = torch.randint(-2, nb + 2, (B, width), generator=g)  # stray entries and shared pages
    counts = torch.randint(0, 5, (nb,), generator=g, dtype=torch.int32)
    rows = torch.randint(-1, B + 1, (B + 2,), generator=g, dtype=torch.int32)
    rows[-1] = rows[0]  # the same row twice
    want_t, want_c = page_oracle.free(table, rows, counts)
    t, rc = table.to(DEV), counts.to(DEV)
    kv_free(t, rows.to(DEV), rc)
    assert torch.equal(t.cpu(), want_t) and torch.equal(rc.cpu(), want_c)
    kv_free(t, rows.to(DEV), rc)  # and once more
    assert torch.equal(t.cpu(), want_t) and torch.equal(rc.cpu(), want_c)


@pytest.mark.parametrize("nb", [1, 2, 17, 4095, 4096, 4097, 50000, 300001])
@pytest.mark.parametrize("free", [0.0, 0.03, 0.5, 0.97, 1.0])
def test_compact(native, nb, free):
    g = torch.Generator().manual_seed(nb)
    counts = torch.randint(1, 4, (nb,), generator=g, dtype=torch.int32)
    counts[torch.rand(nb, generator=g) < free] = 0
    table = torch.randint(-2, nb + 2, (7, 301), generator=g)
    page_map, new_table, new_counts, moving, holes = page_oracle.compact(table, counts)
    t, rc = table.to(DEV), counts.to(DEV)
    got_map, moves = kv_compact(t, rc)
    m = int(moves.count)
    assert m == len(moving)
    assert moves.src[:m].tolist() == moving and moves.dst[:m].tolist() == holes
    assert torch.equal(got_map.cpu(), page_map) and torch.equal(t.cpu(), new_table) and torch.equal(rc.cpu(), new_counts)


def test_compact_without_table(native):
    counts = torch.tensor([0, 2, 0, 1, 0, 0, 3], dtype=torch.int32, device=DEV)
    page_map, moves = kv_compact(torch.empty(0, 0, dtype=torch.int64, device=DEV), counts)
    assert page_map.tolist() == [-1, 1, -1, 2, -1, -1, 0] and counts.tolist() == [3, 2, 1, 0, 0, 0, 0]
    assert moves.src[:int(moves.count)].tolist() == [6, 3] and moves.dst[:2].tolist() == [0, 2]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H,bs,D", [(2, 16, 128), (1, 1, 8), (3, 5, 20), (4, 64, 256), (2, 7, 3), (1, 300, 64)])
@pytest.mark.parametrize("layers", [1, 3])
def test_copy(native, H, bs, D, dtype, layers):
    nb = 12
    g = torch.Generator().manual_seed(D)
    ks = [torch.randn(nb, H, bs, D, generator=g).to(dtype) for _ in range(layers)]
    vs = [torch.randn(nb, H, bs, D, generator=g).to(dtype) for _ in range(layers)]
    src = torch.tensor([0, 1, -1, 2, 5, nb, 3, 0])
    dst = torch.tensor([4, 6, 7, -1, 5, 8, 10, 11])
    rows = torch.tensor([bs, 0, bs, bs, bs, bs, max(1, bs // 2), bs + 9], dtype=torch.int32)
    for r in (None, rows):
        gk, gv = [t.to(DEV) for t in ks], [t.to(DEV) for t in vs]
        args = (gk[0], gv[0]) if layers == 1 else (gk, gv)
        kv_copy_pages(*args, PageMoves(src.to(DEV), dst.to(DEV), None if r is None else r.to(DEV)))
        for got, was in zip(gk + gv, ks + vs):
            assert torch.equal(got.cpu(), page_oracle.copy(was, src, dst, r))
    # only the first pairs count; a strided pool (the heads of a larger one); a base off the 16-byte grid
    count = torch.tensor([1], dtype=torch.int32, device=DEV)
    wide = torch.zeros(nb, 2 * H, bs, D, dtype=dtype, device=DEV)
    k2, v2 = wide[:, :H], wide[:, H:]
    k2.copy_(ks[0]); v2.copy_(vs[0])
    kv_copy_pages(k2, v2, PageMoves(src.to(DEV), dst.to(DEV), None, count))
    assert torch.equal(k2.cpu(), page_oracle.copy(ks[0], src[:1], dst[:1])) and torch.equal(v2.cpu(), page_oracle.copy(vs[0], src[:1], dst[:1]))
    flat = torch.zeros(2 * ks[0].numel() + 1, dtype=dtype, device=DEV)
    k3, v3 = flat[1:1 + ks[0].numel()].view(ks[0].shape), flat[1 + ks[0].numel():].view(ks[0].shape)
    k3.copy_(ks[0]); v3.copy_(vs[0])
    kv_copy_pages(k3, v3, PageMoves(src.to(DEV), dst.to(DEV), rows.to(DEV)))
    assert torch.equal(k3.cpu(), page_oracle.copy(ks[0], src, dst, rows)) and torch.equal(v3.cpu(), page_oracle.copy(vs[0], src, dst, rows))


def test_copy_positions_apart(native):
    """Pool views whose positions are not next to one another."""
    base = torch.randn(6, 2, 8, 2, 32, device=DEV)
    k, v = base[:, :, :, 0], base[:, :, :, 1]
    was_k, was_v = k.cpu().clone(), v.cpu().clone()
    src, dst, rows = torch.tensor([0, 1]), torch.tensor([3, 5]), torch.tensor([8, 3], dtype=torch.int32)
    kv_copy_pages(k, v, PageMoves(src.to(DEV), dst.to(DEV), rows.to(DEV)))
    assert torch.equal(k.cpu(), page_oracle.copy(was_k, src, dst, rows)) and torch.equal(v.cpu(), page_oracle.copy(was_v, src, dst, rows))


@pytest.mark.parametrize("D", [128, 33])
def test_copy_int8(native, D):
    nb, H, bs = 9, 3, 16
    kc, vc, ks, vs = int8_pool(nb, H, bs, D, DEV)
    kc.random_(-127, 128); vc.random_(-127, 128); ks.uniform_(); vs.uniform_()
    was = [t.cpu().clone() for t in (kc, vc, ks, vs)]
    src, dst, rows = torch.tensor([0, 2]), torch.tensor([7, 4]), torch.tensor([16, 5], dtype=torch.int32)
    kv_copy_pages(kc, vc, PageMoves(src.to(DEV), dst.to(DEV), rows.to(DEV)), k_scales=ks, v_scales=vs)
    for got, w in zip((kc, vc), was):
        assert torch.equal(got.cpu(), page_oracle.copy(w, src, dst, rows))
    for got, w in zip((ks, vs), was[2:]):
        assert torch.equal(got.cpu(), page_oracle.copy(w[..., None], src, dst, rows)[..., 0])


def test_copy_many_layers(native):
    """More layers than one launch takes."""
    ks = [torch.randn(3, 1, 4, 8, device=DEV) for _ in range(70)]
    vs = [torch.randn(3, 1, 4, 8, device=DEV) for _ in range(70)]
    kv_copy_pages(ks, vs, PageMoves(torch.tensor([0], device=DEV), torch.tensor([2], device=DEV)))
    assert all(torch.equal(t[0], t[2]) for t in ks + vs)


def test_copy_far_offsets(native):
    """Element offsets beyond 2^32: pages at both ends of a 9 GB cache."""
    nb, H, bs, D = 1 << 19, 1, 64, 130
    k = torch.zeros(nb, H, bs, D, dtype=torch.bfloat16, device=DEV)
    v = torch.zeros_like(k)
    assert k.numel() > 1 << 32
    k[nb - 1] = torch.randn(H, bs, D, device=DEV).to(torch.bfloat16); v[nb - 1] = 1.5
    k[nb - 2] = 3.0
    src = torch.tensor([nb - 1, nb - 2], device=DEV)
    dst = torch.tensor([0, nb - 5], device=DEV)
    kv_copy_pages(k, v, PageMoves(src, dst))
    assert torch.equal(k[0], k[nb - 1]) and torch.equal(v[0], v[nb - 1]) and bool((k[nb - 5] == 3.0).all())
    assert not k[1:1000].any() and not k[nb - 4:nb - 2].any()


def test_refusals(native):
    t = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    lens, parents = torch.ones(2, dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    rc = torch.ones(8, dtype=torch.int32, device=DEV)
    k = torch.zeros(8, 2, 4, 8, dtype=torch.bfloat16, device=DEV)
    one = torch.zeros(1, dtype=torch.int64, device=DEV)
    for bad in (lambda: kv_fork(t.int(), lens, parents, rc, 4), lambda: kv_fork(t, lens[:1], parents, rc, 4),
                lambda: kv_fork(t, lens, parents.float(), rc, 4), lambda: kv_fork(t, lens, parents, rc.long(), 4),
                lambda: kv_fork(t, lens, parents, rc, 0), lambda: kv_fork(t, lens, parents, rc[:0], 4),
                lambda: kv_fork(t, lens, parents, rc[::2], 4), lambda: kv_fork(t.t().contiguous().t(), lens, parents, rc, 4),
                lambda: kv_free(t[:1].expand(2, 3), parents, rc), lambda: kv_free(t, parents, rc, backend="mps"),
                lambda: kv_compact(t[0], rc), lambda: kv_compact(t, rc.view(2, 4)),
                lambda: kv_copy_pages([k], [k, k], PageMoves(one, one)), lambda: kv_copy_pages([], [], PageMoves(one, one)),
                lambda: kv_copy_pages(k, k[:, :1], PageMoves(one, one)), lambda: kv_copy_pages(k, k.clone(), PageMoves(one.int(), one)),
                lambda: kv_copy_pages([k, k.float()], [k, k], PageMoves(one, one)),
                lambda: kv_copy_pages(k, k.clone(), PageMoves(one, one, parents)),
                lambda: kv_copy_pages(k, k.clone(), PageMoves(one, one, None, one)),
                lambda: kv_copy_pages(k.to(torch.int8), k.to(torch.int8), PageMoves(one, one)),
                lambda: kv_copy_pages(k.double(), k.double(), PageMoves(one, one))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: kv_fork(t.cpu(), lens, parents, rc, 4), lambda: kv_copy_pages(k, k.clone(), PageMoves(one.cpu(), one))):
        with pytest.raises(RuntimeError):
            bad()
    # nothing to do
    kv_copy_pages(k, k.clone(), PageMoves(one[:0], one[:0]))
    kv_free(t, parents[:0], rc)
    child, moves = kv_fork(t, lens, parents[:0], rc, 4)
    assert child.shape == (0, 3) and moves.src.shape == (0,)


def test_streams_and_graph(native):
    """Fork, copy and free on a side stream, then captured and replayed on other contents."""
    table, lens, counts = _pool(11, 6, 16, 300, 400)
    parents = torch.randint(0, 6, (20,), generator=torch.Generator().manual_seed(0), dtype=torch.int32)
    k = torch.randn(300, 2, 16, 64).to(torch.bfloat16)
    gt, gl, gp, rc = table.to(DEV), lens.to(DEV), parents.to(DEV), counts.to(DEV)
    gk, gv = k.to(DEV), (2 * k).to(DEV)
    rows = torch.arange(6, dtype=torch.int32, device=DEV)

    def step():
        child, moves = kv_fork(gt, gl, gp, rc, 16)
        kv_copy_pages(gk, gv, moves)
        kv_free(gt, rows, rc)
        return child, moves

    def reset(tbl, cnt):
        gt.copy_(tbl); rc.copy_(cnt); gk.copy_(k); gv.copy_(2 * k)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        child, moves = step()
    for seed in (12, 13):
        t2, l2, c2 = _pool(seed, 6, 16, 300, 400, width=table.shape[1])
        reset(t2, c2); gl.copy_(l2)
        graph.replay()
        torch.cuda.synchronize()
        wc, ws, wd, wr, wn = page_oracle.fork(t2, l2, parents, c2, 16)
        wt, wn = page_oracle.free(t2, rows.cpu(), wn)
        assert torch.equal(child.cpu(), wc) and torch.equal(gt.cpu(), wt) and torch.equal(rc.cpu(), wn)
        assert torch.equal(gk.cpu(), page_oracle.copy(k, ws, wd, wr)) and torch.equal(gv.cpu(), page_oracle.copy(2 * k, ws, wd, wr))
