"""Steps launched without a gap on one workspace. A decode step's plan is made in the workspace that the attention of
the step before may still be reading; with one batch the arrival counts of split pairs are at stake, with two batches
in turn the plan itself. Every step has to give, bit for bit, what it gives alone."""
from __future__ import annotations

import pytest
import torch

from kernels.attention import PagedAttentionCall, PagedWorkspace, int8_pool, paged_attention, paged_decode_step, qk_norm_rope_append
from kernels.kv_cache import kv_compact, kv_copy_pages, kv_fork, kv_free
from kernels.rope import build_rope_tables
from kernels.softmax import online_softmax, sample_tokens

pytestmark = [pytest.mark.gpu]
DEV = "cuda"
BS = 32


class _Batch:
    """One decode batch over a pool of its own: `lens` keys a request, the last of them this step's token."""

    def __init__(self, seed, lens, Hq, Hkv, D, dtype, int8, index=torch.int32):
        g = torch.Generator(device=DEV).manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
        B = len(lens)
        self.lens = torch.tensor(lens, dtype=index, device=DEV)
        pages = (max(lens) + BS - 1) // BS
        nb = B * pages + 3
        self.table = torch.randperm(nb, generator=g, device=DEV)[:B * pages].view(B, pages)
        self.pos = self.lens - 1
        self.slots = (self.table.gather(1, (self.pos // BS).long()[:, None])[:, 0] * BS + self.pos % BS).to(torch.int64)
        if index != torch.int32:
            self.slots = self.slots.to(torch.int32)  # widened by the call
        self.q, self.k, self.v = (rnd(B, h, D).to(dtype) for h in (Hq, Hkv, Hkv))
        self.wq, self.wk = ((1 + 0.2 * rnd(D)).to(dtype) for _ in range(2))
        self.cos, self.sin = build_rope_tables(max(lens), D, dtype=torch.float32, device=DEV)
        self.scales = {}
        if int8:
            self.kc, self.vc, ks, vs = int8_pool(nb, Hkv, BS, D, DEV)
            self.kc.random_(-127, 128, generator=g); self.vc.random_(-127, 128, generator=g)
            ks.uniform_(0.01, 0.02, generator=g); vs.uniform_(0.01, 0.02, generator=g)
            self.scales = dict(k_scales=ks, v_scales=vs)
        else:
            self.kc, self.vc = (rnd(nb, Hkv, BS, D).to(dtype) for _ in range(2))

    def step(self, ws, out=None):
        return paged_decode_step(self.q, self.k, self.v, self.kc, self.vc, self.table, self.lens, self.slots, self.pos, self.cos,
                                 self.sin, workspace=ws, out=out, q_norm_weight=self.wq, k_norm_weight=self.wk, **self.scales)

    def attend(self, ws, out=None):
        return paged_attention(self.q, self.kc, self.vc, self.table, self.lens, workspace=ws, out=out, max_q_len=1, **self.scales)


def _lens(seed, n, most):
    return (torch.randint(most // 8, most + 1, (n,), generator=torch.Generator().manual_seed(seed))).tolist()


def _batches(D, dtype, int8, index=torch.int32):
    """Many requests of ragged lengths, and a few with other heads and lengths: other items, rows and tables."""
    return (_Batch(1, _lens(1, 32, 3000), 32, 4, D, dtype, int8, index), _Batch(2, _lens(2, 5, 9000) + [1, 70], 16, 2, D, dtype, int8, index))


def _run(batches, order, call, ws):
    """The calls of `order` in one graph, replayed twice without a gap, and eagerly, against each call alone."""
    want = []
    for b in batches:
        call(b, ws, None)  # sizes the workspace
    for b in batches:
        torch.cuda.synchronize()
        want.append(call(b, PagedWorkspace(DEV), None).clone())
        torch.cuda.synchronize()
    outs = [torch.full_like(want[i], float("nan")) for i in order]
    for i, o in zip(order, outs):
        call(batches[i], ws, o)
    torch.cuda.synchronize()
    for i, o in zip(order, outs):
        assert torch.equal(o, want[i])
        o.fill_(float("nan"))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i, o in zip(order, outs):
            call(batches[i], ws, o)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    for i, o in zip(order, outs):
        assert torch.equal(o, want[i])
    assert ws.status() == 0


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.bfloat16), (128, torch.float16)])
def test_steps_with_norm_of_two_batches_in_turn(native, D, dtype, int8):
    _run(_batches(D, dtype, int8), [0, 1, 0, 1, 1, 0, 0, 1] * 2, lambda b, ws, o: b.step(ws, o), PagedWorkspace(DEV))


def test_steps_of_one_batch(native):
    """The same batch again and again: pairs that are cut over several CTAs are counted in the workspace."""
    _run(_batches(128, torch.bfloat16, False)[:1], [0] * 24, lambda b, ws, o: b.step(ws, o), PagedWorkspace(DEV))


def test_steps_with_arguments_that_are_cast(native):
    """64-bit positions and lengths and 32-bit slots: the calls make temporaries, whose memory the next call may get."""
    _run(_batches(128, torch.bfloat16, False, torch.int64), [0, 1] * 6, lambda b, ws, o: b.step(None, o) if o is not None else b.step(ws), PagedWorkspace(DEV))


def test_steps_on_the_built_in_scratch(native):
    """The same with the scratch that is part of the library in place of a workspace: every call plans there afresh."""
    batches = _batches(128, torch.bfloat16, False)

    def call(b, ws, o):
        q = qk_norm_rope_append(b.q, b.k, b.v, b.kc, b.vc, b.slots, b.pos, b.cos, b.sin, b.wq, b.wk)
        return PagedAttentionCall(q, b.kc, b.vc, b.table, b.lens, out=o, max_q_len=1).run_static()

    _run(batches, [0, 1, 0, 1, 1, 0, 0, 1], call, PagedWorkspace(DEV))


@pytest.mark.parametrize("between", ["sample", "pages", "softmax", "nothing"])
def test_other_operators_between_two_plans(native, between):
    """Attention, an operator of the serving step on data of its own, and the next attention's plan."""
    batches = _batches(128, torch.bfloat16, False)
    logits, u = torch.randn(3, 500, device=DEV), torch.rand(3, device=DEV)
    table = torch.arange(6, device=DEV).view(2, 3)
    lens, parents = torch.tensor([9, 5], dtype=torch.int32, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    counts = torch.ones(12, dtype=torch.int32, device=DEV)
    counts[6:] = 0
    kc, vc = (torch.randn(12, 1, 4, 64, device=DEV) for _ in range(2))

    def call(b, ws, o):
        o = b.attend(ws, o)
        if between == "sample":
            sample_tokens(logits, u, top_k=5)
        elif between == "softmax":
            online_softmax(logits)
        elif between == "pages":
            rc = counts.clone()
            child, moves = kv_fork(table, lens, parents, rc, 4)
            kv_copy_pages(kc, vc, moves)
            kv_free(child, parents, rc)
            kv_compact(child, rc)
        return o

    _run(batches, [0, 1, 0, 0, 1, 1, 0, 1], call, PagedWorkspace(DEV))


def test_lengths_that_a_fork_has_written(native):
    """The filled positions of the forked pages as context lengths, right behind the fork: attention over the children's
    own pages alone."""
    g = torch.Generator(device=DEV).manual_seed(4)
    B, Hq, Hkv, D, nb = 40, 16, 2, 128, 400
    kc, vc = (torch.randn(nb, Hkv, BS, D, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    q = torch.randn(B, Hq, D, generator=g, device=DEV).to(torch.bfloat16)
    table = torch.randperm(nb // 2, generator=g, device=DEV)[:6 * 8].view(6, 8)
    lens = torch.randint(1, 8 * BS, (6,), generator=g, device=DEV, dtype=torch.int32)
    parents = torch.arange(B, device=DEV, dtype=torch.int32) % 6
    counts = torch.zeros(nb, dtype=torch.int32, device=DEV)
    counts[table.flatten()] = 1
    ws = PagedWorkspace(DEV)

    def run():
        rc = counts.clone()
        child, moves = kv_fork(table, lens, parents, rc, BS)
        kv_copy_pages(kc, vc, moves)
        return moves, paged_attention(q, kc, vc, moves.dst[:, None], moves.rows, workspace=ws, max_q_len=1)

    def fork_only():
        moves = kv_fork(table, lens, parents, counts.clone(), BS)[1]
        return moves, paged_attention(q, kc, vc, moves.dst[:, None], moves.rows, workspace=ws, max_q_len=1)

    moves, _ = run()
    torch.cuda.synchronize()
    rows, dst = moves.rows.clone(), moves.dst.clone()
    want = paged_attention(q, kc, vc, dst[:, None], rows, max_q_len=1).clone()
    torch.cuda.synchronize()
    for call in (run, fork_only):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = [call() for _ in range(6)]
        graph.replay()
        torch.cuda.synchronize()
        for m, o in got:
            assert torch.equal(m.rows, rows) and torch.equal(o, want)
