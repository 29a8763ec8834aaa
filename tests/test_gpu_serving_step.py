"""The operators of a serving step together, as they are used: prompts are prefilled with normed and rotated
queries and keys, each forks into several continuations, every continuation decodes and samples its tokens on
the pool it shares, finished ones give their pages up, and the pool is compacted in between. Everything that
moves pages is exact, so the paged run has to give bit for bit the tokens and attention outputs of a run that
keeps every continuation's keys in pages of its own."""
from __future__ import annotations

import pytest
import torch

from kernels.attention import paged_attention, paged_decode_step, qk_norm_rope_append
from kernels.kv_cache import kv_compact, kv_copy_pages, kv_fork, kv_free, kv_paged_lookup
from kernels.rope import build_rope_tables
from kernels.softmax import sample_tokens

pytestmark = [pytest.mark.gpu]
DEV = "cuda"
HQ, HKV, D, BS, VOCAB, LAYERS = 8, 2, 128, 16, 2000, 2


class _Model:
    """Two attention layers over random projections of an embedding; only here to give q, k, v and logits."""

    def __init__(self, dtype):
        g = torch.Generator(device=DEV).manual_seed(1)
        rnd = lambda *s: torch.randn(*s, generator=g, device=DEV).to(dtype)  # noqa: E731
        self.emb = rnd(VOCAB, 64)
        self.qkv = [rnd(64, (HQ + 2 * HKV) * D) * 0.125 for _ in range(LAYERS)]
        self.out = [rnd(HQ * D, 64) * 0.05 for _ in range(LAYERS)]
        self.head = rnd(64, VOCAB)
        self.wq, self.wk = rnd(D) * 0.2 + 1, rnd(D) * 0.2 + 1
        self.cos, self.sin = build_rope_tables(512, D, dtype=torch.float32, device=DEV)

    def project(self, layer, x):
        # row by row, so that a token's numbers do not depend on the batch it comes in
        qkv = (x[:, None, :].float() @ self.qkv[layer].float()).to(x.dtype).view(-1, HQ + 2 * HKV, D)
        return qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:]

    def mix(self, layer, x, a):
        return x + (a.reshape(-1, 1, HQ * D).float() @ self.out[layer].float()).to(x.dtype)[:, 0]

    def logits(self, x):
        return (x[:, None, :].float() @ self.head.float())[:, 0]


def _slots(table, lens):
    page = table.gather(1, (lens // BS).long()[:, None])[:, 0]
    return page * BS + (lens % BS).long()


def _open_pages(table, lens, counts):
    """A page for every row whose next token begins one: the lowest free pages, in row order."""
    rows = (lens % BS == 0).nonzero()[:, 0]
    if rows.numel():
        free = (counts == 0).nonzero()[:rows.numel(), 0]
        table[rows, (lens[rows] // BS).long()] = free
        counts[free] = 1


def _decode(model, pools, table, lens, tokens, counts):
    _open_pages(table, lens, counts)
    slots, ctx = _slots(table, lens), (lens + 1).to(torch.int32)
    x = model.emb[tokens]
    for layer, (k_cache, v_cache) in enumerate(pools):
        q, k, v = model.project(layer, x)
        a = paged_decode_step(q, k, v, k_cache, v_cache, table, ctx, slots, lens.to(torch.int32), model.cos, model.sin,
                              q_norm_weight=model.wq, k_norm_weight=model.wk)
        x = model.mix(layer, x, a)
    return model.logits(x)


def _prefill(model, pools, table, prompts, counts):
    for b, prompt in enumerate(prompts):
        n = prompt.shape[0]
        pages = (n + BS - 1) // BS
        free = (counts == 0).nonzero()[:pages, 0]
        table[b, :pages] = free
        counts[free] = 1
        pos = torch.arange(n, device=DEV, dtype=torch.int32)
        slots = table[b][(pos // BS).long()] * BS + pos % BS
        x = model.emb[prompt]
        for layer, (k_cache, v_cache) in enumerate(pools):
            q, k, v = model.project(layer, x)
            q = qk_norm_rope_append(q, k, v, k_cache, v_cache, slots, pos, model.cos, model.sin, model.wq, model.wk)
            a = paged_attention(q, k_cache, v_cache, table[b:b + 1], torch.tensor([n], dtype=torch.int32, device=DEV),
                                q_start=torch.tensor([0, n], dtype=torch.int32, device=DEV), max_q_len=n)
            x = model.mix(layer, x, a)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_parallel_sampling_on_shared_pages(native, dtype):
    model = _Model(dtype)
    g = torch.Generator(device=DEV).manual_seed(7)
    prompts = [torch.randint(0, VOCAB, (n,), generator=g, device=DEV) for n in (37, 64, 1, 90)]
    B, children, steps, width, blocks = len(prompts), 3, 20, 9, 120
    parents = torch.arange(B, device=DEV, dtype=torch.int32).repeat_interleave(children)
    u = torch.rand(steps, B * children, generator=g, device=DEV)
    settings = dict(temperature=0.9, top_k=50, top_p=0.95, min_p=0.01)

    def pools():
        return [tuple(torch.zeros(blocks, HKV, BS, D, dtype=dtype, device=DEV) for _ in range(2)) for _ in range(LAYERS)]

    # shared: prefill once, fork, free the prompts' own rows, decode with a compaction on the way
    shared = pools()
    counts = torch.zeros(blocks, dtype=torch.int32, device=DEV)
    counts[::5] = 1  # pages of somebody else, so that the pool has holes
    table = torch.full((B, width), -1, dtype=torch.int64, device=DEV)
    _prefill(model, shared, table, prompts, counts)
    lens = torch.tensor([p.shape[0] for p in prompts], device=DEV, dtype=torch.int32)
    child, moves = kv_fork(table, lens, parents, counts, BS)
    kv_copy_pages([p[0] for p in shared], [p[1] for p in shared], moves)
    kv_free(table, torch.arange(B, device=DEV, dtype=torch.int32), counts)
    lens = lens[parents.long()]
    tokens = torch.stack([prompts[int(p)][-1] for p in parents])
    got = []
    for step in range(steps):
        if step == 6:  # somebody else's pages go, and the pool is compacted
            counts[::5] -= 1
            counts.clamp_(min=0)
            _, moves = kv_compact(child, counts)
            kv_copy_pages([p[0] for p in shared], [p[1] for p in shared], moves)
            live = int((counts > 0).sum())
            assert not counts[live:].any() and int(child.max()) < live
        logits = _decode(model, shared, child, lens, tokens, counts)
        tokens = sample_tokens(logits, u[step], **settings)
        lens = lens + 1
        got.append((logits, tokens))

    # apart: every continuation with its own pages and its own prefill
    apart = [tuple(torch.zeros(200, HKV, BS, D, dtype=dtype, device=DEV) for _ in range(2)) for _ in range(LAYERS)]
    counts2 = torch.zeros(200, dtype=torch.int32, device=DEV)
    table2 = torch.full((B * children, width), -1, dtype=torch.int64, device=DEV)
    _prefill(model, apart, table2, [prompts[int(p)] for p in parents], counts2)
    lens2 = torch.tensor([prompts[int(p)].shape[0] for p in parents], device=DEV, dtype=torch.int32)
    tokens2 = torch.stack([prompts[int(p)][-1] for p in parents])
    for step in range(steps):
        logits = _decode(model, apart, table2, lens2, tokens2, counts2)
        tokens2 = sample_tokens(logits, u[step], **settings)
        lens2 = lens2 + 1
        assert torch.equal(logits, got[step][0]), step
        assert torch.equal(tokens2, got[step][1]), step
    for (k1, v1), (k2, v2) in zip(shared, apart):
        a = kv_paged_lookup(k1, v1, child, lens, int(lens.max()))
        b = kv_paged_lookup(k2, v2, table2, lens2, int(lens2.max()))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # the continuations differ, and all pages come back
    assert len({tuple(t.tolist()) for t in torch.stack([t for _, t in got], 1)}) > B
    kv_free(child, torch.arange(B * children, device=DEV, dtype=torch.int32), counts)
    assert not counts.any() and bool((child == -1).all())
