"""Norm + rotation of every query and key head in one pass, dense and straight into the pool, against the
formula in 64 bits.

Tolerance, derived before the first run: with u = 2^-24 the fp32 sum of D squares is off by at most D*u of
its value, so the factor 1/sqrt is off by D*u/2 and 5u of roundings (inv_d and the sum with eps, halved by the
root; the reciprocal root's 2 ulp); an output's weight times table factor, product, sum and product with 1/sqrt
add 4u: every output is within (D/2 + 9) * u * (|n_i c| + |n_j s|) of the formula before it is rounded once to
the type (half a step, eps / 2, relative; half the smallest subnormal below the normal range)."""
from __future__ import annotations

import pytest
import torch

import oracle
import workloads
from kernels.attention import int8_pool, paged_decode, paged_decode_step, qk_norm_rope_append
from kernels.rope import qk_norm_rope, qk_norm_rope_

pytestmark = [pytest.mark.gpu]
DEV = "cuda"
U = 2.0 ** -24
HALF_SUBNORMAL = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def _tables(rows, D, interleaved, dtype, seed=1):
    half = D // 2
    ang = torch.arange(rows, dtype=torch.float64)[:, None] / 1e4 ** (torch.arange(half, dtype=torch.float64) / half)
    ang = ang.repeat_interleave(2, 1) if interleaved else torch.cat([ang, ang], 1)
    return ang.cos().to(dtype).to(DEV), ang.sin().to(dtype).to(DEV)


def _formula(x, w, cos, sin, eps, interleaved):
    """(values, |n_i c| + |n_j s|) in 64 bits."""
    x = x.double()
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    half = x.shape[-1] // 2
    c, s = cos.double()[:, None], sin.double()[:, None]
    if interleaved:
        i, j = n[..., 0::2], n[..., 1::2]
        c, s = c[..., 0::2], s[..., 0::2]
        pair = lambda a, b: torch.stack([a, b], -1).flatten(-2)  # noqa: E731
    else:
        i, j = n[..., :half], n[..., half:]
        c, s = c[..., :half], s[..., :half]
        pair = lambda a, b: torch.cat([a, b], -1)  # noqa: E731
    return pair(i * c - j * s, i * s + j * c), pair((i * c).abs() + (j * s).abs(), (i * s).abs() + (j * c).abs())


def _check(got, want, mag, D):
    off = (D / 2 + 9) * U * mag
    tol = off + (want.abs() + off) * torch.finfo(got.dtype).eps / 2 + HALF_SUBNORMAL[got.dtype]
    bad = ((got.double() - want).abs() > tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside, worst {((got.double() - want).abs() / tol).max():.3g}"


def _inputs(n, hq, hkv, D, dtype, seed, packed=True, shift=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    heads = hq + 2 * hkv
    flat = torch.empty(n * heads * D + shift, dtype=dtype, device=DEV)
    qkv = flat[shift:].view(n, heads, D)
    qkv.copy_(torch.randn(n, heads, D, generator=g, device=DEV) * 2.0 ** torch.randint(-3, 4, (1, heads, 1), generator=g, device=DEV))
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    wq = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dtype)
    wk = (1 + 0.3 * torch.randn(D, generator=g, device=DEV)).to(dtype)
    return q, k, v, wq, wk


@pytest.mark.parametrize("tables", ["float32", "same"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [2, 6, 34, 64, 80, 96, 128, 256, 320, 512])
def test_dense_against_formula(native, D, dtype, interleaved, tables):
    for n, hq, hkv, shift in ((1, 16, 2, 0), (33, 7, 1, 0), (5, 1, 1, 1)):
        q, k, _, wq, wk = _inputs(n, hq, hkv, D, dtype, D + n, shift=shift)
        cos, sin = _tables(70, D, interleaved, torch.float32 if tables == "float32" else dtype)
        pos = torch.randint(0, 70, (n,), generator=torch.Generator().manual_seed(n)).to(torch.int32).to(DEV)
        qo, ko = qk_norm_rope(q, k, wq, wk, cos, sin, positions=pos, eps=1e-5, interleaved=interleaved)
        for got, x, w in ((qo, q, wq), (ko, k, wk)):
            want, mag = _formula(x, w, cos[pos.long()], sin[pos.long()], 1e-5, interleaved)
            _check(got, want, mag, D)


def test_edges(native):
    q, k, _, wq, wk = _inputs(6, 3, 2, 64, torch.bfloat16, 5)
    cos, sin = _tables(6, 64, False, torch.float32)
    # without positions token n has row n
    a = qk_norm_rope(q, k, wq, wk, cos, sin)
    b = qk_norm_rope(q, k, wq, wk, cos, sin, positions=torch.arange(6, device=DEV))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # in place, inside a packed projection: the same values, and nothing else touched
    q2, k2, v2, _, _ = _inputs(6, 3, 2, 64, torch.bfloat16, 5)
    v0 = v2.clone()
    r = qk_norm_rope_(q2, k2, wq, wk, cos, sin)
    assert r[0] is q2 and torch.equal(q2, a[0]) and torch.equal(k2, a[1]) and torch.equal(v2, v0)
    # a token without a table row: zeros in new tensors, unchanged in place
    pos = torch.tensor([0, 6, -1, 3, 4, 5], dtype=torch.int32, device=DEV)
    qo, ko = qk_norm_rope(q, k, wq, wk, cos, sin, positions=pos)
    assert not qo[1:3].any() and not ko[1:3].any() and torch.equal(qo[3:], a[0][3:]) and torch.equal(qo[0], a[0][0])
    q3, k3, _, _, _ = _inputs(6, 3, 2, 64, torch.bfloat16, 5)
    qk_norm_rope_(q3, k3, wq, wk, cos, sin, positions=pos)
    assert torch.equal(q3[1:3], q[1:3]) and torch.equal(k3[1:3], k[1:3]) and torch.equal(q3[3:], a[0][3:])
    # a head of zeros stays zero; no tokens, no heads
    z = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV)
    assert not qk_norm_rope(z, z, wq, wk, cos, sin)[0].any()
    assert qk_norm_rope(q[:0], k[:0], wq, wk, cos, sin)[0].shape == (0, 3, 64)
    only_k = qk_norm_rope(q[:, :0], k, wq, wk, cos, sin)
    assert only_k[0].shape == (6, 0, 64) and torch.equal(only_k[1], a[1])
    # a strided last axis is read through a copy
    t = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(qk_norm_rope(t, k, wq, wk, cos, sin)[0], a[0])


def test_refusals(native):
    q, k, v, wq, wk = _inputs(4, 2, 2, 64, torch.bfloat16, 6)
    cos, sin = _tables(8, 64, False, torch.float32)
    for bad in (lambda: qk_norm_rope(q[:3], k, wq, wk, cos, sin),
                lambda: qk_norm_rope(q[..., :32], k, wq, wk, cos, sin),
                lambda: qk_norm_rope(q, k, wq[:32], wk, cos, sin),
                lambda: qk_norm_rope(q, k, wq, wk, cos[:, :32], sin[:, :32]),
                lambda: qk_norm_rope(q, k, wq, wk, cos[:3], sin[:3]),
                lambda: qk_norm_rope(q, k, wq, wk, cos, sin, positions=torch.zeros(3, device=DEV)),
                lambda: qk_norm_rope(q, k, wq, wk, cos, sin, eps=-1.0),
                lambda: qk_norm_rope(q, k, wq, wk, cos, sin, backend="rocm"),
                lambda: qk_norm_rope(q[..., :63], k[..., :63], wq[:63], wk[:63], cos[:, :63], sin[:, :63]),
                lambda: qk_norm_rope_(q.transpose(1, 2).contiguous().transpose(1, 2), k, wq, wk, cos, sin),
                lambda: qk_norm_rope_(q[:, :1].expand(4, 2, 64), k, wq, wk, cos, sin)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: qk_norm_rope(q.float(), k, wq, wk, cos, sin),
                lambda: qk_norm_rope(q, k, wq.float(), wk, cos, sin),
                lambda: qk_norm_rope(q.cpu(), k, wq, wk, cos, sin)):
        with pytest.raises(RuntimeError):
            bad()
    big = torch.zeros(1, 1, 514, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="512"):
        qk_norm_rope(big, big, big[0, 0], big[0, 0], big[0], big[0])
    kc = torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16, device=DEV)
    slots, pos = torch.arange(4, device=DEV), torch.arange(4, device=DEV, dtype=torch.int32)
    with pytest.raises(ValueError):
        qk_norm_rope_append(q, k, v, kc[:, :1], kc[:, :1], slots, pos, cos, sin, wq, wk)
    with pytest.raises(ValueError):
        qk_norm_rope_append(q, k, v, kc, kc.clone(), slots[:3], pos, cos, sin, wq, wk)
    with pytest.raises(RuntimeError):
        qk_norm_rope_append(q, k, v, kc.float(), kc.float(), slots, pos, cos, sin, wq, wk)
    with pytest.raises(ValueError):
        qk_norm_rope_append(q, k, v, kc.to(torch.int8), kc.to(torch.int8), slots, pos, cos, sin, wq, wk)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D,hq,hkv,bs", [(64, 16, 16, 16), (128, 28, 4, 16), (80, 2, 1, 3), (34, 3, 3, 8), (256, 8, 1, 1)])
def test_append_against_dense(native, D, hq, hkv, bs, dtype, interleaved):
    """The pool holds bit for bit what the dense form gives and V as it came; other slots are left alone."""
    n, nb = 41, 60
    q, k, v, wq, wk = _inputs(n, hq, hkv, D, dtype, D)
    cos, sin = _tables(500, D, interleaved, dtype)
    g = torch.Generator().manual_seed(D)
    slots = torch.randperm(nb * bs, generator=g)[:n]
    pos = torch.randint(0, 500, (n,), generator=g).to(torch.int32)
    if nb * bs >= n:
        slots[3], slots[9] = -1, nb * bs
    pos[5], pos[11] = 500, -7
    kc = torch.randn(nb, hkv, bs, D, device=DEV).to(dtype)
    vc = torch.randn(nb, hkv, bs, D, device=DEV).to(dtype)
    want_k, want_v = kc.clone(), vc.clone()
    qd, kd = qk_norm_rope(q, k, wq, wk, cos, sin, positions=pos.to(DEV), interleaved=interleaved)
    keep = (slots >= 0) & (slots < nb * bs) & (pos >= 0) & (pos < 500)
    s = slots[keep].to(DEV)
    want_k[s // bs, :, s % bs] = kd[keep.to(DEV)]
    want_v[s // bs, :, s % bs] = v[keep.to(DEV)]
    out = qk_norm_rope_append(q, k, v, kc, vc, slots.to(DEV), pos.to(DEV), cos, sin, wq, wk, interleaved=interleaved)
    assert torch.equal(out, qd) and torch.equal(kc, want_k) and torch.equal(vc, want_v)
    # K and V alone; a pool view of another stride (a slice of a larger pool)
    wide = torch.zeros(nb, 2 * hkv, bs, D, dtype=dtype, device=DEV)
    k2, v2 = wide[:, :hkv], torch.zeros_like(wide)[:, :hkv]
    k2.copy_(want_k); v2.zero_()
    assert qk_norm_rope_append(None, k, v, k2, v2, slots.to(DEV), pos.to(DEV), cos, sin, wq, wk, interleaved=interleaved) is None
    assert torch.equal(k2, want_k) and not wide[:, hkv:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [128, 66])
def test_append_int8(native, D, dtype):
    n, hq, hkv, bs, nb = 29, 4, 2, 16, 4
    q, k, v, wq, wk = _inputs(n, hq, hkv, D, dtype, 3)
    v[4] = 0
    cos, sin = _tables(64, D, False, torch.float32)
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    slots = torch.randperm(nb * bs, generator=torch.Generator().manual_seed(1))[:n].to(DEV)
    kc, vc, ks, vs = int8_pool(nb, hkv, bs, D, DEV)
    out = qk_norm_rope_append(q, k, v, kc, vc, slots, pos, cos, sin, wq, wk, k_scales=ks, v_scales=vs)
    assert torch.equal(out, qk_norm_rope(q, k, wq, wk, cos, sin, positions=pos)[0])
    want, mag = _formula(k, wk, cos[pos.long()], sin[pos.long()], 1e-6, False)
    for rows, off, cache, scales in ((want, (D / 2 + 9) * U * mag, kc, ks), (v.double(), torch.zeros_like(want), vc, vs)):
        q8 = cache[slots // bs, :, slots % bs].double()
        sc = scales[slots // bs, :, slots % bs].double()
        top = rows.abs().amax(-1)
        # the scale is the largest of the fp32 rows / 127, rounded once more
        assert ((sc - torch.where(top > 0, top / 127, 1.0)).abs() <= off.amax(-1) / 127 + U * sc * 2).all()
        # a value is off by half a step, by the fp32 row's own error and by the quotient's rounding
        assert ((q8 * sc[..., None] - rows).abs() <= sc[..., None] * (0.5 + 130 * U) + off).all()
    untouched = torch.ones(nb * bs, dtype=torch.bool, device=DEV)
    untouched[slots] = False
    assert not kc.permute(0, 2, 1, 3).reshape(nb * bs, -1)[untouched].any()


def test_decode_step_with_norm(native):
    """paged_decode_step with norm weights = append with norm, then paged decode of the rotated queries; and
    the attention of a 64-bit softmax over the pool's own contents within the 16-bit attention tolerance."""
    cos, sin = _tables(700, 128, False, torch.bfloat16)
    b = workloads.make_paged_batch("norm", B=5, Hq=16, Hkv=2, D=128, block_size=16, ctx_range=(1, 600), num_blocks=256,
                                   device=DEV, seed=8, tables=(cos, sin))
    wq = torch.linspace(0.5, 1.5, 128, device=DEV).to(torch.bfloat16)
    wk = torch.linspace(1.5, 0.5, 128, device=DEV).to(torch.bfloat16)
    kc, vc = b.k_cache.clone(), b.v_cache.clone()
    got = paged_decode_step(b.q_new, b.k_new, b.v_new, b.k_cache, b.v_cache, b.block_table, b.context_lens,
                            b.slot_mapping, b.positions, cos, sin, q_norm_weight=wq, k_norm_weight=wk)
    qr = qk_norm_rope_append(b.q_new, b.k_new, b.v_new, kc, vc, b.slot_mapping, b.positions, cos, sin, wq, wk)
    want = paged_decode(qr, kc, vc, b.block_table, b.context_lens)
    assert torch.equal(kc, b.k_cache) and torch.equal(vc, b.v_cache) and torch.equal(got, want)
    ref = oracle.paged_attention_composed(qr.cpu(), kc.cpu(), vc.cpu(), b.block_table.cpu(), b.context_lens.cpu())
    torch.testing.assert_close(got.cpu().float(), ref.float(), atol=2e-2, rtol=2e-2)
    with pytest.raises(ValueError):
        paged_decode_step(b.q_new, b.k_new, b.v_new, b.k_cache, b.v_cache, b.block_table, b.context_lens,
                          b.slot_mapping, b.positions, cos, sin, q_norm_weight=wq)


def test_stream_and_graph(native):
    q, k, v, wq, wk = _inputs(64, 16, 2, 128, torch.bfloat16, 9)
    cos, sin = _tables(64, 128, False, torch.float32)
    pos = torch.arange(64, dtype=torch.int32, device=DEV)
    kc = torch.zeros(8, 2, 16, 128, dtype=torch.bfloat16, device=DEV)
    vc, slots = torch.zeros_like(kc), torch.randperm(128, device=DEV)[:64]
    q_out = torch.empty_like(q)
    call = lambda: qk_norm_rope_append(q, k, v, kc, vc, slots, pos, cos, sin, wq, wk, q_out=q_out)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    q.copy_(torch.randn_like(q)); k.copy_(torch.randn_like(k))
    graph.replay()
    torch.cuda.synchronize()
    want_q, want_k = qk_norm_rope(q, k, wq, wk, cos, sin, positions=pos)
    assert torch.equal(q_out, want_q) and torch.equal(kc[slots // 16, :, slots % 16], want_k)


@pytest.mark.parametrize("interleaved", [False, True])
def test_decode_step_with_norm_int8(native, interleaved):
    """The same step on an int8 pool equals the append with norm and the decode kernel's int8 form."""
    B, bs, nb = 4, 16, 40
    cos, sin = _tables(300, 128, interleaved, torch.float32)
    g = torch.Generator(device=DEV).manual_seed(2)
    q, k, v, wq, wk = _inputs(B, 8, 2, 128, torch.bfloat16, 4)
    pools = [int8_pool(nb, 2, bs, 128, DEV) for _ in range(2)]
    for kc, vc, ks, vs in pools:
        g.manual_seed(3)
        kc.random_(-127, 128, generator=g); vc.random_(-127, 128, generator=g)
        ks.uniform_(0.01, 0.02, generator=g); vs.uniform_(0.01, 0.02, generator=g)
    table = torch.randperm(nb, device=DEV, generator=g)[:B * 10].view(B, 10)
    lens = torch.tensor([1, 17, 64, 160], dtype=torch.int32, device=DEV)
    pos = lens - 1
    slots = table.gather(1, (pos // bs).long()[:, None])[:, 0] * bs + pos % bs
    (k1, v1, ks1, vs1), (k2, v2, ks2, vs2) = pools
    got = paged_decode_step(q, k, v, k1, v1, table, lens, slots, pos, cos, sin, interleaved=interleaved, k_scales=ks1,
                            v_scales=vs1, q_norm_weight=wq, k_norm_weight=wk, norm_eps=1e-5)
    qr = qk_norm_rope_append(q, k, v, k2, v2, slots, pos, cos, sin, wq, wk, eps=1e-5, interleaved=interleaved, k_scales=ks2,
                             v_scales=vs2)
    want = paged_decode(qr, k2, v2, table, lens, k_scales=ks2, v_scales=vs2)
    for a, b in ((got, want), (k1, k2), (v1, v2), (ks1, ks2), (vs1, vs2)):
        assert torch.equal(a, b)
