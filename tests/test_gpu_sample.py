"""Token sampling against the definition in 64 bits, row by row. Tokens are whole numbers and have to be
equal. The operator's weights are off by 2^-39 of themselves or half of 2^-45 of the largest, so a running sum is
off by 2e-12 of the total: a row differs only where the number drawn, or top-p, meets one of its V borders that
closely, which of some 3000 seeded rows of at most 900001 logits happens with a chance of 1e-3 in all."""
from __future__ import annotations

import math

import pytest
import torch

import sample_oracle
from kernels.softmax import sample_tokens

pytestmark = [pytest.mark.gpu]
DEV = "cuda"
SETTINGS = [dict(), dict(top_k=1), dict(top_k=40), dict(top_k=700, temperature=1.7), dict(top_p=0.9), dict(top_p=0.3, temperature=0.6),
            dict(min_p=0.05), dict(top_k=50, top_p=0.95, min_p=0.01, temperature=0.8), dict(top_k=3000, top_p=0.8),
            dict(temperature=0.0), dict(top_p=0.0), dict(min_p=1.0), dict(top_p=0.999, min_p=1e-4)]


def _rows(B, V, dtype, seed, kind="peaks"):
    g = torch.Generator().manual_seed(seed)
    x = 2.0 * torch.randn(B, V, generator=g)
    if kind == "peaks":
        n = min(V, 40)
        at = torch.randint(0, V, (B, n), generator=g)
        x.scatter_(1, at, 14.0 * torch.rand(B, 1, generator=g) - 0.3 * torch.arange(n))
    elif kind == "ties":  # a handful of values, so thousands of equal logits
        x = torch.round(x)
    return x.to(dtype), torch.rand(B, generator=g)


def _same(x, u, x_dev=None, **kw):
    want = sample_oracle.tokens(x, u, **kw)
    dev = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in kw.items()}
    got = sample_tokens((x.to(DEV) if x_dev is None else x_dev), u.to(DEV), **dev)
    assert got.dtype == torch.int64 and got.tolist() == want, kw


@pytest.mark.parametrize("kind", ["peaks", "flat", "ties"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V,B", [(1, 3), (2, 5), (7, 4), (33, 9), (1000, 30), (4097, 6), (32000, 1), (50257, 3), (131072, 2)])
def test_settings(native, V, B, dtype, kind):
    x, u = _rows(B, V, dtype, V + B, kind)
    for kw in SETTINGS:
        _same(x, u, **kw)


@pytest.mark.parametrize("V,dtype", [(200003, torch.float32), (500001, torch.float32), (900001, torch.float16)])
def test_long_rows(native, V, dtype):
    """Slices of one CTA an SM, and rows that do not fit the cluster's shared memory."""
    x, u = _rows(2, V, dtype, V)
    for kw in (dict(), dict(top_k=60, top_p=0.9), dict(top_p=0.9), dict(top_k=5000), dict(temperature=0.0)):
        _same(x, u, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_settings_per_row_and_batch_sizes(native, dtype):
    """Every row its own settings; a row gives the same token alone and in any batch (any cluster size)."""
    B, V = 333, 9001
    x, u = _rows(B, V, dtype, 4)
    g = torch.Generator().manual_seed(5)
    pick = lambda *v: torch.tensor(v)[torch.randint(0, len(v), (B,), generator=g)]  # noqa: E731
    kw = dict(temperature=pick(0.0, 0.5, 1.0, 2.0, -1.0), top_k=pick(0, 1, 30, 600, 9001, -5, 20000).to(torch.int32),
              top_p=pick(1.0, 0.5, 0.95, 0.0, 1.5), min_p=pick(0.0, 0.1, 2.0, -1.0))
    _same(x, u, **kw)
    whole = sample_tokens(x.to(DEV), u.to(DEV), **{k: v.to(DEV) for k, v in kw.items()}).tolist()
    for n in (1, 3, 20, 100):
        part = {k: v[:n].to(DEV) for k, v in kw.items()}
        assert sample_tokens(x[:n].to(DEV), u[:n].to(DEV), **part).tolist() == whole[:n]


@pytest.mark.parametrize("B,V", [(100, 9001), (200, 70001)])
def test_list_rows_beside_others(native, B, V):
    """Rows with a small top-k in a batch with others, in one launch and in two; among them some whose thousands
    of equal logits overflow the list."""
    x, u = _rows(B, V, torch.bfloat16, 6)
    x[::5] = torch.round(x[::5])
    x[7] = -math.inf
    top_k = torch.tensor([30, 0, 511, 1])[torch.arange(B) % 4].to(torch.int32)
    _same(x, u, top_k=top_k, top_p=torch.tensor([0.9, 1.0])[torch.arange(B) % 2])


@pytest.mark.parametrize("V", [64, 5000, 40000])
def test_equal_logits(native, V):
    """All logits equal: every border is a whole number of tokens, hit exactly; far more ties than a list takes."""
    for value in (0.0, -3.5, torch.finfo(torch.float32).min):
        x = torch.full((6, V), value)
        u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1.0])
        for kw in (dict(), dict(top_k=V // 2), dict(top_p=0.5), dict(top_k=V // 4, top_p=0.5), dict(top_k=3), dict(min_p=1.0)):
            _same(x, u, **kw)
    x[:, ::2] = 0.0  # -0 and +0 are one value
    x[:, 1::2] = -0.0
    _same(x, u, top_k=V // 2)
    _same(x, u, temperature=0.0)


@pytest.mark.parametrize("offset", [0.0, -40.0, 3e4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V,width", [(1500, 0.05), (1999, 1e-3), (4097, 0.1), (50257, 0.5)])
def test_crowded_borders(native, V, width, dtype, offset):
    """Rows so narrow that hundreds of logits, distinct and equal ones, share the border's bin."""
    g = torch.Generator().manual_seed(V)
    x = (offset + width * torch.randn(4, V, generator=g)).to(dtype)
    x[3, ::7] = offset
    u = torch.rand(4, generator=g)
    for kw in (dict(top_p=0.9), dict(top_p=0.37), dict(top_k=V - 600), dict(top_k=V // 2, top_p=0.6),
               dict(top_p=0.5, temperature=40.0), dict(top_k=V - 700, temperature=1e30), dict(top_p=0.8, temperature=1e-3)):
        _same(x, u, **kw)


def test_masks_infinities_and_nan(native):
    V = 6000
    x, _ = _rows(10, V, torch.float32, 9)
    u = torch.linspace(0.0, 0.999, 10)
    lowest = torch.finfo(torch.float32).min
    x[0] = -math.inf
    x[1] = float("nan")
    x[2] = -math.inf; x[2, 4321] = -7.0
    x[3, :] = lowest; x[3, 17] = 2.0
    x[4, 10:5990] = -math.inf
    x[5, 100] = math.inf; x[5, 2000] = math.inf
    x[6, ::3] = float("nan")
    x[7] = lowest
    x[8, 5:] = lowest
    x[9] = 3e38; x[9, 0] = -3e38
    for kw in SETTINGS + [dict(temperature=math.inf), dict(temperature=1e-38), dict(temperature=1e30, top_k=7)]:
        if kw.get("temperature") == math.inf:
            keep = [0, 1, 2, 4, 6]  # at T = inf every finite logit weighs the same, lowest values too
            want = []
            for b in keep:
                row = torch.nan_to_num(x[b].double(), nan=-math.inf, neginf=-math.inf)
                idx = (row > -math.inf).nonzero()[:, 0].tolist()
                want.append(idx[min(len(idx) - 1, int(float(u[b]) * len(idx)))] if idx else -1)
            assert sample_tokens(x[keep].to(DEV), u[keep].to(DEV), **kw).tolist() == want
            continue
        _same(x, u, **kw)
    half = x.clamp(-6e4, 6e4).to(torch.float16)
    half[0] = -math.inf
    _same(half, u, top_p=0.9)


def test_uniform_out_of_range(native):
    x, _ = _rows(4, 3000, torch.float32, 10)
    u = torch.tensor([1.0, 7.0, -0.5, float("nan")])
    for kw in (dict(), dict(top_k=20)):
        got = sample_tokens(x.to(DEV), u.to(DEV), **kw).tolist()
        lo = sample_oracle.tokens(x, torch.zeros(4), **kw)
        hi = sample_oracle.tokens(x, torch.full((4,), 2.0), **kw)
        assert got == [hi[0], hi[1], lo[2], lo[3]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(native, dtype):
    B, V = 5, 3001
    x, u = _rows(B, V, dtype, 11)
    big = torch.full((B, V + 37), 50.0, dtype=dtype, device=DEV)
    for shift in range(0, 9):
        view = big[:, shift:shift + V]
        view.copy_(x)
        for kw in (dict(top_k=30, top_p=0.9), dict(top_p=0.9), dict(), dict(temperature=0.0)):
            _same(x, u, x_dev=view, **kw)
        big.fill_(50.0)
    one = x[:1].to(DEV).expand(B, V)  # one row of logits, several draws
    _same(x[:1].expand(B, V), u, x_dev=one, top_p=0.95)
    turned = x.t().contiguous().t()
    _same(x, u, x_dev=turned.to(DEV).t().contiguous().t(), top_k=9)
    out = torch.full((B,), -9, dtype=torch.int64, device=DEV)
    assert sample_tokens(x.to(DEV), u.to(DEV), out=out) is out and out.tolist() == sample_oracle.tokens(x, u)


def test_distribution(native):
    """Draws at evenly spaced numbers give every token its share, to one draw."""
    p = torch.tensor([0.5, 0.25, 0.125, 0.0625, 0.0625])
    n = 4096
    x = p.log().expand(n, 5).contiguous()
    u = (torch.arange(n) + 0.5) / n
    got = sample_tokens(x.to(DEV), u.to(DEV)).bincount(minlength=5).cpu()
    assert (got - p * n).abs().max() <= 1


@pytest.mark.parametrize("B,V,dtype", [(300, 60000, torch.float32), (300, 60001, torch.bfloat16), (64, 200003, torch.float16)])
def test_draws_along_a_row(native, B, V, dtype):
    """Evenly spaced numbers on one flat row: the token lies in every stretch of it, of every CTA and warp."""
    x, _ = _rows(1, V, dtype, 21, "flat")
    u = (torch.arange(B) + 0.25) / B
    for kw in (dict(), dict(top_p=0.9, min_p=1e-4)):
        _same(x.expand(B, V), u, x_dev=x.to(DEV).expand(B, V), **kw)


def test_refusals(native):
    x, u = torch.zeros(2, 8, device=DEV), torch.zeros(2, device=DEV)
    for bad in (lambda: sample_tokens(x[0], u), lambda: sample_tokens(x, u[:1]), lambda: sample_tokens(x[:, :0], u),
                lambda: sample_tokens(x, u, temperature=-1.0), lambda: sample_tokens(x, u, temperature=float("nan")),
                lambda: sample_tokens(x, u, top_p=1.5), lambda: sample_tokens(x, u, min_p=-0.1),
                lambda: sample_tokens(x, u, top_k=-1), lambda: sample_tokens(x, u, top_k=torch.zeros(3, device=DEV)),
                lambda: sample_tokens(x, u, out=torch.zeros(2, device=DEV)), lambda: sample_tokens(x.double(), u),
                lambda: sample_tokens(x, u, backend="metal")):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: sample_tokens(x.cpu(), u), lambda: sample_tokens(x, u.cpu()),
                lambda: sample_tokens(x, u, top_p=torch.ones(2))):
        with pytest.raises(RuntimeError):
            bad()
    assert sample_tokens(x[:0], u[:0]).shape == (0,)


def test_stream_and_graph(native):
    x, u = _rows(40, 20000, torch.bfloat16, 12)
    gx, gu, out = x.to(DEV), u.to(DEV), torch.empty(40, dtype=torch.int64, device=DEV)
    kw = dict(top_k=50, top_p=0.9, temperature=0.7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample_tokens(gx, gu, **kw)
    side.synchronize()
    assert got.tolist() == sample_oracle.tokens(x, u, **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sample_tokens(gx, gu, out=out, **kw)
    x2, u2 = _rows(40, 20000, torch.bfloat16, 13)
    gx.copy_(x2); gu.copy_(u2)
    graph.replay()
    torch.cuda.synchronize()
    assert out.tolist() == sample_oracle.tokens(x2, u2, **kw)
