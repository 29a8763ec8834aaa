"""Token sampling where its arithmetic is at an end."""
from __future__ import annotations

import math

import pytest
import torch

import sample_oracle
from kernels.softmax import sample_tokens

pytestmark = [pytest.mark.gpu]
DEV = "cuda"


@pytest.mark.parametrize("top,temperature", [(1000.0, 1e-6), (1000.0, 2e-6), (1e8, 0.15), (-1000.0, 1e-6), (10.0, 2e-8), (1.5, 3e-9)])
def test_weights_that_end_within_a_step_of_the_largest_logit(native, top, temperature):
    """Neighbours of the largest logit one and two steps down, at temperatures around a 36th of a step: in the histograms their bins
    are the last ones. Their weights are below 2^-20 of the largest, so no sum comes near a border: all tokens are exact."""
    V = 3000
    g = torch.Generator().manual_seed(1)
    t = torch.tensor(top)
    down = [t]
    for _ in range(3):
        down.append(torch.nextafter(down[-1], torch.tensor(-math.inf)))
    x = torch.stack(down)[torch.randint(1, 4, (6, V), generator=g)]
    x[torch.arange(6)[:, None], torch.randint(0, V, (6, 5), generator=g)] = t
    step = float(down[0] - down[1])
    assert math.exp(-step / temperature) < 2.0 ** -20
    u = torch.linspace(0.05, 0.95, 6)
    for kw in (dict(top_p=0.9), dict(top_k=700), dict(top_k=2500, top_p=0.7), dict(), dict(top_k=40, top_p=0.9), dict(min_p=0.5)):
        want = sample_oracle.tokens(x, u, temperature=temperature, **kw)
        assert sample_tokens(x.to(DEV), u.to(DEV), temperature=temperature, **kw).tolist() == want, kw


def _off(M, w):
    """How far a running sum may be off, in units of the largest weight, on a row with M logits that can weigh anything (top-k, or
    all), one of them the largest and the others of weight w: half a unit and 2^-39 of itself for each. The unit is 2^-S, S =
    min(50, 63 - ceil(log2 M)) up to M = 2^18 (which top-k = 2^18 makes of a longer row); beyond, 2^-50 as long as the row's total,
    here below 2, leaves room for it (2^24 logits: 2^-27 in all)."""
    S = 50 if M > 1 << 18 else min(50, 63 - (M - 1).bit_length())
    return M * (2.0 ** -(S + 1) + 2.0 ** -39 * w)


def _peak_over_floor(V, peak, gap, dtype):
    """The row on the device, and the floor's weight."""
    x = torch.full((1, V), -gap, dtype=torch.float32).to(dtype)
    w = math.exp(float(x[0, 0]))
    x[0, peak] = 0.0
    return x.to(DEV), w


@pytest.mark.parametrize("V,dtype", [(50257, torch.float32), (131072, torch.float32), (1 << 18, torch.bfloat16), ((1 << 18) + 1, torch.float32),
                                     (900001, torch.float32), (1 << 24, torch.float32), (1 << 24, torch.bfloat16)])
@pytest.mark.parametrize("where", [0, 0.5, 1])
def test_one_token_over_a_floor_of_equal_ones(native, V, dtype, where):
    """Nearly all mass in one token, the rest in equal weights near or below the unit of the sums: each draw has to lie
    where the exact running sum says, to the bound. (Equal weights all round the same way, so nothing cancels.)"""
    peak = int(where * (V - 1))
    u = torch.tensor([0.0, 1e-9, 3e-8, 1e-6, 1e-5, 0.5, 1 - 2.0 ** -17, 1 - 2.0 ** -20, 1 - 2.0 ** -24])
    for gap in (20.0, 24.0, 26.5, 27.1, 28.5, 30.0, 31.9):
        x, w = _peak_over_floor(V, peak, gap, dtype)
        for factor, kw in ((1, dict()), (2, dict(temperature=2.0)), (1, dict(top_k=V - 1))):
            got = sample_tokens((x * factor).expand(len(u), V), u.to(DEV), **kw).tolist()
            out = V - 1 - (peak == V - 1) if "top_k" in kw else V  # the index that top-k drops: the last of the floor
            total = 1.0 + (V - 2 if out < V else V - 1) * w
            off = _off(kw.get("top_k", V), w)
            for t, r in zip(got, u.double().tolist()):
                assert t != out
                before = (t - (t > out)) * w + (1 - w if t > peak else 0)
                after = before + (1 if t == peak else w)
                assert before / total - 2 * off <= r <= after / total + 2 * off, (gap, kw, t, r)


@pytest.mark.parametrize("V", [131072, 900001, 1 << 24])
def test_top_p_that_cuts_such_a_floor(native, V):
    """A floor of 3e-5 of the mass, of which top-p = 1 - 2^-17 keeps some three quarters: the last token kept is the one at which the
    exact sum reaches the border, to the bound."""
    p = 1 - 2.0 ** -17
    for dtype in (torch.float32, torch.bfloat16):
        x, w = _peak_over_floor(V, 0, math.log(V / 3e-5), dtype)
        for kw in (dict(), dict(top_k=V - 1)):
            off = _off(kw.get("top_k", V), w)
            total = 1.0 + (kw.get("top_k", V) - 1) * w
            assert 1 + w < p * total < total - w
            last = sample_tokens(x, torch.ones(1, device=DEV), top_p=p, **kw).tolist()[0]
            assert 1 + (last - 1) * w - 2 * off <= p * total <= 1 + last * w + 2 * off, (dtype, last)


def test_long_rows_in_batches_and_with_top_k(native):
    """Top-k at and around the number of logits from which a row's sum decides its unit; rows give the same token alone and
    in a batch, whatever the CTAs of a row."""
    B, V = 40, 300007
    g = torch.Generator().manual_seed(3)
    x = (2 * torch.randn(B, V, generator=g)).to(torch.bfloat16)
    x[::3] = torch.round(x[::3].float()).to(torch.bfloat16)
    x[4] = -math.inf
    x[5] = -3.0
    u = torch.rand(B, generator=g)
    top_k = torch.tensor([0, 1 << 18, (1 << 18) + 1, V - 1, 5, 9000])[torch.arange(B) % 6].to(torch.int32)
    top_p = torch.tensor([1.0, 0.9])[torch.arange(B) % 2]
    want = sample_oracle.tokens(x, u, top_k=top_k, top_p=top_p)
    gx, gu, gk, gp = (t.to(DEV) for t in (x, u, top_k, top_p))
    assert sample_tokens(gx, gu, top_k=gk, top_p=gp).tolist() == want
    for b in (0, 1, 2, 3, 5, 11):
        assert sample_tokens(gx[b:b + 1], gu[b:b + 1], top_k=int(top_k[b]), top_p=float(top_p[b])).tolist() == want[b:b + 1]


@pytest.mark.parametrize("V,B", [(600, 7), (5000, 9), (40001, 4), (131072, 3)])
def test_top_k_up_to_the_longest_list(native, V, B):
    """Top-k rows with more kept than are ranked by comparing pairs, up to the 512 that the list way takes and one beyond."""
    g = torch.Generator().manual_seed(V)
    x = 2 * torch.randn(B, V, generator=g)
    x[0] = torch.round(x[0])
    x[1, V // 2:] = -math.inf
    u = torch.rand(B, generator=g)
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        for k in (128, 129, 227, 228, 300, 511, 512, 513):
            for kw in (dict(), dict(top_p=0.95), dict(top_p=0.6, min_p=0.02), dict(temperature=30.0), dict(min_p=1e-3, temperature=0.5)):
                assert sample_tokens(y.to(DEV), u.to(DEV), top_k=k, **kw).tolist() == sample_oracle.tokens(y, u, top_k=k, **kw), (k, kw)


@pytest.mark.parametrize("V", [20000, 60000, 128000])
def test_rows_masked_but_for_a_stretch(native, V):
    """Rows that several CTAs take, with whole slices of nothing but -inf: the few CTAs with logits give the answer."""
    g = torch.Generator().manual_seed(V)
    x = torch.full((6, V), -math.inf)
    x[0, :V // 8] = 2 * torch.randn(V // 8, generator=g)
    x[1, -V // 5:] = 2 * torch.randn(x[1, -V // 5:].shape, generator=g)
    x[2, V // 2:V // 2 + 30] = torch.randn(30, generator=g)
    x[3, ::997] = 1.5
    x[4, V - 1] = -4.0
    x[5] = torch.finfo(torch.float32).min
    x[5, 100:V // 3] = 2 * torch.randn(V // 3 - 100, generator=g)
    u = torch.tensor([0.1, 0.9, 0.5, 0.99, 0.3, 0.7])
    for dtype in (torch.float32, torch.bfloat16):
        y = x.to(dtype)
        for kw in (dict(), dict(top_k=40), dict(top_k=300, top_p=0.9), dict(top_p=0.9), dict(top_k=2000), dict(min_p=0.1), dict(temperature=0.0)):
            want = sample_oracle.tokens(y, u, **kw)
            assert sample_tokens(y.to(DEV), u.to(DEV), **kw).tolist() == want, kw
            assert sample_tokens(y[:1].to(DEV), u[:1].to(DEV), **kw).tolist() == want[:1], kw


def test_long_rows_in_a_launch_for_each_kind(native):
    """As many long rows as make top-k row by row two launches: the tokens that the rows have in small batches."""
    B, V = 160, (1 << 18) + 3
    g = torch.Generator(device=DEV).manual_seed(5)
    x = (2 * torch.randn(B, V, generator=g, device=DEV)).to(torch.bfloat16)
    u = torch.rand(B, generator=g, device=DEV)
    top_k = torch.tensor([30, 0, 5000, V - 1, 512, (1 << 18) + 1], device=DEV)[torch.arange(B, device=DEV) % 6].to(torch.int32)
    whole = sample_tokens(x, u, top_k=top_k, top_p=0.95)
    for b in range(0, B, 8):
        assert torch.equal(sample_tokens(x[b:b + 8], u[b:b + 8], top_k=top_k[b:b + 8], top_p=0.95), whole[b:b + 8])
