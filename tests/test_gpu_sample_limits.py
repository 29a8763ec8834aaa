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
