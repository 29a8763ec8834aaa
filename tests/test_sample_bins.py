"""The bins of the sampling kernel's histogram, in the kernel's own arithmetic on the host: whatever the largest logit and the
temperature, a logit that is given a bin is given one of kBins. (The kernel does not check the index.)"""
from __future__ import annotations

import re
from pathlib import Path

import numpy as np

SOURCE = (Path(__file__).resolve().parent.parent / "reflex-infer_b200" / "csrc" / "sample.cu").read_text()
LOWEST = np.float32(-3.402823466e38)


def _zero_below(top, scale, shift, rounds_up):
    wide = np.float64(min(np.float32(top), -LOWEST))
    exact = wide - 32.0 * (shift + 2) / scale
    if exact <= LOWEST:
        return LOWEST
    f = np.float32(exact)
    if rounds_up and np.float64(f) < exact:
        f = np.nextafter(f, np.float32(np.inf))
    return max(LOWEST, f)


def _largest_bin(top, temperature, shift, rounds_up):
    """Of the smallest float that weighs anything beside `top`."""
    t = max(np.float64(np.float32(temperature)), 1e-20)
    scale = max(32.0 * 1.4426950408889634 / t, 1e-300)
    v = _zero_below(top, scale, shift, rounds_up)
    d = np.float64(min(v, -LOWEST)) - np.float64(min(np.float32(top), -LOWEST))
    return int(-np.rint(d * scale))


def test_every_bin_is_inside_the_histogram():
    bins = int(re.search(r"kBins = (\d+)", SOURCE).group(1))
    body = SOURCE[SOURCE.index("void set_top("):]
    rounds_up = "__double2float_ru" in body[:body.index("\n    }")]
    rng = np.random.default_rng(0)
    cases = [(1000.0, 1e-6), (999.99994, 1e-6), (1e8, 0.15), (-1000.0, 1e-6), (0.0, 1.0), (3e38, 1e30), (1e-30, 1e-38), (10.0, 2e-8)]
    for _ in range(20000):  # temperatures whose whole range of weights is near one step of the type at the largest logit
        top = np.float32(rng.choice([-1, 1]) * 10.0 ** rng.uniform(-6, 38))
        cases.append((top, np.spacing(abs(top)) / 36.0 * rng.uniform(0.2, 4.0)))
    for _ in range(5000):
        cases.append((np.float32(rng.normal() * 10.0 ** rng.uniform(-3, 6)), 10.0 ** rng.uniform(-20, 6)))
    with np.errstate(over="ignore"):
        for top, t in cases:
            for shift in (38, 45, 50):
                b = _largest_bin(top, t, shift, rounds_up)
                assert 0 <= b < bins, (top, t, shift, b)
