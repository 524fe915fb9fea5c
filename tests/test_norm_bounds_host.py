"""The bounds that layer norm's statistics are held to (norm_bounds.py), without a
GPU: sums in 64 bits keep them, the same sums in 32 bits, or of differences in 32
bits, do not."""
import numpy as np
import pytest

import norm_bounds
from norm_ref import F32


def statistics(x, eps, sums, differences):
    """mean and rstd from one pass over x - x[0], summed in short chains"""
    f = x[:, :1].astype(np.float32)
    d = (x.astype(differences) - f.astype(differences)).astype(sums)
    n = x.shape[1]
    s, q = (v.sum(1, dtype=sums) / sums(n) for v in (d, d * d))
    var = np.maximum(q - s * s, 0).astype(np.float64) + eps
    return ((f[:, 0].astype(np.float64) + s).astype(np.float32),
            (1 / np.sqrt(var.astype(np.float32).astype(np.float64))).astype(np.float32))


def within(x, eps, sums, differences):
    want = norm_bounds.forward(x, None, None, eps, F32)
    got = statistics(x, eps, sums, differences)
    return [(np.abs(g - want[name][0]) <= want[name][1]).all() for name, g in zip(("mean", "rstd"), got)]


def rows(n, background):
    rng = np.random.default_rng(n)
    x = rng.standard_normal((6, n)) + 0.3 if background is None else np.full((6, n), background)
    if background is not None:
        x[:, 0] = 1000, -1000, 3e4, 1e6, 17, 300
    return x.astype(np.float32).astype(np.float64)


@pytest.mark.parametrize("n", [100, 1000, 10000, 100000])
@pytest.mark.parametrize("eps", [1e-12, 1e-5, 1.0])
@pytest.mark.parametrize("background", [None, 0.3])
def test_bounds(n, eps, background):
    x = rows(n, background)
    assert within(x, eps, np.float64, np.float64) == [True, True]
    if background is None:
        assert not all(within(x, eps, np.float32, np.float32))
    else:
        assert not within(x, eps, np.float64, np.float32)[0]
