"""Layer norm's statistics against bounds of 64-bit sums (norm_bounds.py), where
a row's first value is far from the others."""
import numpy as np
import pytest

import norm_bounds
from aetcnn import BF16, F16, F32
from test_gpu_checkpoint import activations
from test_gpu_layernorm import SIZES, Backward, Forward, parameters
from test_gpu_logits import Rows

pytestmark = pytest.mark.gpu


def check_forward(gpu, x, s, b, eps=1e-5, keep=True):
    f = Forward(gpu, x, s, b, eps, keep=keep)
    f.want = norm_bounds.forward(x.x, s, b, eps, x.kind)
    f.call()
    f.check()
    return f


# rows of a part of a wave, a wave, workgroups of every size, and in parts
LENGTHS = [8, 40, 300, 1000, 4096, 9000, 16384, 17001, 186624]


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("n", LENGTHS)
def test_a_first_value_far_from_the_others(gpu, n, kind):
    """a constant background, whose differences from the first value all round
    alike, and one that is not; the same values in the other order"""
    rng = np.random.default_rng(n)
    s, b = parameters(rng, n)
    far = np.array([1000.0, -1000.0, 3e4, 0.3])
    for spread in (0.0, 0.01):
        x = 0.3 + spread * rng.standard_normal((4, n))
        x[:, 0] = far
        seen = []
        for order in (slice(None), slice(None, None, -1)):
            f = check_forward(gpu, Rows(x[:, order], kind), s, b)
            seen.append(f.stats.numpy()[:, 0].astype(np.float64))
        # the order of the values is of no consequence for their mean
        assert (np.abs(seen[0] - seen[1]) <= 2.0 ** -22 * np.abs(seen[1]) + 2.0 ** -30).all()


@pytest.mark.parametrize("n", LENGTHS)
def test_a_first_value_far_above_all(gpu, n):
    rng = np.random.default_rng(n + 1)
    s, b = parameters(rng, n)
    x = rng.standard_normal((5, n))
    x[:, 0] = 1e3, 1e6, -1e9, 1e15, 3e37
    check_forward(gpu, Rows(x, F32), s, b)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("n", [3, 33, 300, 1000, 4096, 9000, 17001])
def test_values_further_apart_than_the_largest(gpu, n, kind):
    """differences pass a float's range, from the first value or from the mean;
    statistics and outputs do not, whatever the order"""
    rng = np.random.default_rng(n)
    s, b = parameters(rng, n)
    x = np.full((6, n), 3e38)
    x[0, 0], x[0, -1] = 0, -3e38         # behind a small first value
    x[1, 0] = -3e38                      # all far from the first
    x[2, n // 2] = -3e38
    x[3, ::2] = -3e38
    x[4] = rng.uniform(-3.3e38, 3.3e38, n)
    x[5] = -3e38 * (np.arange(n) == n - 1) + 1e38
    f = check_forward(gpu, Rows(x, kind), s, b)
    st = f.stats.numpy().astype(np.float64)
    with np.errstate(over="raise"):
        assert np.isfinite(st).all() and (np.abs(st[:, 1] / f.want["rstd"][0] - 1) < 2.0 ** -20).all()
    g = Backward(gpu, Rows(rng.standard_normal((6, n)), kind), (f.x, 1e-5), s)
    g.call()
    g.check()


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("rows,n,pad,shift", SIZES + [(1500, 600, 0, 0), (700, 3000, 0, 0), (70, 60001, 0, 0)])
def test_ordinary_rows(gpu, rows, n, pad, shift, kind):
    """each with a level of its own, up to far above its deviations"""
    rng = np.random.default_rng(rows * 3 + n)
    x = activations(rng, rows, n) + rng.standard_normal((rows, 1)) * 10.0 ** rng.integers(-2, 4, (rows, 1))
    s, b = parameters(rng, n)
    check_forward(gpu, Rows(x, kind, pad, shift), s, b)


@pytest.mark.parametrize("n", [20, 1000, 5000, 40000])
@pytest.mark.parametrize("eps", [1e-12, 1e-5, 1.0])
def test_values_at_the_ends(gpu, n, eps):
    rng = np.random.default_rng(n)
    x = activations(rng, 8, n)
    x[0] = 3.25
    x[1] = 1e4 + rng.standard_normal(n) * 0.01
    x[2] = 1e4 + np.arange(n) % 2 * 2.0 ** -10        # one step apart
    x[3, 0] = 1e6
    x[4] *= 1e-30
    x[5] *= 1e15
    x[6] = np.where(np.arange(n) % 2, 1e25, -1e25)
    x[7] = 0
    s, b = parameters(rng, n)
    check_forward(gpu, Rows(x, F32), s, b, eps)
