"""Logits whose difference is beyond the largest number of 32 bits while their
log probabilities, at a high temperature, are not."""
import numpy as np
import pytest

import logits_ref as ref
from aetcnn import BF16, F32
from test_gpu_logits import Forward, Rows, near, sample

pytestmark = pytest.mark.gpu

BIG = 3.3895313892515355e38  # the largest bf16 value


def far_rows(rng, n):
    x = sample(rng, 4, n)
    x[0, 3], x[0, 5] = BIG, -BIG
    x[1] = rng.choice([BIG, -BIG, BIG / 2, -BIG / 4], n)
    x[2] = -BIG
    x[2, n // 2] = BIG
    x[3, ::2] = -BIG
    return x


@pytest.mark.parametrize("n", [12, 3000, 131072])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("t", [4.0, 1000.0, 1e6])
def test_log_probabilities(gpu, n, kind, t):
    rng = np.random.default_rng(n)
    rows = Rows(far_rows(rng, n), kind)
    ids = np.array([5, int(rows.x[1].argmin()), 0, 0])
    f = Forward(gpu, rows, ids, 12, t)
    f.call()
    want = ref.logprobs(rows.x, ids, 12, t)
    assert np.isfinite(want["logprobs"][0]).all() and want["logprobs"][0].min() < -1e31
    for name, v in f.read().items():
        near(v, want[name], name)
