"""Distillation of rows whose logits are all low, or all far from 0 at a low
temperature, with listed classes that the student has masked: a masked class
has no probability, wherever the logits of its row lie.  The bounds are those
of logits_ref.py."""
import numpy as np
import pytest

from aetcnn import BF16, F16, F32, DISTILL_RENORM, DISTILL_TAIL
from test_gpu_logits import Distill, Rows

pytestmark = pytest.mark.gpu

ALLOWED = 40  # classes that rows of many listed ones leave unmasked


def rows_at(rng, n, k, base, spread):
    """0: of k listed classes some are masked (with k over 64: all of a wave's),
    and the teacher gives these no probability; 1: every listed class is masked;
    2: the label is, and the teacher does not list it; 3: nothing is masked"""
    x = base + spread * rng.standard_normal((4, n))
    ids = np.stack([rng.permutation(n)[:k] for _ in range(4)])
    values = np.log(rng.dirichlet(np.ones(k), 4) * 0.9)
    few = min(ALLOWED, k // 2)
    keep = np.zeros(n, bool)
    keep[ids[0, :few]] = True
    x[0, ~keep] = -np.inf
    values[0, few:] = -np.inf
    x[1, ids[1]] = -np.inf
    labels = np.array([ids[0, 0], ids[1, 0], 0, ids[3, 1]])
    labels[2] = np.setdiff1d(np.arange(n), ids[2])[0]
    x[2, labels[2]] = -np.inf
    return x, ids, values, labels


@pytest.mark.parametrize("base", [-1000.0, -100.0, -9.0, 100.0])
@pytest.mark.parametrize("t", [1.0, 0.25, 0.05])
@pytest.mark.parametrize("n,k,kind", [(12, 4, F32), (300, 128, F32), (1000, 10, F16),
                                      (6000, 100, BF16), (131072, 4, BF16), (40000, 128, F32)])
def test_masked_listed_classes(gpu, n, k, kind, t, base):
    rng = np.random.default_rng(n + k)
    x, ids, values, labels = rows_at(rng, n, k, base, max(t, 2.0 ** -7 * abs(base)))
    rows = Rows(x, kind)
    for mode in (DISTILL_RENORM, DISTILL_TAIL):
        for soft, hard in ((1.0, 0.0), (0.5, 0.5), (0.0, 1.0)):
            d = Distill(gpu, rows, ids, values, labels, None, t, mode, soft, hard)
            d.call()
            d.check()
            assert np.isfinite(d.out.read()).all()
            loss = d.loss.numpy()
            assert np.isposinf(loss[1]) and np.isfinite(loss[[0, 3]]).all()
            assert np.isposinf(loss[2]) == (hard != 0)
