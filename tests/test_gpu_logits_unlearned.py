"""Distillation of rows from which nothing is learned, no entry of the teacher
and no label being left: like rows of weight 0 their loss and delta are 0,
whatever their logits hold.  Rows that do have a term and hold a NaN or a +inf
give NaN in both."""
import numpy as np
import pytest

import logits_ref as ref
from aetcnn import BF16, F16, F32, DISTILL_RENORM, DISTILL_TAIL
from test_gpu_logits import Distill, Rows, near, sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("soft,hard", [(1.0, 0.0), (0.5, 0.25), (0.0, 1.0)])
@pytest.mark.parametrize("mode", [DISTILL_RENORM, DISTILL_TAIL])
@pytest.mark.parametrize("n,kind", [(10, F32), (1000, BF16), (9000, F32), (20000, F16),
                                    (131072, BF16)])
def test_rows_without_a_term(gpu, n, kind, mode, soft, hard):
    rng = np.random.default_rng(n)
    k = 4
    x = sample(rng, 12, n)
    ids = np.stack([rng.permutation(n)[:k] for _ in range(12)])
    values = np.log(rng.dirichlet(np.ones(k), 12) * 0.9)
    labels = np.full(12, -1)
    x[0] = np.nan               # garbage, and nothing to learn
    x[1, n // 2] = np.inf
    x[2] = -np.inf
    ids[:4] = -1                # 3: finite logits
    ids[4] = (-5, n, n + 7, 2 ** 31 - 1)
    labels[4] = n
    x[4, 1] = np.nan
    x[5, 0] = np.nan            # learned from the teacher
    values[6] = -np.inf         # from a teacher without probability
    x[6, n - 1] = np.inf
    x[7, n // 3] = np.nan       # from the label
    ids[7] = -1
    labels[7] = 2
    labels[8] = 0               # 8 to 11: finite
    ids[9] = -1
    labels[9] = n - 1
    x[10, 1:] = -np.inf
    rows = Rows(x, kind)
    listed = ((ids >= 0) & (ids < n)).any(1) if soft else np.zeros(12, bool)
    term = listed | ((labels >= 0) & (labels < n) if hard else False)
    spoilt = (np.isnan(rows.x) | np.isposinf(rows.x)).any(1)
    clean = np.where(spoilt[:, None], 0.0, rows.x)
    loss, lerr, delta, derr = ref.distill(clean, ids, values, labels, None, 1.0,
                                          mode == DISTILL_TAIL, soft, hard, kind)
    loss, delta = np.where(term, loss, 0), np.where(term[:, None], delta, 0)
    loss, delta = (np.where(term & spoilt, np.nan, loss),
                   np.where((term & spoilt)[:, None], np.nan, delta))
    d = Distill(gpu, rows, ids, values, labels, None, 1.0, mode, soft, hard)
    d.call()
    got, out = d.loss.numpy(), d.out.read()
    near(got, (loss, lerr), "loss")
    near(out, (delta, derr), "delta")
    assert not got[~term].any() and not out[~term].any()
    assert np.isnan(d.cost.numpy()[0])
    weights = np.where(term & spoilt, 0.0, 1.0)  # without these rows the sum is a number
    e = Distill(gpu, rows, ids, values, labels, weights, 1.0, mode, soft, hard)
    e.call()
    loss = np.where(weights == 0, 0, loss)
    near(e.loss.numpy(), (loss, lerr), "loss")
    near(e.cost.numpy()[0], (loss.sum(), lerr.sum() + 2 * ref.U * np.abs(loss).sum()), "cost")
    assert np.isfinite(e.out.read()).all()
