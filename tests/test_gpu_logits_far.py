"""Logits whose difference is beyond the largest number of 32 bits while their
log probabilities, at a high temperature, are not."""
import numpy as np
import pytest

import logits_ref as ref
from aetcnn import BF16, F32, DISTILL_RENORM, DISTILL_TAIL
from test_gpu_logits import Distill, Forward, Rows, near, sample

pytestmark = pytest.mark.gpu

U = ref.U
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


def row_in_64_bits(x, ids, values, label, t, tail, soft, hard):
    """loss, delta and their bounds; logarithms of sums relative to their own
    largest term, so that no gap makes a probability 0 where it is not.  The
    loss is a sum of terms each of which is formed with 8 roundings or fewer,
    the exponentials and their sums have the errors that logits_ref.py counts, d."""
    d = (5 * 60 + 2 * len(x) / 64 + 48) * U
    member = np.zeros(len(x), bool)
    member[ids] = True
    p = np.zeros(len(x))
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        v = values if tail else (values - values.max()) / t
        p[ids] = np.exp(v) if tail else np.exp(v) / np.exp(v).sum()

        def softmax(y, scale, keep):
            m = y[keep].max()
            e = np.where(keep, np.exp((y - m) / scale), 0)
            return m, e / e.sum(), np.log(e.sum())

        every = np.ones(len(x), bool)
        m, q, lse = softmax(x, t, every)
        use = p > 0
        terms = p[use] * (np.log(p[use]) - ((x[use] - m) / t - lse))
        size, P, out, rest = np.abs(terms).sum() + lse, p.sum(), 0.0, 0.0
        kd = terms.sum()
        if tail:
            rest = 1 - P
            mr, out, lser = softmax(x, t, ~member)
            kd += rest * (np.log(rest) - ((mr - m) / t + lser - lse))
            size += rest * (abs(np.log(rest)) + abs(mr - m) / t + lser + lse)
            P = 1.0
        m1, q1, lse1 = softmax(x, 1.0, every)
        loss = soft * t * t * kd + hard * (lse1 - (x[label] - m1))
        lerr = 16 * U * (soft * t * t * size + hard * (lse1 + np.abs(x[label] - m1))) + \
            d * (2 * soft * t * t + hard)
    y = np.arange(len(x)) == label
    delta = -(soft * t * (P * q - p - rest * out) + hard * (q1 - y))
    derr = 2 * d * (soft * t * (P * q + p + rest * out) + hard * (q1 + y))
    return loss, lerr, delta, derr


@pytest.mark.parametrize("n", [300, 131072])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("t,soft", [(4.0, 2.0 ** -6), (1000.0, 2.0 ** -20)])
@pytest.mark.parametrize("mode", [DISTILL_RENORM, DISTILL_TAIL])
@pytest.mark.parametrize("hard", [0.0, 2.0 ** -3])
def test_distillation(gpu, n, kind, t, soft, mode, hard):
    """Losses of some 1e37 are numbers.  0: a listed class far below the best;
    1: the label; 2: all that the teacher does not list.  3: an entry of little
    probability that the student has masked makes the loss +inf, though in 32
    bits its probability next to the others, which another wave holds, is 0.
    4: logits of the teacher at both ends of the type."""
    rng = np.random.default_rng(n)
    k, tail = 100, mode == DISTILL_TAIL
    x = sample(rng, 5, n)
    ids = np.stack([rng.permutation(n)[:k] for _ in range(5)])
    values = np.log(rng.dirichlet(np.ones(k), 5) * 0.5)
    x[0, ids[0, 0]], x[0, ids[0, 1]] = BIG, -BIG
    values[0, 1] = np.log(0.25)
    labels = ids[:, 2].copy()
    x[1, labels[1]], x[1, ids[1, 3]] = -BIG, BIG
    values[1, 2] = -np.inf
    x[2] = -BIG
    x[2, ids[2]] = BIG
    values[3, 64:] = values[3, :64].max() - 120 * (1 if tail else t)
    x[3, ids[3, 70]] = -np.inf
    values[4, :64], values[4, 64:] = 3e38, -3e38
    weights = np.ones(5)
    if tail:
        weights[4] = 0  # no log probabilities
    rows = Rows(x, kind)
    d = Distill(gpu, rows, ids, values, labels, weights, t, mode, soft, hard)
    d.call()
    loss, delta = d.loss.numpy(), d.out.read()
    for r in range(5):
        if weights[r] == 0:
            assert loss[r] == 0 and not delta[r].any()
            continue
        want, lerr, grad, derr = row_in_64_bits(rows.x[r], ids[r], d.h_values[r], labels[r], t, tail,
                                                soft, hard)
        assert np.isposinf(want) if r == 3 else abs(want) < 3e38
        assert r > (2 if tail else 0) or want > 1e33
        near(loss[r], (want, 2 * U * abs(want) + lerr), "loss")
        near(delta[r], (grad, derr + ref.half_step(grad, kind)), "delta")
    if not tail:
        assert np.isfinite(delta).all()
