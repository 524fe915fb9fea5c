"""The weight gradient from a checkpoint where deltas are small or large."""
import numpy as np
import pytest

from aetcnn import BF16, F16, F32
from norm_ref import U
from test_gpu_checkpoint import Weights, activations
from test_gpu_logits import Rows

pytestmark = pytest.mark.gpu


def check_weights(w, lost=0.0):
    """against exact products and at most as many additions as rows, each off by a
    whole step (norm_ref.weights); `lost`: of a delta, in its place"""
    d, x = w.delta.x, w.k.values
    want, size = d.T @ x, np.abs(d).T @ np.abs(x)
    bound = 2 * (len(d) + 16) * U * size + lost * np.abs(x).sum(0)
    over = np.abs(w.read().astype(np.float64) - want) - bound
    assert over.max() <= 0, (np.unravel_index(over.argmax(), over.shape), (over + bound).max() / size.max())


SMALL = [(F32, e) for e in (-95, -105, -115, -122, -128, -136, -143)] + [
    (BF16, e) for e in (-105, -122, -126, -129, -133)] + [(F16, e) for e in (-12, -15, -20, -24)]


@pytest.mark.parametrize("rows,inputs,outputs", [(40, 96, 70), (700, 200, 300)])
@pytest.mark.parametrize("kind,e", SMALL)
def test_small_deltas(gpu, kind, e, rows, inputs, outputs):
    """to the last bit of the smallest"""
    rng = np.random.default_rng(-e)
    d = Rows(np.ldexp(rng.standard_normal((rows, outputs)), e), kind)
    assert np.abs(d.x).max() > 0
    w = Weights(gpu, d, np.ldexp(activations(rng, rows, inputs), 60))
    w.call()
    check_weights(w)


@pytest.mark.parametrize("rows,inputs,outputs", [(40, 96, 70), (700, 200, 300)])
@pytest.mark.parametrize("kind,e,ex", [
    (F32, 95, 0), (F32, 103, -40), (F32, 104, -40), (F32, 110, -3), (F32, 119, -30), (F32, 124, -126),
    (F32, 30, 76), (F32, 0, 113), (F32, -110, 120), (BF16, 105, -3), (BF16, 124, -126), (BF16, 0, 113)])
def test_large_deltas(gpu, kind, e, ex, rows, inputs, outputs):
    """deltas, or sums, up to near the largest float"""
    rng = np.random.default_rng(abs(e) + 2)
    d = Rows(np.ldexp(np.clip(rng.standard_normal((rows, outputs)), -3, 3), e), kind)
    x = rng.standard_normal((rows, inputs)) if ex > -100 else 1 + np.abs(rng.standard_normal((rows, inputs)))
    w = Weights(gpu, d, np.ldexp(np.clip(x, -4, 4), ex))
    assert np.abs(d.x.T @ w.k.values).max() < 2.0 ** 127
    w.call()
    check_weights(w)


def test_small_deltas_beside_large(gpu):
    """in tiles of their own the small ones keep their last bits, in a tile of the
    large ones all but those below 2^-133, bf16's smallest number"""
    rng = np.random.default_rng(3)
    for outputs, lost in ((600, 0.0), (30, 2.0 ** -133)):
        d = np.ldexp(rng.standard_normal((64, outputs)), -115)
        far = slice(0, outputs // 2)
        d[:, far] = np.ldexp(d[:, far], 225)
        w = Weights(gpu, Rows(d, F32), np.ldexp(activations(rng, 64, 150), -3))
        w.call()
        check_weights(w, lost)


def test_large_deltas_in_one_slice(gpu):
    """rows in slices, of which one sums up the large ones"""
    rng = np.random.default_rng(4)
    d = np.ldexp(rng.standard_normal((5000, 70)), -60)
    d[4100, 3], d[2, 9] = np.ldexp(1.0, 120), -np.ldexp(1.0, 126)
    w = Weights(gpu, Rows(d, F32), np.ldexp(activations(rng, 5000, 90), -20), accumulate=1)
    w.acc = 1
    assert w.nb
    w.call()
    want, size = w.delta.x.T @ w.k.values + w.old, np.abs(w.delta.x).T @ np.abs(w.k.values) + np.abs(w.old)
    assert (np.abs(w.read() - want) <= 2 * (4096 + 16) * U * size).all()


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("sign", [1, 0])
def test_one_long_chain(gpu, kind, sign):
    """so many tiles that one workgroup sums up all rows: every product one after
    the other, of both signs or of one, where all roundings go one way"""
    rng = np.random.default_rng(14)
    rows, inputs, outputs = 6000, 4127, 2101
    x, d = activations(rng, rows, inputs), rng.standard_normal((rows, outputs))
    if not sign:
        x, d = np.abs(x), np.abs(d)
    w = Weights(gpu, Rows(d, kind), x)
    assert w.nb == 0
    w.call()
    some = rng.choice(outputs, 40, replace=False)
    some[:2] = 0, outputs - 1
    dx = w.delta.x[:, some]
    want, size = dx.T @ w.k.values, np.abs(dx).T @ np.abs(w.k.values)
    off = np.abs(w.read()[some].astype(np.float64) - want)
    assert (off <= 2 * (rows + 16) * U * size).all(), (off / size).max() / U
