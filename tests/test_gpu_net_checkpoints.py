"""Which batch-norm layers keep their pre-norm tensor in 8 bits, and what that
takes (an_set_checkpoints)."""
import numpy as np
import pytest

import aetcnn
import norm_ref as ref
from aetcnn import ACH_EUNSUPPORTED, LEAKY, LINEAR
from test_gpu_net_norm import batch

pytestmark = pytest.mark.gpu
B, SIZES = 4, (16 * 12 * 10, 24 * 6 * 5, 32)


def build(on, options=None):
    aetcnn.net_lib().an_rand_seed(3)
    net = aetcnn.Network(B, 12, 10, 3)
    net.checkpoints(on)
    net.hyper(0.01, 0.9, 1e-4)
    net.conv(16, 3, 1, 1, LEAKY, 1)
    net.conv(24, 3, 2, 1, LEAKY, 1)
    net.connected(32, LEAKY, 1)
    net.connected(10, LINEAR, 0)
    net.softmax()
    for i, o in (options or {}).items():
        net.set_layer_options(i, **o)
    net.finalize()
    return net


def kept_bytes(n):
    return aetcnn.ops().ach_checkpoint_bytes(B, n)


@pytest.mark.parametrize("options,reached", [
    ({}, [0, 1, 2]), ({1: dict(stopbackward=1)}, [2]), ({0: dict(stopbackward=2)}, [1, 2]),
    ({4: dict(stopbackward=1)}, []), ({1: dict(onlyforward=1)}, [0, 2])])
def test_layers_without_a_backward_keep_nothing(gpu, options, reached):
    everything, net = build(True), build(True, options)
    assert [i for i in range(3) if net.buffer(i, 17) is not None] == reached
    assert all(net.buffer(i, 12) is None for i in range(3))  # one buffer of all of them
    less = sum(kept_bytes(n) for i, n in enumerate(SIZES) if i not in reached)
    assert abs(everything.device_bytes() - net.device_bytes() - less) <= 3 * 256
    everything.close()
    # what is trained is the same as in 32 bits but for the rounding: the first
    # step's loss, and the parameters of the layers that are not
    plain = build(False, options)
    x, t = batch(11, B, size=12 * 10 * 3)
    for k in range(2):
        a, b = plain.train(x, t), net.train(x, t)
        assert np.isfinite(b) and (k or a == b)
    for i in range(3):
        if i not in reached:
            assert np.array_equal(net.buffer(i, 7), plain.buffer(i, 7))
            with pytest.raises(aetcnn.HipError) as e:
                net.layer_backward(i)
            assert str(ACH_EUNSUPPORTED) in str(e.value)
        plain.layer_backward(i)
    net.train(x, t)  # the refusal changed nothing
    plain.close()
    net.close()


@pytest.mark.parametrize("widths", [(16,), (64, 8), (8, 64, 8), (16, 16, 16)])
def test_never_more_memory(gpu, widths):
    """a shared buffer beside one large layer's codes would be more than its
    tensor: it stays in 32 bits, and training as it is"""
    def small(on):
        aetcnn.net_lib().an_rand_seed(5)
        net = aetcnn.Network(B, 12, 10, 3)
        net.checkpoints(on)
        net.hyper(0.01, 0.9, 1e-4)
        for w in widths:
            net.conv(w, 3, 1, 1, LEAKY, 1)
        net.connected(10, LINEAR, 0)
        net.softmax()
        net.finalize()
        return net
    plain, net = small(False), small(True)
    sizes = [w * 120 for w in widths]
    kept = sum(kept_bytes(n) for n in sizes) + max(sizes) * 4 * B < sum(sizes) * 4 * B
    assert (net.device_bytes() < plain.device_bytes()) == kept and net.device_bytes() <= plain.device_bytes()
    for i in range(len(widths)):
        assert (net.buffer(i, 17) is not None) == kept and (net.buffer(i, 12) is None) == kept
    for k in range(2):
        x, t = batch(40 + k, B, size=12 * 10 * 3)
        assert kept or plain.train(x, t) == net.train(x, t)
    if not kept:
        for i in range(net.n_layers()):
            for which in (2, 4, 6):
                u = plain.buffer(i, which)
                assert u is None or np.array_equal(u, net.buffer(i, which))
    plain.close()
    net.close()


def one_channel_each(on, c, h, w):
    """a first layer whose x is the network's input, and another of its size"""
    aetcnn.net_lib().an_rand_seed(5)
    net = aetcnn.Network(16, h, w, c)
    net.checkpoints(on)
    net.conv(c, 1, 1, 0, LINEAR, 1)
    net.conv(c, 1, 1, 0, LINEAR, 1)
    net.connected(10, LINEAR, 0)
    net.softmax()
    net.finalize()
    net.set_buffer(0, 2, np.eye(c))
    return net


@pytest.mark.parametrize("c,h,w", [(12, 8, 8), (20, 7, 5), (96, 1, 1)])
@pytest.mark.parametrize("mean", [0, 3, 10, 30])
@pytest.mark.parametrize("spread", [1, 30])
def test_how_far_gradients_move(gpu, c, h, w, mean, spread):
    """from those of unrounded values, for channels `mean` deviations away from 0,
    every second one of them `spread` times the others.

    x_norm is off by e, at most half a step times the reciprocal deviation.  With
    g = delta*scales, dx = rstd*(g - mean g - x_norm*mean(g x_norm)) moves by at most
    rstd*(e |mean(g x_norm)| + (|x_norm| + e) mean |g e|), the scales' updates by sum
    |delta e|; the two passes in 32 bits are off by less than 2^-15 of the terms."""
    rng = np.random.default_rng(mean + c)
    size = np.where(np.arange(c) % 2, spread, 1.0)[:, None, None]
    x = ((rng.standard_normal((16, c, h, w)) + mean) * size).astype(np.float32)
    t = np.eye(10, dtype=np.float32)[rng.integers(0, 10, 16)]
    delta = rng.standard_normal(x.shape).astype(np.float32)
    s = rng.standard_normal(c).astype(np.float32)

    def backward(on):
        net = one_channel_each(on, c, h, w)
        net.set_input(x.reshape(16, -1), t)
        net.forward(1)
        for which, values in ((6, s), (1, delta)):
            net.set_buffer(0, which, values)
        before = {which: net.buffer(0, which) for which in (10, 11, 12, 17)}
        net.layer_backward(0)
        after = net.buffer(0, 1).reshape(x.shape).astype(np.float64), net.buffer(0, 7).astype(np.float64)
        net.close()
        return before, after

    (state, plain), (kept, got) = backward(False), backward(True)
    assert np.array_equal(state[12], x.ravel())
    assert all(np.array_equal(state[which], kept[which]) for which in (10, 11))
    _, steps = ref.parts(kept[17], 16, c * h * w)
    m, v = state[10], state[11]
    ax = (0, 2, 3)
    m, rstd, s = (q.astype(np.float64)[:, None, None] for q in (m, 1 / np.sqrt(v.astype(np.float64)), s))
    half = np.repeat(np.ldexp(0.5, steps.astype(int) - 133), 32, axis=1)[:, :c * h * w].reshape(x.shape)
    e, xn, g = half * rstd, (x - m) * rstd, delta * s

    def over(q):
        return q.mean(ax)[:, None, None]

    gx, ge = np.abs(g * xn), np.abs(g) * e
    low = 2.0 ** -15
    bound = rstd * (e * np.abs(over(g * xn)) + (np.abs(xn) + e) * over(ge)
                    + low * (np.abs(g) + over(np.abs(g)) + np.abs(xn) * over(gx)))
    assert (np.abs(got[0] - plain[0]) <= bound).all()
    assert (np.abs(got[1] - plain[1]) <= (np.abs(delta) * (e + low * np.abs(xn))).sum(ax)).all()
    # a plane in blocks of its own: e is a share of the values, mean and deviations together
    if h * w % 32 == 0:
        assert (e <= (np.abs(xn).max((2, 3), keepdims=True) + mean + 1) / 127).all()
