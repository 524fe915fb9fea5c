"""Which batch-norm layers keep their pre-norm tensor in 8 bits, and what that
takes (an_set_checkpoints)."""
import numpy as np
import pytest

import aetcnn
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
