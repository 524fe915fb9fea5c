"""Layer norm layers, and batch-norm layers whose pre-norm tensor is kept in 8
bits, in a network's training step (an_add_layernorm, an_set_checkpoints)."""
import ctypes as C

import numpy as np
import pytest

import aetcnn
import norm_ref as ref
from aetcnn import F32, LEAKY, LINEAR, LOGISTIC, RELU, check, configs
from aetcnn import DeviceArray as D

pytestmark = pytest.mark.gpu
B = 6


def build(seed=1, on=False, sub=1, options=None, decay=0.0):
    """convolution with batch norm, layer norm over its planes, a connected layer,
    layer norm with dropout behind it, a connected layer, softmax"""
    aetcnn.net_lib().an_rand_seed(seed)
    net = aetcnn.Network(B, 9, 7, 3)
    if on:
        net.checkpoints()
    net.subdivisions(sub)
    net.hyper(0.05, 0.9, decay)
    net.conv(5, 3, 1, 1, LEAKY, 1)
    net.layernorm(1e-5)
    net.connected(40, LINEAR, 0)
    net.layernorm(1e-3)
    net.dropout(0.25)
    net.connected(10, LINEAR, 0)
    net.softmax()
    for i, o in (options or {}).items():
        net.set_layer_options(i, **o)
    net.finalize()
    return net


def batch(seed, n=B, classes=10, size=9 * 7 * 3):
    rng = np.random.default_rng(seed)
    t = np.zeros((n, classes), np.float32)
    t[np.arange(n), rng.integers(0, classes, n)] = 1
    return rng.standard_normal((n, size)).astype(np.float32), t


def perturb(net, layers=(1, 3)):
    """scales and biases of the layer norms away from 1 and 0"""
    rng = np.random.default_rng(4)
    for i in layers:
        n = net.buffer(i, 6).size
        net.set_buffer(i, 6, rng.standard_normal(n) * 0.3 + 1)
        net.set_buffer(i, 4, rng.standard_normal(n) * 0.3)


def near(got, want, name):
    value, bound = want
    over = np.abs(got.astype(np.float64).reshape(value.shape) - value) - bound
    assert over.max() <= 0, (name, over.max())


def test_layer_against_its_formula(gpu):
    net = build()
    perturb(net)
    x, t = batch(3)
    net.set_input(x, t)
    net.forward(1)
    for i, eps in ((1, 1e-5), (3, 1e-3)):
        inp = net.buffer(i - 1, 0).reshape(B, -1).astype(np.float64)
        s, b = net.buffer(i, 6), net.buffer(i, 4)
        want = ref.forward(inp, s, b, eps, F32)
        st = net.buffer(i, 16).reshape(B, 2)
        near(st[:, 0], want["mean"], "mean")
        near(st[:, 1], want["rstd"], "rstd")
        if i == 1:  # (the other's output is masked by the dropout behind it)
            near(net.buffer(i, 0), want["y"], "y")
    net.backward()
    for i in (3, 1):
        inp = net.buffer(i - 1, 0).reshape(B, -1).astype(np.float64)
        st = net.buffer(i, 16).reshape(B, 2).astype(np.float64)
        xn = (inp - st[:, :1]) * st[:, 1:]
        d = net.buffer(i, 1).reshape(B, -1).astype(np.float64)
        want = ref.backward(d, xn, 3 * ref.U * np.abs(xn), st[:, 1], net.buffer(i, 6), F32)
        near(net.buffer(i, 7), want["scales"], "scale_updates")
        near(net.buffer(i, 5), want["biases"], "bias_updates")
        if i == 3:  # the connected layer below is linear: its delta stays as written
            near(net.buffer(i - 1, 1), want["dx"], "dx")
    net.close()


def test_gradients_against_differences(gpu):
    """of the loss, by scales and biases of both layer norms (dropout off: a
    difference changes no mask, but its forward's are drawn by step)"""
    def run(grad):
        net = build(seed=2)
        perturb(net)
        if grad is not None:
            i, which, j, h = grad
            v = net.buffer(i, which)
            v[j] += h
            net.set_buffer(i, which, v)
        x, t = batch(5)
        net.set_input(x, t)
        net.forward(1)
        p = net.buffer(6, 0).reshape(B, -1).astype(np.float64)
        loss = -np.log((p * t).sum(1)).sum()
        net.backward()
        ups = {(i, w): net.buffer(i, w) for i in (1, 3) for w in (5, 7)}
        net.close()
        return loss, ups
    _, ups = run(None)
    h = 0.02
    for i, which in ((1, 6), (1, 4), (3, 6), (3, 4)):
        g = ups[i, which + 1]
        j = int(np.abs(g).argmax())
        up, down = run((i, which, j, h))[0], run((i, which, j, -h))[0]
        want = -(up - down) / (2 * h)  # the updates hold the negative gradient
        assert abs(g[j] - want) <= 0.02 * abs(want) + 2e-3, (i, which, g[j], want)


def steps(net, n, seed=7):
    for k in range(n):
        x, t = batch(seed + k)
        net.train(x, t)
    return [net.buffer(i, w) for i in range(net.n_layers()) for w in (2, 3, 4, 5, 6, 7)]


def test_update_forms_agree(gpu):
    """the update that the backward enqueues, layer by layer (an option of one
    layer that changes nothing) and flat after the loops: the same bits"""
    early, by_layer = build(decay=0.01), build(decay=0.01, options={0: dict(stopbackward=2)})
    a, b = steps(early, 1), steps(by_layer, 1)
    i = [k for k in range(len(a)) if k // 6 >= 1]  # the first layer's backward is skipped
    for k in i:
        assert (a[k] is None) == (b[k] is None)
        if a[k] is not None:
            assert np.array_equal(a[k], b[k]), (k // 6, k % 6)
    flat = build(decay=0.01)
    x, t = batch(7)
    flat.set_input(x, t)
    flat.forward(1)
    flat.backward()
    flat.update()
    for k in range(flat.n_layers() * 6):
        v = flat.buffer(k // 6, k % 6 + 2)
        if v is not None:
            assert np.array_equal(a[k], v), (k // 6, k % 6)
    for net in (early, by_layer, flat):
        net.close()


def test_frozen_and_scaled_rates(gpu):
    net = build(options={1: dict(learning_rate_scale=0.0)})
    before = net.buffer(1, 6).copy()
    top = net.buffer(3, 6).copy()
    steps(net, 2)
    assert np.array_equal(net.buffer(1, 6), before)
    assert not np.array_equal(net.buffer(3, 6), top)
    net.close()
    net = build(options={2: dict(stopbackward=1)})  # freezes the layers below
    before = net.buffer(1, 6).copy()
    steps(net, 2)
    assert np.array_equal(net.buffer(1, 6), before)
    assert not net.buffer(1, 7).any()
    net.close()


def test_subdivisions_add_up(gpu):
    """two minibatches before an update: their gradients' sum"""
    net = build(sub=2)
    (x0, t0), (x1, t1) = batch(21), batch(22)
    net.set_input(x0, t0)
    net.train_step()
    one = net.buffer(3, 5).copy()
    assert one.any()
    net.set_input(x1, t1)
    net.forward(1)
    net.backward()
    both = net.buffer(3, 5)
    d = net.buffer(3, 1).reshape(B, -1).astype(np.float64).sum(0)
    assert np.allclose(both, one + d, rtol=1e-5, atol=1e-6)
    net.close()


def test_weights_file(gpu, tmp_path):
    a, b = build(seed=1), build(seed=9)
    perturb(a)
    path = str(tmp_path / "a.weights")
    a.save_weights(path)
    b.load_weights(path)
    for i in range(a.n_layers()):
        for w in (2, 4, 6, 8, 9):
            u, v = a.buffer(i, w), b.buffer(i, w)
            assert (u is None) == (v is None)
            if u is not None:
                assert np.array_equal(u, v), (i, w)
    n = sum(a.buffer(i, w).size for i in range(a.n_layers()) for w in (2, 4, 6, 8, 9)
            if a.buffer(i, w) is not None)
    assert (tmp_path / "a.weights").stat().st_size == 20 + 4 * n
    x, _ = batch(1)
    assert np.array_equal(a.predict(x), b.predict(x))
    a.close()
    b.close()


def test_first_layer(gpu):
    """no delta below it"""
    aetcnn.net_lib().an_rand_seed(1)
    net = aetcnn.Network(B, 9, 7, 3)
    net.hyper(0.1, 0.9, 0.0)
    net.layernorm()
    net.connected(10, LINEAR, 0)
    net.softmax()
    net.finalize()
    x, t = batch(2)
    losses = [net.train(x, t) for _ in range(3)]
    assert np.isfinite(losses).all() and not np.array_equal(net.buffer(0, 6), np.ones(9 * 7 * 3))
    net.close()


# ---- checkpoints ----------------------------------------------------------------
def bn_net(on, act=LEAKY, batchsize=4, dropout=False):
    aetcnn.net_lib().an_rand_seed(3)
    net = aetcnn.Network(batchsize, 12, 10, 3)
    net.checkpoints(on)
    net.hyper(0.01, 0.9, 1e-4)
    net.conv(16, 3, 1, 1, act, 1)
    net.conv(24, 3, 2, 1, act, 1)
    if dropout:
        net.dropout(0.3)
    net.connected(32, act, 1)
    net.connected(10, LINEAR, 0)
    net.softmax()
    net.finalize()
    return net


def bn_layers(net):
    return [i for i in range(net.n_layers()) if net.buffer(i, 8) is not None]


@pytest.mark.parametrize("act", [LEAKY, RELU, LINEAR, LOGISTIC])
@pytest.mark.parametrize("dropout", [False, True])
def test_backward_from_the_kept_values(gpu, act, dropout):
    """the forward is the same bit for bit; what is kept are the definition's codes
    of the pre-norm tensor; the backward is ach_bn_bwd on their values, with the
    activation's gradient from the output"""
    plain, net = bn_net(False, act, dropout=dropout), bn_net(True, act, dropout=dropout)
    x, t = batch(11, 4, size=12 * 10 * 3)
    for n in (plain, net):
        n.set_input(x, t)
        n.forward(1)
    for i in range(net.n_layers()):
        for w in (0, 10, 11, 8, 9):
            u, v = plain.buffer(i, w), net.buffer(i, w)
            assert (u is None) == (v is None)
            if u is not None:
                assert np.array_equal(u, v), (i, w)
    assert len(bn_layers(net)) == 3
    for i in reversed(range(net.n_layers())):
        if i not in bn_layers(net):
            net.layer_backward(i)
            continue
        xs = plain.buffer(i, 12).reshape(4, -1)
        codes, st = ref.pack(xs.astype(np.float64))
        assert np.array_equal(net.buffer(i, 17), ref.buffer(codes, st))
        assert net.buffer(i, 12) is None
        v = ref.values(codes, st, xs.shape[1]).astype(np.float32)
        _, c, h, w = net.shape(i)[:4]
        delta, dx, dv, dy = (D.from_numpy(a) for a in (net.buffer(i, 1), v, net.buffer(i, 0),
                                                       net.buffer(i, 7)))
        par = [D.from_numpy(net.buffer(i, k)) for k in (10, 11, 6, 4)]
        nb = gpu.ach_bn_workspace(4, c, h * w)
        ws = D(max(nb, 16), np.uint8)
        check(gpu.ach_gradient(dv.ptr, v.size, act, delta.ptr, None))
        check(gpu.ach_bn_bwd(delta.ptr, 4, c, h * w, dx.ptr, None, par[0].ptr, par[1].ptr, par[2].ptr,
                             par[3].ptr, dy.ptr, None, None, LINEAR, ws.ptr, nb, None))
        net.layer_backward(i)
        assert np.array_equal(net.buffer(i, 1), delta.numpy()), i
        assert np.array_equal(net.buffer(i, 7), dy.numpy()), i
    plain.close()
    net.close()


def test_less_memory(gpu):
    plain, net = bn_net(False, batchsize=64), bn_net(True, batchsize=64)
    n = [64 * np.prod(net.shape(i)[1:4]) for i in bn_layers(net)]
    saved = plain.device_bytes() - net.device_bytes()
    assert saved >= sum(4 * v for v in n) - max(n) * 4 - sum(v * 33 / 32 for v in n) - 4096 * len(n)
    assert saved > 0
    plain.close()
    net.close()


def test_training_with_checkpoints(gpu):
    """steps run, inference between them is as ever, folded layers too"""
    plain, net = bn_net(False), bn_net(True)
    x, t = batch(12, 4, size=12 * 10 * 3)
    assert np.array_equal(plain.predict(x), net.predict(x))
    for k in range(4):
        xk, tk = batch(30 + k, 4, size=12 * 10 * 3)
        a, b = plain.train(xk, tk), net.train(xk, tk)
        assert np.isfinite(b)
        if k == 0:
            assert a == b
        net.predict(x)
    first = net.predict(x)
    net.fuse_conv_batchnorm()
    assert np.allclose(net.predict(x), first, rtol=1e-3, atol=1e-4)
    plain.close()
    net.close()


def test_a_nan_is_found(gpu):
    net = bn_net(True)
    x, t = batch(13, 4, size=12 * 10 * 3)
    x[1, 5] = np.nan
    net.set_input(x, t)
    net.train_step()
    assert net.nan_status() is not None
    with pytest.raises(aetcnn.HipError):
        net.loss()
    net.close()


@pytest.mark.parametrize("name", ["tiny", "darknet"])
def test_configurations(gpu, name):
    """the repository's networks with and without, one step"""
    nets = []
    for on in (False, True):
        aetcnn.net_lib().an_rand_seed(1)
        net = aetcnn.Network(*configs.dims(name, 4))
        net.checkpoints(on)
        configs.build(net, name)
        net.finalize()
        nets.append(net)
    x, t, _ = configs.synthetic_batch(name, 5, 4)
    a, b = (n.train(x, t) for n in nets)
    assert a == b  # the first step's loss is the forward's
    assert nets[1].device_bytes() < nets[0].device_bytes()
    for n in nets:
        n.close()
