"""Layer norm, checkpoints and the weight gradient from them without a GPU:
which calls are refused, before anything is launched, and the 64-bit forms that
the kernels are tested against, themselves against differences."""
import ctypes as C

import numpy as np
import pytest

import aetcnn
import norm_ref as ref
from aetcnn import ACH_EINVAL, ACH_EWORKSPACE, BF16, F16, F32
from aetcnn import CheckpointDesc, FcDesc, LayernormDesc

MEM = 4096  # an address that is never read: the calls are refused
BIG = 1 << 40


def at(d):
    return C.byref(d) if d else None


def fwd(ops, d, x=MEM, scales=MEM, biases=MEM, y=2 * MEM, stride=0, stats=MEM, kept=None, ws=MEM,
        nb=BIG):
    return ops.ach_layernorm_fwd(at(d), x, scales, biases, y, stride, stats, kept, ws, nb, None)


def bwd(ops, d, delta=MEM, d_stride=0, x=MEM, kept=None, stats=MEM, scales=MEM, dx=2 * MEM,
        dx_stride=0, ds=MEM, db=MEM, accumulate=0, ws=MEM, nb=BIG):
    return ops.ach_layernorm_bwd(at(d), delta, d_stride, x, kept, stats, scales, dx, dx_stride, ds,
                                 db, accumulate, ws, nb, None)


def fc(ops, d, kept=MEM, delta=MEM, dw=MEM, accumulate=0, ws=MEM, nb=BIG):
    return ops.ach_fc_bwd_filter_checkpoint(at(d), kept, delta, dw, accumulate, ws, nb, None)


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("d", [
    LayernormDesc(-1, 10, F32, 1e-5), LayernormDesc(2, 0, F32, 1e-5), LayernormDesc(2, -1, F32, 1e-5),
    LayernormDesc(2, (1 << 30) + 1, F32, 1e-5), LayernormDesc((1 << 30) + 1, 2, F32, 1e-5),
    LayernormDesc(2, 10, 3, 1e-5),
    LayernormDesc(2, 10, -1, 1e-5), LayernormDesc(2, 10, F32, 0.0), LayernormDesc(2, 10, F32, -1.0),
    LayernormDesc(2, 10, F32, 1e-13), LayernormDesc(2, 10, F32, 2.0), LayernormDesc(2, 10, F32, NAN),
    LayernormDesc(2, 10, F32, INF), LayernormDesc(2, 10, F32, 1e-5, 9),
    LayernormDesc(2, 10, F32, 1e-5, -10), None])
def test_bad_layernorm_descriptors(d):
    ops = aetcnn.ops()
    assert fwd(ops, d) == bwd(ops, d) == ACH_EINVAL
    assert ops.ach_layernorm_fwd_workspace(at(d)) == ops.ach_layernorm_bwd_workspace(at(d)) == 0


def test_layernorm_refusals():
    ops = aetcnn.ops()
    d, h = LayernormDesc(2, 10, F32, 1e-5, 12), LayernormDesc(2, 10, BF16, 1e-5)
    assert fwd(ops, d, x=None) == fwd(ops, d, x=MEM + 2) == fwd(ops, h, x=MEM + 1) == ACH_EINVAL
    assert fwd(ops, d, y=None, stats=None) == ACH_EINVAL            # nothing asked
    assert fwd(ops, d, y=MEM + 2) == fwd(ops, d, stride=9) == fwd(ops, d, stride=-1) == ACH_EINVAL
    assert fwd(ops, d, y=MEM) == fwd(ops, d, y=MEM, stride=10) == ACH_EINVAL  # in place, restrided
    assert fwd(ops, d, kept=MEM + 8) == fwd(ops, d, stats=MEM + 2) == ACH_EINVAL
    assert fwd(ops, d, scales=MEM + 1) == fwd(ops, d, biases=MEM + 1) == ACH_EINVAL
    few = LayernormDesc(1, 1 << 20, F32, 1e-5)
    nb = ops.ach_layernorm_fwd_workspace(at(few))
    if nb:
        assert fwd(ops, few, ws=None) == fwd(ops, few, nb=nb - 1) == ACH_EWORKSPACE
        assert fwd(ops, few, ws=MEM + 4) == ACH_EWORKSPACE

    assert bwd(ops, d, delta=None) == bwd(ops, d, stats=None) == ACH_EINVAL
    assert bwd(ops, d, x=None) == bwd(ops, d, kept=MEM) == ACH_EINVAL  # neither, both
    assert bwd(ops, d, dx=None, ds=None, db=None) == ACH_EINVAL
    assert bwd(ops, d, accumulate=2) == bwd(ops, d, accumulate=-1) == ACH_EINVAL
    assert bwd(ops, d, d_stride=9) == bwd(ops, d, dx_stride=9) == bwd(ops, d, d_stride=-1) == ACH_EINVAL
    assert bwd(ops, d, dx=MEM, dx_stride=11) == ACH_EINVAL
    assert bwd(ops, d, delta=MEM + 2) == bwd(ops, d, x=MEM + 2) == bwd(ops, d, dx=MEM + 2) == ACH_EINVAL
    assert bwd(ops, d, x=None, kept=MEM + 4) == bwd(ops, d, stats=MEM + 1) == ACH_EINVAL
    assert bwd(ops, d, ds=MEM + 2) == bwd(ops, d, db=MEM + 2) == bwd(ops, d, scales=MEM + 2) == ACH_EINVAL
    nb = ops.ach_layernorm_bwd_workspace(at(d))
    assert nb > 0
    assert bwd(ops, d, ws=None) == bwd(ops, d, nb=nb - 1) == bwd(ops, d, ws=MEM + 8) == ACH_EWORKSPACE


@pytest.mark.parametrize("d", [
    CheckpointDesc(-1, 10, F32), CheckpointDesc(2, 0, F32), CheckpointDesc(2, (1 << 30) + 1, F32),
    CheckpointDesc((1 << 30) + 1, 2, F32),
    CheckpointDesc(2, 10, 3), CheckpointDesc(2, 10, -1), CheckpointDesc(2, 10, F32, 9),
    CheckpointDesc(2, 10, F32, -10), None])
def test_bad_checkpoint_descriptors(d):
    ops = aetcnn.ops()
    assert ops.ach_checkpoint_pack(at(d), MEM, 2 * MEM, None) == ACH_EINVAL
    assert ops.ach_checkpoint_unpack(at(d), MEM, 2 * MEM, None) == ACH_EINVAL


def test_checkpoint_refusals_and_sizes():
    ops = aetcnn.ops()
    d = CheckpointDesc(2, 10, F32)
    for call in (ops.ach_checkpoint_pack, ops.ach_checkpoint_unpack):
        assert call(at(d), None, MEM, None) == call(at(d), MEM, None, None) == ACH_EINVAL
    assert ops.ach_checkpoint_pack(at(d), MEM + 2, 2 * MEM, None) == ACH_EINVAL
    assert ops.ach_checkpoint_pack(at(d), MEM, 2 * MEM + 8, None) == ACH_EINVAL
    assert ops.ach_checkpoint_unpack(at(d), MEM + 8, 2 * MEM, None) == ACH_EINVAL
    assert ops.ach_checkpoint_pack(at(CheckpointDesc(0, 10, F32)), MEM, 2 * MEM, None) == 0  # no rows
    size = ops.ach_checkpoint_bytes
    assert size(3, 1) == size(3, 32) == 3 * 33 and size(3, 33) == 3 * 66 and size(0, 5) == 0
    assert size(-1, 5) == size(1, 0) == size(1, -4) == size(1, (1 << 30) + 1) == size((1 << 30) + 1, 1) == 0
    assert size(100000, 1 << 30) == 100000 * (1 << 30) // 32 * 33  # past 32 bits


@pytest.mark.parametrize("d", [
    FcDesc(-1, 10, 10, F32), FcDesc(2, 0, 10, F32), FcDesc(2, 10, 0, F32), FcDesc(2, 10, 10, 3),
    FcDesc(2, 10, 10, -1), FcDesc(2, 10, 10, F32, 9), FcDesc(2, 10, 10, F32, -10),
    FcDesc(2, (1 << 23) + 1, 10, F32), FcDesc((1 << 30) + 1, 10, 10, F32),
    FcDesc(2, 10, (1 << 23) + 1, F32), FcDesc(2, 10, 10, F32, (1 << 23) + 1), None])
def test_bad_fc_descriptors(d):
    ops = aetcnn.ops()
    assert fc(ops, d) == ACH_EINVAL
    assert ops.ach_fc_bwd_filter_checkpoint_workspace(at(d)) == 0


def test_fc_refusals():
    ops = aetcnn.ops()
    d = FcDesc(2, 10, 10, BF16)
    assert fc(ops, d, kept=None) == fc(ops, d, delta=None) == fc(ops, d, dw=None) == ACH_EINVAL
    assert fc(ops, d, kept=MEM + 8) == fc(ops, d, delta=MEM + 1) == fc(ops, d, dw=MEM + 2) == ACH_EINVAL
    assert fc(ops, d, accumulate=2) == ACH_EINVAL
    long = FcDesc(100000, 64, 64, F16)  # one tile: its rows are shared out
    nb = ops.ach_fc_bwd_filter_checkpoint_workspace(at(long))
    if nb:
        assert fc(ops, long, ws=None) == fc(ops, long, nb=nb - 1) == ACH_EWORKSPACE
        assert fc(ops, long, ws=MEM + 8) == ACH_EWORKSPACE


# ---- the 64-bit forms ---------------------------------------------------------
def differences(f, a, h=1e-5):
    g = np.zeros_like(a)
    for i in np.ndindex(a.shape):
        b = a.copy()
        b[i] += h
        up = f(b)
        b[i] -= 2 * h
        g[i] = (up - f(b)) / (2 * h)
    return g


def test_layernorm_gradients_against_differences():
    rng = np.random.default_rng(1)
    x, d = rng.standard_normal((3, 7)), rng.standard_normal((3, 7))
    s, b, eps = rng.standard_normal(7), rng.standard_normal(7), 1e-3

    def loss(x, s=s, b=b):
        return (ref.forward(x, s, b, eps, F32)["y"][0] * d).sum()

    f = ref.forward(x, s, b, eps, F32)
    got = ref.backward(d, f["x_norm"][0], 0.0, f["rstd"][0], s, F32)
    assert np.allclose(got["dx"][0], differences(loss, x), atol=1e-7)
    assert np.allclose(got["scales"][0], differences(lambda v: loss(x, v), s), atol=1e-7)
    assert np.allclose(got["biases"][0], differences(lambda v: loss(x, s, v), b), atol=1e-7)


def test_checkpoint_form():
    """its own words: the error is at most half a step, and a 127th of the largest
    magnitude; a step less would not hold that"""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((50, 100)) * 10.0 ** rng.integers(-30, 30, (50, 100))
    codes, steps = ref.pack(x)
    v = ref.values(codes, steps, 100)
    top = np.abs(np.pad(x, ((0, 0), (0, 28))).reshape(50, 4, 32)).max(2)
    off = np.abs(np.pad(v - x, ((0, 0), (0, 28))).reshape(50, 4, 32)).max(2)
    assert (off <= np.ldexp(1.0, steps.astype(int) - 134)).all()
    assert (off <= top / 127).all()
    assert (np.abs(codes).reshape(50, 4, 32).max(2) >= 64).all()
    edge = np.array([[127.0, 127.49, 127.5, 128.0]]).T  # alone in their blocks
    codes, steps = ref.pack(edge)
    assert list(steps[:, 0]) == [133, 133, 134, 134] and list(codes[:, 0]) == [127, 127, 64, 64]


# ---- in a network, before it is finalized ------------------------------------------
def test_network_refusals(tmp_path, capfd):
    lib = aetcnn.net_lib()
    h = lib.an_network_create(2, 4, 4, 3)
    for eps in (0.0, -1.0, 1e-13, 2.0, NAN, INF):
        assert lib.an_add_layernorm(h, eps) == ACH_EINVAL
    assert lib.an_add_layernorm(None, 1e-5) == ACH_EINVAL
    assert lib.an_add_layernorm(h, 1e-5) == 0
    assert lib.an_set_checkpoints(None, 1) == lib.an_set_checkpoints(h, 2) == ACH_EINVAL
    assert lib.an_set_checkpoints(h, 1) == lib.an_set_checkpoints(h, 0) == 0
    lib.an_free(h)
    cfg = tmp_path / "n.cfg"
    text = ("[net]\nbatch=4\nheight=6\nwidth=5\nchannels=3\nactivation_checkpoints={}\n"
            "[convolutional]\nfilters=8\nsize=3\npad=1\nbatch_normalize=1\nactivation=leaky\n"
            "[layernorm]\neps={}\nlearning_rate=2\n[connected]\noutput=7\nactivation=linear\n[layernorm]\n"
            "[softmax]\n")
    cfg.write_text(text.format(1, 0.001))
    net = aetcnn.Network.from_cfg(str(cfg), finalize=False)
    assert "unused" not in capfd.readouterr().err
    assert [net.shape(i)[:4] for i in range(5)] == [[0, 8, 6, 5], [5, 8, 6, 5], [0, 7, 1, 1],
                                                    [5, 7, 1, 1], [4, 7, 1, 1]]
    assert net.layer_options(1)["learning_rate_scale"] == 2.0
    net.close()
    for bad in (text.format(2, 0.001), text.format(0, 0)):
        cfg.write_text(bad)
        with pytest.raises(ValueError):
            aetcnn.Network.from_cfg(str(cfg), finalize=False)
