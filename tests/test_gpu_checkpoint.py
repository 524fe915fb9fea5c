"""Activation checkpoints in 8 bits and a fully connected layer's weight
gradient from them, against their definitions in 64 bits (norm_ref.py): codes
and steps have to be equal."""
import ctypes as C

import numpy as np
import pytest

import aetcnn
import norm_ref as ref
from aetcnn import BF16, F16, F32, check
from aetcnn import DeviceArray as D
from test_gpu_logits import Hip, Rows, like

pytestmark = pytest.mark.gpu
GUARD = 64  # bytes behind a checkpoint that have to stay as they are


def activations(rng, rows, n):
    x = rng.standard_normal((rows, n)) * rng.exponential(1.0, n)
    x[:, rng.random(n) < 0.02] *= 50
    return x


class Kept:
    """A checkpoint's bytes on the device, and a pattern behind them."""

    def __init__(self, rows, n, raw=None):
        self.rows, self.n = rows, n
        self.nb = aetcnn.ops().ach_checkpoint_bytes(rows, n)
        assert self.nb == rows * ref.width(n) // 32 * 33
        host = np.full(self.nb + GUARD, 0x5a, np.uint8)
        if raw is not None:
            host[:self.nb] = raw
        self.dev = D.from_numpy(host)
        self.ptr = self.dev.ptr

    @classmethod
    def of(cls, x):
        k = cls(*x.shape, ref.buffer(*ref.pack(x)))
        k.values = ref.values(*ref.pack(x), x.shape[1])
        return k

    def read(self):
        raw = self.dev.numpy()
        assert (raw[self.nb:] == 0x5a).all(), "written behind the checkpoint"
        return ref.parts(raw[:self.nb], self.rows, self.n)


def pack(gpu, x, stream=None):
    k = Kept(x.rows, x.n)
    check(gpu.ach_checkpoint_pack(C.byref(aetcnn.CheckpointDesc(x.rows, x.n, x.kind, x.stride)),
                                  x.ptr, k.ptr, stream))
    return k


def unpack(gpu, k, kind, pad=0, shift=0):
    out = Rows(np.full((k.rows, k.n), np.nan), kind, pad, shift)
    check(gpu.ach_checkpoint_unpack(C.byref(aetcnn.CheckpointDesc(k.rows, k.n, kind, out.stride)),
                                    k.ptr, out.ptr, None))
    return out.read()


def check_pack(gpu, x):
    k = pack(gpu, x)
    codes, steps = k.read()
    want_codes, want_steps = ref.pack(x.x)
    assert np.array_equal(steps, want_steps)
    fine = np.repeat(want_steps != 255, 32, axis=1)
    assert np.array_equal(codes[fine], want_codes[fine])
    v = ref.values(want_codes, want_steps, x.n)
    for kind in (F32, BF16, F16):
        got = unpack(gpu, k, kind, pad=x.stride - x.n, shift=x.shift)
        most = ref.LARGEST[kind]
        want = ref.from_bits(ref.to_bits(np.clip(v, -most, most), kind), kind)
        assert np.array_equal(got, want, equal_nan=True), kind


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("rows,n,pad,shift", [
    (1, 1, 0, 0), (1, 31, 0, 1), (3, 32, 0, 0), (2, 33, 1, 0), (7, 63, 0, 3), (5, 100, 3, 1),
    (4, 1003, 5, 0), (300, 129, 0, 0), (2, 20000, 0, 1), (128, 4096, 0, 0), (5000, 7, 2, 1)])
def test_pack_and_unpack(gpu, rows, n, pad, shift, kind):
    rng = np.random.default_rng(rows * 1000 + n)
    check_pack(gpu, Rows(activations(rng, rows, n), kind, pad, shift))


@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_blocks_at_the_ends(gpu, kind):
    """zeros, both signs of them, values at a code's border, the smallest and the
    largest of the type, infinities and NaN: of each block's own alone"""
    rng = np.random.default_rng(5)
    most, tiny = ref.LARGEST[kind], {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}[kind]
    x = activations(rng, 40, 160)
    x[0] = 0
    x[1] = -0.0
    x[2, :32] = np.arange(32) * 8 - 120.5          # ties to even
    x[3, :32] = np.arange(32) + 96.5               # up to 127.5: the next step
    x[4, :32] = np.minimum(np.arange(32) + 96.5, 127)
    x[5] = tiny
    x[6, ::2] = tiny * 3
    x[7, ::3] = most
    x[8, ::5] = -most
    x[9, 40] = np.inf
    x[10, 70] = -np.inf
    x[11, [1, 159]] = np.nan
    x[12, 64:96] = np.nan
    x[13] = np.ldexp(1.0, np.arange(160) % 30 - 14)
    x[14, :64] *= 2.0 ** -120 if kind != F16 else 2.0 ** -20
    x[15, :64] *= 2.0 ** 120 if kind != F16 else 2.0 ** 8
    check_pack(gpu, Rows(x, kind))


def test_long_rows_and_many(gpu):
    """more chunks than a launch's grid has threads"""
    rng = np.random.default_rng(6)
    x = Rows(np.tile(activations(rng, 64, 4097), (160, 1)), BF16)
    codes, steps = pack(gpu, x).read()
    want = ref.pack(x.x[:64])
    assert np.array_equal(codes, np.tile(want[0], (160, 1)))
    assert np.array_equal(steps, np.tile(want[1], (160, 1)))


# ---- the weight gradient ---------------------------------------------------------
class Weights:
    def __init__(self, gpu, delta, x, accumulate=0, seed=0):
        """delta: Rows, x: [rows][inputs] before it is packed"""
        self.gpu, self.delta, self.acc = gpu, delta, accumulate
        self.k = Kept.of(x)
        self.desc = aetcnn.FcDesc(delta.rows, x.shape[1], delta.n, delta.kind, delta.stride)
        rng = np.random.default_rng(seed)
        self.old = rng.standard_normal((delta.n, x.shape[1])).astype(np.float32)
        self.dw = D((delta.n * x.shape[1] + 16,), np.float32)
        self.restart()
        self.nb = gpu.ach_fc_bwd_filter_checkpoint_workspace(C.byref(self.desc))
        self.ws = D(max(self.nb, 4), np.uint8)
        self.ws.upload(np.full(self.ws.shape, 0xff, np.uint8))

    def restart(self):
        self.dw.upload(np.concatenate([self.old.ravel(), np.full(16, 77, np.float32)]))

    def call(self, stream=None):
        check(self.gpu.ach_fc_bwd_filter_checkpoint(C.byref(self.desc), self.k.ptr, self.delta.ptr,
                                                    self.dw.ptr, self.acc, self.ws.ptr, self.nb,
                                                    stream))

    def read(self):
        v = self.dw.numpy()
        assert (v[-16:] == 77).all(), "written behind dw"
        return v[:-16].reshape(self.old.shape)

    def check(self):
        want, bound = ref.weights(self.delta.x, self.k.values)
        if self.acc:
            want = want + self.old
            bound = bound + ref.U * (np.abs(want) + np.abs(self.old))
        got = self.read().astype(np.float64)
        fin = np.isfinite(want)
        assert not np.isfinite(got[~fin]).any()
        off = np.abs(np.where(fin, got, 0) - np.where(fin, want, 0)) - np.where(fin, bound, 0)
        assert np.isfinite(off).all()
        assert off.max() <= 0, (np.unravel_index(off.argmax(), off.shape), off.max())


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("rows,inputs,outputs,pad,shift", [
    (1, 1, 1, 0, 0), (1, 40, 3, 0, 1), (50, 300, 7, 1, 0), (70, 31, 8, 0, 1), (40, 65, 263, 0, 1), (2, 33, 65, 1, 0), (15, 64, 64, 0, 0), (16, 100, 31, 0, 0),
    (17, 129, 127, 3, 1), (33, 31, 200, 0, 0), (64, 256, 128, 0, 0), (100, 1003, 77, 5, 3),
    (128, 512, 300, 0, 0), (130, 257, 1000, 0, 0), (1531, 203, 177, 2, 1), (5000, 70, 9, 0, 0),
    (9000, 32, 16, 0, 0)])
def test_weight_gradient(gpu, rows, inputs, outputs, pad, shift, kind):
    rng = np.random.default_rng(rows + inputs)
    d = Rows(rng.standard_normal((rows, outputs)) / rows * 64, kind, pad, shift)
    for accumulate in (0, 1):
        w = Weights(gpu, d, activations(rng, rows, inputs), accumulate)
        w.call()
        w.check()


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("rows,inputs,outputs,pad,shift", [
    (30, 4128, 2100, 0, 0), (30, 4101, 2101, 0, 0), (300, 4128, 2048, 0, 0), (270, 4128, 2101, 1, 1),
    (300, 90, 6, 0, 1), (2000, 300, 5, 1, 0), (700, 1003, 301, 0, 0), (1200, 2050, 520, 3, 0)])
def test_weight_gradient_by_tiles(gpu, rows, inputs, outputs, pad, shift, kind):
    """tiles of every kind, in slices and not, and dw of more than the caches"""
    rng = np.random.default_rng(rows + inputs)
    d = Rows(rng.standard_normal((rows, outputs)) / rows * 64, kind, pad, shift)
    w = Weights(gpu, d, activations(rng, rows, inputs), int(rows % 20 == 0))
    w.call()
    w.check()


@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_weight_gradient_of_far_magnitudes(gpu, kind):
    """deltas and activations from near the smallest to near the largest: each
    output's own size decides its error"""
    rng = np.random.default_rng(8)
    e = (-14, 15) if kind == F16 else (-60, 61)
    d = rng.standard_normal((150, 96)) * np.ldexp(1.0, rng.integers(*e, 96))
    x = rng.standard_normal((150, 320)) * np.repeat(np.ldexp(1.0, rng.integers(-60, 61, 10)), 32)
    w = Weights(gpu, Rows(d, kind), x)
    w.call()
    w.check()


@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_weight_gradient_of_what_is_not_finite(gpu, kind):
    """reaches what it is summed into, and nothing else"""
    rng = np.random.default_rng(9)
    d = rng.standard_normal((70, 130))
    x = activations(rng, 70, 200)
    d[3, 7], d[69, 129], d[20, 64] = np.nan, np.inf, -np.inf
    x[5, 100] = np.nan
    w = Weights(gpu, Rows(d, kind), x)
    w.call()
    got = w.read()
    bad = np.zeros_like(got, bool)
    bad[[7, 129, 64]] = True
    bad[:, 96:128] = True
    assert np.array_equal(~np.isfinite(got), bad)
    w.delta.x[[3, 69, 20], [7, 129, 64]] = 0
    w.k.values[5, 96:128] = 0
    want, bound = ref.weights(w.delta.x, w.k.values)
    assert (np.abs(got - want)[~bad] <= bound[~bad]).all()


def test_no_rows(gpu):
    d = Rows(np.zeros((1, 40)), F32)
    for accumulate in (0, 1):
        w = Weights(gpu, d, np.zeros((1, 33)), accumulate)
        w.desc.rows = 0
        w.nb = gpu.ach_fc_bwd_filter_checkpoint_workspace(C.byref(w.desc))
        w.call()
        assert np.array_equal(w.read(), w.old if accumulate else np.zeros((40, 33), np.float32))


@pytest.fixture
def stream(gpu):
    s = C.c_void_p()
    check(gpu.ach_stream_create(C.byref(s)))
    yield s.value
    check(gpu.ach_stream_destroy(s.value))


def test_graph_replays(gpu, stream):
    """pack and the weight gradient from it, captured and replayed on other
    values, with eager calls between; two graphs share a workspace"""
    hip, rng = Hip(), np.random.default_rng(10)
    jobs = []
    for rows, inputs, outputs, kind in ((3000, 100, 60, BF16), (200, 300, 70, F32)):
        x = Rows(activations(rng, rows, inputs), kind)
        jobs.append((x, Weights(gpu, Rows(rng.standard_normal((rows, outputs)), kind), x.x)))
    ws = D(max(max(w.nb for _, w in jobs), 4), np.uint8)
    graphs = []
    for x, w in jobs:
        w.ws = ws
        pd = aetcnn.CheckpointDesc(x.rows, x.n, x.kind, x.stride)

        def both(s=stream, x=x, w=w, pd=pd):
            check(gpu.ach_checkpoint_pack(C.byref(pd), x.ptr, w.k.ptr, s))
            w.call(s)
        graphs.append((hip.capture(stream, both), both))
    for replay in range(4):
        for x, w in jobs:
            new = Rows(activations(rng, x.rows, x.n), x.kind)
            x.dev.upload(new.raw)
            w.k.values = ref.values(*ref.pack(new.x), x.n)
            w.restart()
        for g, _ in graphs:
            hip.launch(g, stream)
        check(gpu.ach_stream_sync(stream))
        for (x, w), (_, eager) in zip(jobs, graphs):
            w.check()
            first = w.read().tobytes()
            eager()
            check(gpu.ach_stream_sync(stream))
            assert w.read().tobytes() == first


def test_two_streams_at_once(gpu, stream):
    rng = np.random.default_rng(11)
    other = C.c_void_p()
    check(gpu.ach_stream_create(C.byref(other)))
    jobs = [(s, Weights(gpu, Rows(rng.standard_normal((2000, 100)), BF16), activations(rng, 2000, 90)))
            for s in (stream, other.value)]
    for _ in range(5):
        for s, w in jobs:
            w.call(s)
    for s, w in jobs:
        check(gpu.ach_stream_sync(s))
        w.check()
    check(gpu.ach_stream_destroy(other.value))


@pytest.mark.parametrize("kind", [F32, BF16])
def test_runs_are_equal(gpu, kind):
    rng = np.random.default_rng(12)
    w = Weights(gpu, Rows(rng.standard_normal((4000, 150)), kind), activations(rng, 4000, 170))
    seen = set()
    for _ in range(8):
        w.call()
        seen.add(w.read().tobytes())
    assert len(seen) == 1
