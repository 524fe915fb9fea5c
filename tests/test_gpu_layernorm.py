"""Layer norm, forward and backward, against 64-bit references (norm_ref.py,
where the error bounds are derived), at the sizes, types, strides and values
where its kernels can go wrong."""
import ctypes as C

import numpy as np
import pytest

import aetcnn
import norm_ref as ref
from aetcnn import BF16, F16, F32, check
from aetcnn import DeviceArray as D
from test_gpu_checkpoint import Kept, activations, stream, unpack  # noqa: F401
from test_gpu_logits import Hip, Rows, like

pytestmark = pytest.mark.gpu
FLOOR = 2.0 ** -120  # absolute: products below the smallest normal may be 0


def near(got, want, name, rows=None):
    value, bound = want
    got = np.asarray(got, np.float64)
    if rows is not None:
        got, value, bound = got[rows], value[rows], bound[rows]
    assert np.isfinite(got).all(), name
    over = np.abs(got - value) - bound - FLOOR
    assert over.max(initial=-1) <= 0, (name, np.unravel_index(over.argmax(), over.shape), over.max())


def floats(a):
    return None if a is None else D.from_numpy(np.ascontiguousarray(a, np.float32))


def ptr(a):
    return None if a is None else a.ptr


class Forward:
    def __init__(self, gpu, x, scales, biases, eps=1e-5, keep=False, outputs=("y", "stats"), pad=0,
                 shift=0, in_place=False):
        self.gpu, self.x, self.eps = gpu, x, eps
        self.s, self.b = floats(scales), floats(biases)
        self.y = (x if in_place else like(x, pad, shift)) if "y" in outputs else None
        self.stats = D((x.rows, 2)) if "stats" in outputs else None
        if self.stats:
            self.stats.upload(np.full((x.rows, 2), -7, np.float32))
        self.k = Kept(x.rows, x.n) if keep else None
        self.desc = aetcnn.LayernormDesc(x.rows, x.n, x.kind, eps, x.stride)
        self.nb = gpu.ach_layernorm_fwd_workspace(C.byref(self.desc))
        self.ws = D(max(self.nb, 4), np.uint8)
        self.ws.upload(np.full(self.ws.shape, 0xff, np.uint8))
        self.want = ref.forward(x.x, scales, biases, eps, x.kind)

    def call(self, stream=None):
        check(self.gpu.ach_layernorm_fwd(
            C.byref(self.desc), self.x.ptr, ptr(self.s), ptr(self.b), ptr(self.y),
            self.y.stride if self.y else 0, ptr(self.stats), ptr(self.k), self.ws.ptr, self.nb, stream))

    def check(self, rows=None):
        if self.y:
            near(self.y.read(), self.want["y"], "y", rows)
        if self.stats:
            st = self.stats.numpy()
            near(st[:, 0], self.want["mean"], "mean", rows)
            near(st[:, 1], self.want["rstd"], "rstd", rows)
        if self.k:
            self.check_kept(rows)

    def check_kept(self, rows=None):
        """codes of x_norm: within half a step, and its error, of it"""
        codes, steps = self.k.read()
        n = self.x.n
        assert not codes[:, n:].any()
        v, (xn, e) = ref.values(codes, steps, n), self.want["x_norm"]
        half = np.repeat(np.ldexp(0.5, steps.astype(int) - 133), 32, axis=1)[:, :n]
        near(v, (xn, e * 1.01 + half), "x_norm", rows)
        # the steps are those of the largest magnitudes, but for their errors
        low, high = (ref.pack(np.abs(xn) * 1.0 + d)[1] for d in (-e * (np.abs(xn) > e), e))
        ok = (steps >= low) & (steps <= high)
        assert ok.all() if rows is None else ok[rows].all()


class Backward:
    def __init__(self, gpu, delta, f, scales, from_kept=False, accumulate=0, pad=0, shift=0,
                 in_place=False, outputs=("dx", "scales", "biases")):
        """f: what ref.forward gives and the rows it was given"""
        self.gpu, self.delta, self.acc = gpu, delta, accumulate
        x, eps = f
        self.s = floats(scales)
        w = ref.forward(x.x, None, None, eps, F32)
        stats = np.stack([w["mean"][0], w["rstd"][0]], 1).astype(np.float32)
        self.stats = D.from_numpy(stats)
        st = stats.astype(np.float64)
        xn = (x.x - st[:, :1]) * st[:, 1:]
        self.x, self.k, e_xn = x, None, 3 * ref.U * np.abs(xn)
        if from_kept:
            self.x, self.k = None, Kept.of(xn)
            xn, e_xn = self.k.values, 0.0
        self.dx = (delta if in_place else like(delta, pad, shift)) if "dx" in outputs else None
        rng = np.random.default_rng(3)
        self.old = rng.standard_normal((2, delta.n)).astype(np.float32)
        self.up = [D((delta.n + 8,)) if v in outputs else None for v in ("scales", "biases")]
        self.restart()
        self.desc = aetcnn.LayernormDesc(x.rows, x.n, x.kind, eps, x.stride)
        self.nb = gpu.ach_layernorm_bwd_workspace(C.byref(self.desc))
        self.ws = D(max(self.nb, 4), np.uint8)
        self.ws.upload(np.full(self.ws.shape, 0xff, np.uint8))
        self.want = ref.backward(delta.x, xn, e_xn, st[:, 1], scales, x.kind)

    def restart(self):
        for u, o in zip(self.up, self.old):
            if u:
                u.upload(np.concatenate([o, np.full(8, 77, np.float32)]))

    def call(self, stream=None):
        check(self.gpu.ach_layernorm_bwd(
            C.byref(self.desc), self.delta.ptr, self.delta.stride, ptr(self.x), ptr(self.k),
            self.stats.ptr, ptr(self.s), ptr(self.dx), self.dx.stride if self.dx else 0,
            ptr(self.up[0]), ptr(self.up[1]), self.acc, self.ws.ptr, self.nb, stream))

    def read(self):
        out = {} if self.dx is None else dict(dx=self.dx.read())
        for name, u in zip(("scales", "biases"), self.up):
            if u:
                v = u.numpy()
                assert (v[-8:] == 77).all(), "written behind the updates"
                out[name] = v[:-8]
        return out

    def check(self):
        for name, v in self.read().items():
            value, bound = self.want[name]
            if self.acc and name != "dx":
                old = self.old[0 if name == "scales" else 1].astype(np.float64)
                value, bound = value + old, bound + ref.U * (np.abs(value + old) + np.abs(old))
            near(v, (value, bound), name)


def parameters(rng, n):
    return (rng.standard_normal(n) * 0.3 + 1).astype(np.float32), rng.standard_normal(n).astype(np.float32)


SIZES = [
    # rows, features, pad, shift
    (1, 1, 0, 0), (5, 2, 1, 0), (1, 7, 0, 1), (3, 31, 0, 0), (33, 32, 0, 0), (9, 33, 3, 1),
    (17, 64, 0, 0), (1000, 10, 2, 0), (70, 127, 0, 1), (6, 128, 0, 0), (300, 129, 1, 0),
    (5, 255, 0, 0), (4, 257, 0, 1), (130, 500, 4, 0), (3, 512, 0, 0), (2, 1000, 0, 3),
    (600, 1024, 0, 0), (9, 1025, 7, 0), (5, 2047, 0, 0), (3, 2048, 0, 0), (7, 2049, 0, 1),
    (128, 4096, 0, 0), (2, 4097, 0, 0), (5, 5003, 13, 1), (3, 8192, 0, 0), (2, 8193, 0, 0),
    (3, 12289, 0, 0), (2, 16384, 0, 0), (2, 16391, 1, 0), (1, 32768, 0, 0), (3, 32801, 0, 1),
    (1, 65536, 0, 0), (2, 65541, 3, 0), (1, 200003, 0, 0), (20, 186624 // 4, 0, 0)]


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("rows,n,pad,shift", SIZES)
def test_forward(gpu, rows, n, pad, shift, kind):
    rng = np.random.default_rng(rows * 7 + n)
    x = Rows(activations(rng, rows, n) + rng.standard_normal(n) * 0.5, kind, pad, shift)
    s, b = parameters(rng, n)
    for keep in (False, True):
        f = Forward(gpu, x, s, b, keep=keep, pad=shift, shift=pad)
        f.call()
        f.check()


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("rows,n,pad,shift", SIZES)
def test_backward(gpu, rows, n, pad, shift, kind):
    rng = np.random.default_rng(rows * 11 + n)
    x = Rows(activations(rng, rows, n) + rng.standard_normal(n) * 0.5, kind, pad, shift)
    s, _ = parameters(rng, n)
    d = Rows(rng.standard_normal((rows, n)) / rows, kind, shift, pad)
    for from_kept in (False, True):
        b = Backward(gpu, d, (x, 1e-5), s, from_kept, accumulate=int(rows % 2 == 0), pad=pad, shift=shift)
        b.call()
        b.check()


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("rows,n", [(3000, 40), (20000, 24), (1500, 600), (700, 3000), (3000, 1000)])
def test_many_rows(gpu, rows, n, kind):
    """more rows than workgroups, long sums over rows"""
    rng = np.random.default_rng(n)
    x = Rows(activations(rng, rows, n), kind)
    s, b = parameters(rng, n)
    f = Forward(gpu, x, s, b, keep=True)
    f.call()
    f.check()
    d = Rows(rng.standard_normal((rows, n)) + 0.1, kind)
    for from_kept in (False, True):
        g = Backward(gpu, d, (x, 1e-5), s, from_kept)
        g.call()
        g.check()


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("rows,n", [(515, 9001), (333, 16500), (70, 60001)])
def test_many_long_rows(gpu, rows, n, kind):
    """rows of 1024 threads in turns, spans of rows in parts"""
    rng = np.random.default_rng(n)
    x = Rows(rng.standard_normal((rows, n)) + rng.standard_normal((rows, 1)), kind)
    s, b = parameters(rng, n)
    f = Forward(gpu, x, s, b, keep=True)
    f.call()
    f.check()
    d = Rows(rng.standard_normal((rows, n)) + 0.1, kind)
    for from_kept in (False, True):
        g = Backward(gpu, d, (x, 1e-5), s, from_kept, accumulate=int(from_kept))
        g.call()
        g.check()


@pytest.mark.parametrize("n", [5, 300, 2500, 20000, 140000])
def test_optional_arguments(gpu, n):
    """no scales, no biases, each output alone"""
    rng = np.random.default_rng(n)
    x = Rows(activations(rng, 3, n), F32)
    s, b = parameters(rng, n)
    for scales, biases in ((None, None), (s, None), (None, b)):
        f = Forward(gpu, x, scales, biases)
        f.call()
        f.check()
    for outputs, keep in ((("y",), False), (("stats",), False), ((), True), (("stats",), True)):
        f = Forward(gpu, x, s, b, keep=keep, outputs=outputs)
        f.call()
        f.check()
    d = Rows(rng.standard_normal((3, n)), F32)
    for outputs in (("dx",), ("scales",), ("biases",), ("dx", "biases"), ("scales", "biases")):
        for from_kept in (False, True):
            g = Backward(gpu, d, (x, 1e-5), s, from_kept, outputs=outputs)
            g.call()
            g.check()
    g = Backward(gpu, d, (x, 1e-5), None)
    g.call()
    g.check()


@pytest.mark.parametrize("n,pad", [(7, 0), (64, 0), (300, 1), (3000, 0), (20001, 3), (100000, 0)])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_in_place(gpu, n, pad, kind):
    rng = np.random.default_rng(n)
    s, b = parameters(rng, n)
    f = Forward(gpu, Rows(activations(rng, 5, n), kind, pad), s, b, keep=True, in_place=True)
    f.call()
    f.check()
    x = Rows(activations(rng, 5, n), kind, pad)
    g = Backward(gpu, Rows(rng.standard_normal((5, n)), kind, pad), (x, 1e-5), s, in_place=True)
    g.call()
    g.check()


@pytest.mark.parametrize("n", [20, 1000, 5000, 40000])
@pytest.mark.parametrize("eps", [1e-12, 1e-5, 1.0])
def test_values_at_the_ends(gpu, n, eps):
    """constant rows, a mean far above the deviations, an outlier in front, tiny and
    huge values, zeros"""
    rng = np.random.default_rng(n)
    x = activations(rng, 9, n)
    x[0] = 3.25
    x[1] = 0
    x[2] = 1e4 + rng.standard_normal(n) * 0.01
    x[3, 0] = 1e6
    x[4] *= 1e-30
    x[5] *= 1e15
    x[6] = np.where(np.arange(n) % 2, 1e25, -1e25)   # squares above the largest float
    x[7] *= 1e-6
    s, b = parameters(rng, n)
    f = Forward(gpu, Rows(x, F32), s, b, eps, keep=True)
    f.call()
    f.check()


@pytest.mark.parametrize("n", [3, 101, 1001, 5003, 30001, 70001])
def test_large_constant_rows(gpu, n):
    """x_norm is 0 there; what stands behind a row's last value must not count,
    though 0 in its place would be infinitely many deviations away"""
    x = Rows(np.full((3, n), 1e35), F32)
    rng = np.random.default_rng(n)
    s, b = parameters(rng, n)
    f = Forward(gpu, x, s, b, 1e-12, keep=True)
    f.call()
    f.check()
    g = Backward(gpu, Rows(rng.standard_normal((3, n)) * 1e-8, F32), (x, 1e-12), s)
    stats = np.stack([np.full(3, x.x[0, 0]), np.full(3, 1e6)], 1).astype(np.float32)
    g.stats.upload(stats)
    g.want = ref.backward(g.delta.x, np.zeros((3, n)), 0.0, stats[:, 1].astype(np.float64), s, F32)
    g.call()
    g.check()


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("n", [3, 100, 3000, 20000, 140000])
def test_rows_that_are_not_finite(gpu, n, kind):
    """they are NaN themselves and touch no other row"""
    rng = np.random.default_rng(n)
    clean = activations(rng, 12, n)
    s, b = parameters(rng, n)
    x = clean.copy()
    x[1, 0], x[4, n // 2], x[5, n - 1], x[9, 0] = np.nan, np.inf, -np.inf, np.inf
    bad, fine = [1, 4, 5, 9], [0, 2, 3, 6, 7, 8, 10, 11]
    f = Forward(gpu, Rows(x, kind), s, b, keep=True)
    f.want = ref.forward(Rows(clean, kind).x, s, b, 1e-5, kind)
    f.call()
    f.check(fine)
    assert np.isnan(f.y.read()[bad]).all()
    assert not np.isfinite(f.stats.numpy()[bad]).all(1).any()
    assert (f.k.read()[1][bad] == 255).all()
    assert np.isnan(unpack(gpu, f.k, F32)[bad]).all()
    # a backward pass over them: dx of the others is theirs, the updates are NaN
    d = Rows(rng.standard_normal((12, n)), kind)
    g = Backward(gpu, d, (Rows(clean, kind), 1e-5), s)
    g.stats.upload(np.where(np.isin(np.arange(12), bad)[:, None], np.nan, g.stats.numpy()).astype(np.float32))
    g.call()
    got = g.read()
    near(got["dx"], g.want["dx"], "dx", fine)
    assert np.isnan(got["dx"][bad]).all()
    assert np.isnan(got["scales"]).all()
    near(got["biases"], g.want["biases"], "biases")


def test_no_rows(gpu):
    x = Rows(np.zeros((1, 50)), F32)
    d = aetcnn.LayernormDesc(0, 50, F32, 1e-5)
    assert gpu.ach_layernorm_fwd(C.byref(d), x.ptr, None, None, x.ptr, 0, None, None, None, 0, None) == 0
    for accumulate in (0, 1):
        g = Backward(gpu, x, (x, 1e-5), None, accumulate=accumulate)
        g.desc.rows = 0
        g.nb = gpu.ach_layernorm_bwd_workspace(C.byref(g.desc))
        g.call()
        for u, o in zip(g.up, g.old):
            assert np.array_equal(u.numpy()[:50], o if accumulate else np.zeros(50))
        assert np.isnan(g.dx.read()).all()  # nothing written


def test_offsets_past_32_bits(gpu):
    """rows far apart in a buffer of more than 2^32 bytes"""
    rows, n, stride = 3, 1000, 900_000_007
    big = C.c_void_p()
    check(gpu.ach_malloc(C.byref(big), (2 * stride + n) * 2))
    rng = np.random.default_rng(0)
    x = Rows(activations(rng, rows, n), BF16)
    s, b = parameters(rng, n)
    for r in range(rows):
        check(gpu.ach_memcpy_h2d(big.value + 2 * r * stride, x.bits[r].ctypes.data, 2 * n, None))
    f = Forward(gpu, x, s, b, keep=True)
    f.desc.stride = stride
    f.x = type("Far", (), dict(ptr=big.value, n=n))
    f.call()
    f.check()
    d = Rows(rng.standard_normal((rows, n)), BF16)
    g = Backward(gpu, d, (x, 1e-5), s)
    g.desc.stride = stride
    g.x = f.x
    g.call()
    g.check()
    k = Kept(rows, n)
    check(gpu.ach_checkpoint_pack(C.byref(aetcnn.CheckpointDesc(rows, n, BF16, stride)), big.value,
                                  k.ptr, None))
    assert np.array_equal(k.read()[0], ref.pack(x.x)[0])
    check(gpu.ach_free(big))


def test_a_row_of_many_values(gpu):
    """over 2^27: more columns than one launch's threads"""
    n = (1 << 27) + 77
    rng = np.random.default_rng(1)
    block = rng.standard_normal(1 << 16).astype(np.float32)
    raw = np.resize(block, n).view(np.uint32)
    bits16 = (raw >> 16).astype(np.uint16)  # bf16, cut off
    v = (bits16.astype(np.uint32) << 16).view(np.float32)
    x, out = D.from_numpy(bits16), D((n,), np.uint16)
    up = [D((n,)), D((n,))]
    st = D((1, 2))
    d = aetcnn.LayernormDesc(1, n, BF16, 1e-5)
    fb, bb = (q(C.byref(d)) for q in (gpu.ach_layernorm_fwd_workspace, gpu.ach_layernorm_bwd_workspace))
    ws = D((max(fb, bb) // 4 + 4,), np.int32)
    check(gpu.ach_layernorm_fwd(C.byref(d), x.ptr, None, None, out.ptr, 0, st.ptr, None, ws.ptr, fb, None))
    mean, var = v.mean(dtype=np.float64), v.var(dtype=np.float64)
    got = st.numpy()[0].astype(np.float64)
    assert abs(got[0] - mean) <= 1e-6 and abs(got[1] * np.sqrt(var + 1e-5) - 1) <= 1e-6
    y = (out.numpy().astype(np.uint32) << 16).view(np.float32)
    want = (v - np.float32(got[0])) * np.float32(got[1])
    assert (np.abs(y - want) <= 2.0 ** -8 * np.abs(want) + 1e-30).all()
    # the row itself as its delta
    check(gpu.ach_layernorm_bwd(C.byref(d), x.ptr, 0, x.ptr, None, st.ptr, None, out.ptr, 0, up[0].ptr,
                                up[1].ptr, 0, ws.ptr, bb, None))
    assert np.array_equal(up[1].numpy(), v)
    ds = up[0].numpy()
    assert (np.abs(ds - v * want) <= 4 * ref.U * np.abs(v * want)).all()
    # the row is nearly its own x_norm, so dx is what cancellation leaves.  Its
    # terms are off by 5 u of their sizes (norm_ref.backward); the two means by that of
    # chains of at most 16 chunks of 8 values a thread and what joins 256 threads
    # (10), the parts' sums in 64 bits: 138 additions, a product, a division: 142 u
    # of the mean of the terms' magnitudes
    m1, m2 = mean, (v * want).mean(dtype=np.float64)
    e1, e2 = (142 * ref.U * np.abs(q).mean(dtype=np.float64) for q in (v, v * want))
    size = np.abs(v) + abs(m1) + np.abs(want * m2)
    bound = got[1] * (5 * ref.U * size + e1 + np.abs(want) * (e2 + 3 * ref.U * abs(m2)))
    y = (out.numpy().astype(np.uint32) << 16).view(np.float32)
    want = got[1] * (v - m1 - want * m2)
    assert (np.abs(y - want) <= bound + 2.0 ** -8 * (np.abs(want) + bound)).all()


def bits(f, g):
    return b"".join([f.y.read().tobytes(), f.stats.numpy().tobytes(), f.k.dev.numpy().tobytes()] +
                    [v.tobytes() for v in g.read().values()])


@pytest.mark.parametrize("shapes", [((2000, 300, BF16), (128, 4096, F32)), ((3, 140000, F32), (40, 20000, F16))])
def test_graph_replays(gpu, stream, shapes):  # noqa: F811
    """a training step's two halves, captured and replayed on other values, with
    eager calls between; two graphs share a workspace"""
    hip, rng = Hip(), np.random.default_rng(7)
    jobs, graphs = [], []
    for rows, n, kind in shapes:
        x = Rows(activations(rng, rows, n), kind)
        s, b = parameters(rng, n)
        f = Forward(gpu, x, s, b, keep=True)
        g = Backward(gpu, Rows(rng.standard_normal((rows, n)), kind), (x, 1e-5), s, from_kept=True)
        g.stats, g.k = f.stats, f.k
        jobs.append((f, g, s, b))
    ws = D(max(max(f.nb, g.nb) for f, g, _, _ in jobs), np.uint8)
    for f, g, _, _ in jobs:
        f.ws = g.ws = ws
        graphs.append(hip.capture(stream, lambda: (f.call(stream), g.call(stream))))
    for replay in range(3):
        for f, g, s, b in jobs:
            new = Rows(activations(rng, f.x.rows, f.x.n), f.x.kind)
            f.x.dev.upload(new.raw)
            f.want = ref.forward(new.x, s, b, 1e-5, f.x.kind)
        for ex in graphs:
            hip.launch(ex, stream)
        check(gpu.ach_stream_sync(stream))
        for f, g, s, b in jobs:
            f.check()
            st = f.stats.numpy().astype(np.float64)
            xn = ref.values(*f.k.read(), f.x.n)
            g.want = ref.backward(g.delta.x, xn, 0.0, st[:, 1], s, f.x.kind)
            g.check()
            graph = bits(f, g)
            f.call(stream)
            g.call(stream)
            check(gpu.ach_stream_sync(stream))
            assert graph == bits(f, g)


def test_two_streams_at_once(gpu, stream):  # noqa: F811
    rng = np.random.default_rng(13)
    other = C.c_void_p()
    check(gpu.ach_stream_create(C.byref(other)))
    jobs = []
    for s, n in ((stream, 4096), (other.value, 50000)):
        x = Rows(activations(rng, 20, n), BF16)
        sc, b = parameters(rng, n)
        jobs.append((s, Forward(gpu, x, sc, b),
                     Backward(gpu, Rows(rng.standard_normal((20, n)), BF16), (x, 1e-5), sc)))
    for _ in range(5):
        for s, f, g in jobs:
            f.call(s)
            g.call(s)
    for s, f, g in jobs:
        check(gpu.ach_stream_sync(s))
        f.check()
        g.check()
    check(gpu.ach_stream_destroy(other.value))


@pytest.mark.parametrize("rows,n,kind", [(900, 200, F32), (700, 4096, BF16), (5, 100000, F32), (3, 30000, F16)])
def test_runs_are_equal(gpu, rows, n, kind):
    rng = np.random.default_rng(n)
    x = Rows(activations(rng, rows, n), kind)
    s, b = parameters(rng, n)
    f = Forward(gpu, x, s, b, keep=True)
    g = Backward(gpu, Rows(rng.standard_normal((rows, n)), kind), (x, 1e-5), s)
    seen = set()
    for _ in range(8):
        f.call()
        g.call()
        seen.add(bits(f, g))
    assert len(seen) == 1


@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_a_layer_from_its_checkpoints(gpu, kind):
    """A fully connected layer behind a layer norm, as a training step runs them:
    the forward keeps x_norm and y in 8 bits and nothing else of the rows, the
    backward takes every gradient from them, and these are the 64-bit ones of
    the kept values."""
    rng = np.random.default_rng(21)
    rows, n, m = 96, 200, 75
    x = Rows(activations(rng, rows, n), kind)
    s, b = parameters(rng, n)
    f = Forward(gpu, x, s, b, keep=True)
    f.call()
    f.check()
    ky = Kept(rows, n)
    check(gpu.ach_checkpoint_pack(C.byref(aetcnn.CheckpointDesc(rows, n, kind, f.y.stride)), f.y.ptr,
                                  ky.ptr, None))
    y = f.y.read()
    codes = ky.read()
    assert np.array_equal(codes[0], ref.pack(y)[0]) and np.array_equal(codes[1], ref.pack(y)[1])
    dz = Rows(rng.standard_normal((rows, m)) / rows, kind)  # of the layer's output
    w = rng.standard_normal((m, n)) / np.sqrt(n)
    dw = D((m, n))
    fd = aetcnn.FcDesc(rows, n, m, kind)
    nb = gpu.ach_fc_bwd_filter_checkpoint_workspace(C.byref(fd))
    ws = D(max(nb, 4), np.uint8)
    check(gpu.ach_fc_bwd_filter_checkpoint(C.byref(fd), ky.ptr, dz.ptr, dw.ptr, 0, ws.ptr, nb, None))
    y8, xn8 = ref.values(*codes, n), ref.values(*f.k.read(), n)
    want, bound = ref.weights(dz.x, y8)
    assert (np.abs(dw.numpy() - want) <= bound).all()
    dy = Rows(dz.x @ w, kind)
    g = Backward(gpu, dy, (x, 1e-5), s, from_kept=True)
    g.stats, g.k = f.stats, f.k
    g.want = ref.backward(dy.x, xn8, 0.0, f.stats.numpy()[:, 1].astype(np.float64), s, kind)
    g.call()
    g.check()
    # and near the gradients of values that were not rounded: a code is at most a
    # 127th of its block's largest value off, half of that on the whole
    full = ref.backward(dy.x, f.want["x_norm"][0], 0.0, f.want["rstd"][0], s, kind)
    for name in ("dx", "scales"):
        a, c = g.read()[name], full[name][0]
        assert np.linalg.norm(a - c) <= 0.05 * np.linalg.norm(c), name
    exact = dz.x.T @ f.want["y"][0]
    assert np.linalg.norm(dw.numpy() - exact) <= 0.05 * np.linalg.norm(exact)
