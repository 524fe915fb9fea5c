"""The operators on logits (logits.hip) against 64-bit references, at the
sizes, types, strides and masks where their kernels can go wrong.  The error
bounds are derived in logits_ref.py; ids and ranks have to be equal."""
import ctypes as C

import numpy as np
import pytest

import aetcnn
import logits_ref as ref
from aetcnn import BF16, F16, F32, DISTILL_RENORM, DISTILL_TAIL, check
from aetcnn import DeviceArray as D

pytestmark = pytest.mark.gpu

BITS = {F32: np.float32, BF16: np.uint16, F16: np.float16}
FLOOR = 2.0 ** -118  # absolute: exponentials below the smallest normal may be 0
CANARY = 0x5a


class Rows:
    """Logits on the device: rows `stride` apart, `shift` elements into an
    allocation whose other bytes hold a pattern."""

    def __init__(self, x, kind, pad=0, shift=0):
        self.kind, (self.rows, self.n) = kind, x.shape
        self.stride, self.shift = self.n + pad, shift
        self.bits = ref.to_bits(x, kind)
        self.x = ref.from_bits(self.bits, kind)
        size = np.dtype(BITS[kind]).itemsize
        self.raw = np.full((self.rows * self.stride + shift + 16) * size, CANARY, np.uint8)
        self.view(self.raw)[:] = self.bits
        self.dev = D.from_numpy(self.raw)
        self.ptr = self.dev.ptr + shift * size

    def view(self, raw):
        flat = raw.view(BITS[self.kind])[self.shift:self.shift + self.rows * self.stride]
        return flat.reshape(self.rows, self.stride)[:, :self.n]

    def read(self):
        """the rows as float64; what lies around them has to be untouched"""
        raw = self.dev.numpy()
        got = self.view(raw).copy()
        self.view(raw)[:] = self.bits
        assert np.array_equal(raw, self.raw), "written outside the rows"
        return ref.from_bits(got, self.kind)


def like(rows, pad=0, shift=0):
    """an output of the rows' shape and type, filled with NaN"""
    return Rows(np.full((rows.rows, rows.n), np.nan), rows.kind, pad, shift)


def dev(a, dtype):
    return None if a is None else D.from_numpy(np.ascontiguousarray(a, dtype))


def ptr(a):
    return None if a is None else a.ptr


def sample(rng, rows, n, spread=2.5):
    x = rng.standard_normal((rows, n)) * spread
    for r in range(rows):
        at = rng.integers(0, n, max(1, min(n // 4, 16)))
        x[r, at] += rng.exponential(4, len(at))
    return x


class Forward:
    def __init__(self, gpu, rows, ids, k, t, outputs=("logprobs", "ranks", "entropy", "stats")):
        self.gpu, self.rows, self.k = gpu, rows, k
        self.desc = aetcnn.LogitsDesc(rows.rows, rows.n, rows.kind, t, rows.stride)
        self.ids = dev(ids, np.int32)
        R = rows.rows
        self.out = {name: D((R, 2) if name == "stats" else R,
                            np.int32 if name == "ranks" else np.float32) for name in outputs}
        if k:
            self.out.update(top_ids=D((R, k), np.int32), top_logprobs=D((R, k)))
        for v in self.out.values():
            v.upload(np.full(v.shape, -7, v.dtype))
        self.nb = gpu.ach_logprobs_workspace(C.byref(self.desc), k)
        self.ws = D(max(self.nb, 4), np.uint8)
        self.ws.upload(np.full(self.ws.shape, 0xff, np.uint8))

    def call(self, stream=None):
        o = [ptr(self.out.get(v)) for v in ("logprobs", "ranks", "entropy", "stats", "top_ids",
                                            "top_logprobs")]
        check(self.gpu.ach_logprobs_fwd(C.byref(self.desc), self.rows.ptr, ptr(self.ids), self.k,
                                        *o, self.ws.ptr, self.nb, stream))

    def read(self, stream=None):
        return {name: v.numpy(stream) for name, v in self.out.items()}


def near(got, want, name=""):
    value, bound = want
    got, value = np.asarray(got, np.float64), np.asarray(value, np.float64)
    fin = np.isfinite(value)
    assert np.array_equal(got[~fin], value[~fin], equal_nan=True), name
    assert np.isfinite(got[fin]).all(), name
    exact = name in ("ranks", "top_ids")
    bound = 0 if exact else np.where(fin, bound, 0) + FLOOR
    over = np.where(fin, np.abs(np.where(fin, got, 0) - np.where(fin, value, 0)) - bound, -1)
    assert over.max(initial=-1) <= 0, (name, np.unravel_index(over.argmax(), over.shape), over.max())


def check_forward(gpu, rows, ids, k, t, **kw):
    f = Forward(gpu, rows, ids, k, t, **kw)
    f.call()
    got = f.read()
    want = ref.logprobs(rows.x, ids if ids is not None else np.full(rows.rows, -1), k, t)
    for name, v in got.items():
        near(v, want[name], name)
    return f, got


FORWARD = [
    # rows, classes, type, k, temperature, pad, shift
    (1, 1, F32, 1, 1.0, 0, 0),
    (3, 2, BF16, 2, 1.0, 3, 1),
    (5, 10, F32, 10, 0.7, 0, 0),           # all classes, sorted
    (4, 63, F16, 63, 1.0, 1, 1),
    (9, 64, BF16, 5, 2.0, 0, 0),
    (7, 65, F32, 20, 1.0, 2, 3),
    (128, 1000, F32, 5, 1.0, 0, 0),
    (3, 1000, BF16, 128, 1.0, 1, 0),       # the most alternatives
    (2, 1023, F16, 33, 1.5, 0, 5),
    (3, 1025, F32, 128, 1.0, 0, 1),
    (2, 2049, BF16, 64, 1.0, 7, 7),
    (300, 2050, F16, 7, 1.0, 0, 0),
    (3, 4099, F32, 33, 4.0, 1, 2),
    (2, 8191, BF16, 17, 1.0, 0, 1),
    (600, 9000, BF16, 20, 1.0, 0, 0),      # more rows than compute units
    (1100, 5000, F32, 20, 1.0, 1, 0),      # a wave per row of some thousands
    (1030, 8192, BF16, 32, 1.0, 0, 0),
    (1025, 8191, F16, 33, 1.0, 0, 1),      # too many alternatives for that
    (3, 16411, F32, 100, 1.0, 0, 0),
    (2, 50021, F16, 20, 0.5, 3, 1),
    (700, 33000, F32, 3, 1.0, 0, 0),
    (1, 131072, BF16, 20, 1.0, 0, 0),      # one row, in parts
    (1, 131071, F32, 1, 1.0, 0, 1),
    (5, 200001, F16, 128, 1.0, 1, 0),
]


@pytest.mark.parametrize("rows,n,kind,k,t,pad,shift", FORWARD)
def test_logprobs(gpu, rows, n, kind, k, t, pad, shift):
    rng = np.random.default_rng(rows * 7 + n)
    x = Rows(sample(rng, rows, n), kind, pad, shift)
    ids = rng.integers(0, n, rows)
    best = rng.random(rows) < 0.5
    ids[best] = x.x.argmax(1)[best]
    ids[rng.random(rows) < 0.2] = -1
    check_forward(gpu, x, ids, k, t)
    x.read()


@pytest.mark.parametrize("n,kind", [(10, F32), (1000, BF16), (5000, F16), (70000, F32)])
def test_each_output_alone(gpu, n, kind):
    """any of the outputs may be missing; ids may where nothing needs them"""
    rng = np.random.default_rng(n)
    x = Rows(sample(rng, 6, n), kind)
    ids = rng.integers(0, n, 6)
    for names in (("logprobs",), ("ranks",), ("logprobs", "ranks")):
        check_forward(gpu, x, ids, 0, 1.0, outputs=names)
    for names, k in ((("entropy",), 0), (("stats",), 0), ((), 7), (("stats", "entropy"), 3)):
        check_forward(gpu, x, None, k, 1.0, outputs=names)


def test_ids_that_are_none(gpu):
    rng = np.random.default_rng(1)
    for n in (10, 3000, 100000):
        x = Rows(sample(rng, 7, n), F32)
        ids = np.array([-1, n, -2 ** 31, 2 ** 31 - 1, 0, n - 1, n + 1], np.int64)
        _, got = check_forward(gpu, x, ids, 2, 1.0)
        assert not got["logprobs"][[0, 1, 2, 3, 6]].any()
        assert (got["ranks"][[0, 1, 2, 3, 6]] == -1).all()


@pytest.mark.parametrize("n,k,times", [(12, 12, 1), (500, 40, 1), (2000, 32, 1), (3000, 128, 1),
                                       (40000, 20, 1), (131072, 64, 1), (6000, 30, 120),
                                       (33000, 64, 32)])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_masked_classes(gpu, n, k, times, kind):
    """-inf: most classes masked, fewer left than alternatives, one left,
    none left; and masks of the type's lowest value"""
    rng = np.random.default_rng(n + k)
    x = sample(rng, 9, n)
    x[0, rng.random(n) < 0.7] = -np.inf
    x[1, rng.permutation(n)[k // 2:]] = -np.inf     # k/2 left
    x[2, :n - 3] = -np.inf                          # the last three
    x[3, 5:] = -np.inf                              # the first five
    x[4] = -np.inf
    x[4, n // 2] = -3.25                            # one left
    x[5] = -np.inf                                  # none
    low = {F32: -np.finfo(np.float32).max, BF16: -3.3895313892515355e38, F16: -65504.0}[kind]
    x[6, rng.random(n) < 0.8] = low
    x[7] = low                                      # an even distribution
    x[8, 1:] = low
    rows = Rows(np.tile(x, (times, 1)), kind)  # many rows: other kernels
    ids = rows.x.argmax(1)
    ids[1] = int(np.flatnonzero(np.isneginf(rows.x[1]))[0])  # a masked class: -inf
    ids[3] = n - 1
    _, got = check_forward(gpu, rows, ids, k, 1.0)
    assert got["entropy"][5] == 0 and np.isneginf(got["logprobs"][5])
    assert got["logprobs"][4] == 0 and got["entropy"][4] == 0


@pytest.mark.parametrize("n,k", [(10, 4), (1000, 5), (5000, 20), (131072, 20)])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_rows_that_are_not_finite(gpu, n, k, kind):
    """a NaN or a +inf anywhere spoils its row and no other"""
    rng = np.random.default_rng(n)
    x = sample(rng, 8, n)
    x[1, n - 1] = np.nan
    x[3, 0] = np.inf
    x[4, n // 2] = np.inf
    x[4, n // 3] = np.nan
    x[6] = np.nan
    bad = np.array([1, 3, 4, 6])
    rows = Rows(x, kind)
    ids = np.full(8, 1)
    ids[3] = 0
    f = Forward(gpu, rows, ids, k, 1.0)
    f.call()
    got = f.read()
    want = ref.logprobs(np.where(np.isin(np.arange(8), bad)[:, None], 0, rows.x), ids, k, 1.0)
    good = np.setdiff1d(np.arange(8), bad)
    for name, v in got.items():
        near(v[good], tuple(np.asarray(w)[good] if np.ndim(w) else w for w in want[name]), name)
        assert (v[bad] == -1).all() if v.dtype == np.int32 else np.isnan(v[bad]).all(), name


@pytest.mark.parametrize("n", [9, 777, 3000, 70001, 131072])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_order_of_equal_logits(gpu, n, kind):
    """equal logits by ascending id, -0 equal to +0, whatever the rows' order"""
    rng = np.random.default_rng(n)
    k = min(n, 128)
    x = np.stack([np.zeros(n), rng.integers(0, 3, n), rng.integers(-2, 2, n) * 0.5,
                  np.arange(n) / n, -np.arange(n) / n, np.where(np.arange(n) % 2, 0.0, -0.0),
                  np.where(np.arange(n) == n - 1, 1, 0), np.repeat(1.5, n)])
    rows = Rows(x, kind)
    ids = rng.integers(0, n, len(x))
    check_forward(gpu, rows, ids, k, 1.0)
    check_forward(gpu, rows, ids, min(k, 3), 1.0)


@pytest.mark.parametrize("n", [4096, 65536, 131072, 150000])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_large_logits_in_one_place(gpu, n, kind):
    """the largest logits are neighbours, or lie at one distance from one
    another: the same lane, wave or part of a row sees all of them, in
    ascending order or descending"""
    rng = np.random.default_rng(n)
    base = rng.standard_normal((1, n))
    x = np.repeat(base, 10, 0)
    j = np.arange(n)
    for r, step in enumerate((1, 8, 64, 512, 1024, 2048, 4096, 8192)):
        at = j[(j % step) < (8 if step >= 8 else 1)][:1500] if step > 1 else j[n // 2:n // 2 + 1500]
        x[r, at] = 20 + (np.arange(len(at)) if r % 2 else -np.arange(len(at))) / 8
    x[8, :3000] = 30 + np.arange(min(n, 3000)) / 16
    x[9, -2000:] = 30 - np.arange(2000) / 16
    rows = Rows(x, kind)
    check_forward(gpu, rows, np.arange(10), 128, 1.0)
    check_forward(gpu, rows, np.arange(10), 20, 1.0)


@pytest.mark.parametrize("n", [40003, 60001, 140000])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_equal_logits_by_groups(gpu, n, kind):
    """most logits are equal, with larger ones, lower ones or none allowed in
    whole stretches: groups of logits are left out, or read and hold no others"""
    rng = np.random.default_rng(n)
    j = np.arange(n)
    x = np.ones((10, n))
    x[1, j < n // 2] = -np.inf                           # half of the groups closed
    x[2, rng.random(n) > 1e-3] = -np.inf                 # some allowed, all equal
    x[3, 37::997] = 2 + np.arange(len(j[37::997])) / 64  # larger ones, late too
    x[4, -5:] = 3                                        # larger ones behind all others
    x[5, :1500] = 2 + np.arange(1500) % 7                # larger ones, equal too
    x[6, j != n - 2] = -np.inf                           # fewer than k allowed
    x[7] = np.where(j % 3, np.finfo(np.float32).min / 2, 1.0)
    x[7, :n // 2] = np.finfo(np.float32).min / 2         # a mask of large finite values
    x[8] = np.where(j < 700, j / 8, 0.0)                 # too many for the list
    x[9, ::2] = -3
    rows = Rows(x, kind)
    ids = rng.integers(0, n, len(x))
    for k in (1, 20, 128):
        check_forward(gpu, rows, ids, k, 1.0)


@pytest.mark.parametrize("n", [10, 1000, 30000, 131072])
def test_certain_rows(gpu, n):
    """where one class has nearly all the probability, its log probability and
    the entropy keep their relative precision"""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((6, n))
    for r, gap in enumerate((2, 10, 15, 25, 30, 60)):
        x[r, n - 1 - r] = gap + np.log(n)
    ids = n - 1 - np.arange(6)
    _, got = check_forward(gpu, Rows(x, F32), ids, 3, 1.0)
    want = ref.logprobs(Rows(x, F32).x, ids, 3, 1.0)
    for name in ("logprobs", "entropy"):
        rel = np.abs(got[name] / want[name][0] - 1)[:5]
        assert rel.max() < 2.0 ** -24 * (5 * 60 + 2 * n / 64 + 56), (name, rel)


BACKWARD = [
    # rows, classes, type, temperature, pad, shift, pad of the output, its shift
    (1, 1, F32, 1.0, 0, 0, 0, 0),
    (3, 2, F16, 1.0, 1, 1, 0, 0),
    (128, 10, F32, 2.0, 0, 0, 0, 0),
    (7, 63, BF16, 1.0, 0, 0, 1, 1),
    (128, 1000, F32, 1.0, 0, 0, 0, 0),
    (5, 1001, BF16, 0.5, 3, 1, 0, 0),
    (9, 4097, F16, 1.0, 0, 3, 2, 1),
    (515, 5003, F32, 1.0, 1, 0, 0, 3),
    (300, 30011, F32, 1.0, 0, 0, 0, 0),    # more than the caches hold
    (2, 50021, BF16, 1.0, 0, 0, 0, 0),
    (1, 131072, F32, 3.0, 0, 0, 0, 0),
    (3, 200001, F16, 1.0, 1, 1, 1, 1),
]


class Backward:
    def __init__(self, gpu, rows, ids, t, g, h, out):
        self.gpu, self.rows, self.out, self.t, self.h_ids = gpu, rows, out, t, ids
        n = rows.n
        clean = np.where(np.isfinite(rows.x) | np.isneginf(rows.x), rows.x, 0)
        o = ref.logprobs(clean, np.full(rows.rows, -1), 0, t)
        self.stats = o["stats"][0].astype(np.float32)
        self.entropy = o["entropy"][0].astype(np.float32)
        self.g = None if g is None else np.asarray(g, np.float32)
        self.h = None if h is None else np.asarray(h, np.float32)
        self.bufs = [dev(ids, np.int32), dev(self.stats, np.float32),
                     dev(self.entropy, np.float32) if h is not None else None,
                     dev(self.g, np.float32), dev(self.h, np.float32)]
        self.desc = aetcnn.LogitsDesc(rows.rows, n, rows.kind, t, rows.stride)

    def call(self, stream=None):
        check(self.gpu.ach_logprobs_bwd(C.byref(self.desc), self.rows.ptr,
                                        *[ptr(b) for b in self.bufs], self.out.ptr,
                                        self.out.stride, stream))

    def want(self):
        f64 = lambda a: None if a is None else a.astype(np.float64)  # noqa: E731
        return ref.logprobs_bwd(self.rows.x, self.h_ids, self.t, f64(self.stats),
                                f64(self.entropy), f64(self.g), f64(self.h), self.rows.kind)


@pytest.mark.parametrize("rows,n,kind,t,pad,shift,opad,oshift", BACKWARD)
@pytest.mark.parametrize("which", ["both", "logprobs", "entropy"])
def test_logprobs_backward(gpu, rows, n, kind, t, pad, shift, opad, oshift, which):
    rng = np.random.default_rng(rows + n)
    x = Rows(sample(rng, rows, n), kind, pad, shift)
    ids = rng.integers(0, n, rows)
    ids[rng.random(rows) < 0.2] = -1
    g = rng.standard_normal(rows) if which != "entropy" else None
    h = rng.standard_normal(rows) * 0.3 if which != "logprobs" else None
    b = Backward(gpu, x, ids if g is not None else None, t, g, h, like(x, opad, oshift))
    b.call()
    near(b.out.read(), b.want(), "dlogits")
    x.read()


@pytest.mark.parametrize("n", [17, 1000, 9001, 131072])
def test_logprobs_backward_in_place_and_masked(gpu, n):
    """dlogits in the logits' memory; masked classes; rows without gradient
    are zeroed whatever their logits hold"""
    rng = np.random.default_rng(n)
    x = sample(rng, 7, n)
    x[0, rng.random(n) < 0.6] = -np.inf
    x[1] = -np.inf                     # no distribution
    x[2] = np.nan                      # ignored
    x[3, 3] = np.inf                   # its weights are zero
    x[4, 1:] = -np.inf                 # certain
    rows = Rows(x, F32, pad=3)
    ids = np.array([int(x[0].argmax()), 2, -1, 0, 0, n, n - 1])
    g = np.array([1.0, 1, np.nan, 0, 1, 1, -2])
    h = np.array([0.5, 1, 0, 0, 1, 0, 0.25])
    b = Backward(gpu, rows, ids, 1.0, g, h, rows)
    want = b.want()
    b.call()
    got = rows.read()
    near(got, want, "dlogits")
    for r in (1, 2, 3, 5):
        assert not got[r].any(), r


def test_logprobs_gradient_against_differences(gpu):
    """central differences of the kernel's own outputs, h = 2^-5: truncation
    h^2/6 |f'''| with |f'''| <= 6 (|g| + |h| log n), rounding 2^-23 |f| / h"""
    rng = np.random.default_rng(8)
    n = 24
    base = rng.standard_normal(n).astype(np.float32)
    h = 2.0 ** -5
    x = np.repeat(base[None], 2 * n, 0)
    x[np.arange(n), np.arange(n)] += h
    x[n + np.arange(n), np.arange(n)] -= h
    rows = Rows(x, F32)
    ids = np.full(2 * n, 3)
    f = Forward(gpu, rows, ids, 0, 1.0)
    f.call()
    got = f.read()
    g, e = 0.75, -0.5
    val = g * got["logprobs"].astype(np.float64) + e * got["entropy"]
    diff = (val[:n] - val[n:]) / (rows.x[np.arange(n), np.arange(n)] - rows.x[n + np.arange(n), np.arange(n)])
    one = Rows(base[None], F32)
    b = Backward(gpu, one, np.array([3]), 1.0, [g], [e], like(one))
    b.call()
    tol = h * h * (g + 0.5 * np.log(n)) + 2.0 ** -23 * np.abs(val).max() / h * 4
    assert np.abs(b.out.read()[0] - diff).max() < tol


class Distill:
    def __init__(self, gpu, rows, ids, values, labels, weights, t, mode, soft, hard, out=None,
                 vkind=F32, outputs=("loss", "delta", "cost")):
        self.gpu, self.rows, self.t, self.mode = gpu, rows, t, mode
        self.soft, self.hard, self.outputs = float(np.float32(soft)), float(np.float32(hard)), outputs
        self.h_ids, self.h_labels = ids, labels
        k = 0 if ids is None else ids.shape[1]
        vbits = None if values is None else ref.to_bits(values, vkind)
        self.h_values = None if values is None else ref.from_bits(vbits, vkind)
        self.h_weights = None if weights is None else np.asarray(weights, np.float32)
        self.out = like(rows) if out is None else out
        self.loss, self.cost = D(rows.rows), D(1)
        self.loss.upload(np.full(rows.rows, np.nan, np.float32))
        self.bufs = [dev(ids, np.int32), dev(vbits, BITS[vkind]), dev(labels, np.int32),
                     dev(self.h_weights, np.float32)]
        self.desc = aetcnn.LogitsDesc(rows.rows, rows.n, rows.kind, t, rows.stride)
        self.teacher = aetcnn.DistillDesc(k, mode, vkind, soft, hard)
        self.nb = gpu.ach_distill_workspace(C.byref(self.desc), C.byref(self.teacher))
        self.ws = D(max(self.nb, 4), np.uint8)
        self.ws.upload(np.full(self.ws.shape, 0xff, np.uint8))

    def call(self, stream=None, ws=None):
        has = lambda name, p: p if name in self.outputs else None  # noqa: E731
        check(self.gpu.ach_distill_xent(
            C.byref(self.desc), C.byref(self.teacher), self.rows.ptr, *[ptr(b) for b in self.bufs],
            has("loss", self.loss.ptr), has("delta", self.out.ptr), self.out.stride,
            has("cost", self.cost.ptr), ws or self.ws.ptr, self.nb, stream))

    def want(self):
        return ref.distill(self.rows.x, self.h_ids, self.h_values, self.h_labels, self.h_weights,
                           float(np.float32(self.t)), self.mode == DISTILL_TAIL, self.soft,
                           self.hard, self.rows.kind)

    def check(self, want=None, stream=None):
        loss, lerr, delta, derr = self.want() if want is None else want
        if "loss" in self.outputs:
            near(self.loss.numpy(stream), (loss, lerr), "loss")
        if "delta" in self.outputs:
            near(self.out.read(), (delta, derr), "delta")
        if "cost" in self.outputs:
            total = loss.sum()
            near(self.cost.numpy(stream)[0], (total, lerr.sum() + 2 * ref.U * np.abs(loss).sum()),
                 "cost")


def teacher(rng, x, k, tail, t):
    """a teacher near the student: its k best, log probabilities"""
    with np.errstate(invalid="ignore"):
        y = np.where(np.isfinite(x), x, -50.0) * 0.6 + rng.standard_normal(x.shape)
    y /= t if tail else 1
    y -= np.log(np.exp(y - y.max(1, keepdims=True)).sum(1, keepdims=True)) + y.max(1, keepdims=True)
    ids = np.argsort(-y, axis=1, kind="stable")[:, :k]
    return ids, np.take_along_axis(y, ids, 1)


DISTILL = [
    # rows, classes, type, k, temperature, pad, shift, pad of delta, teacher's type
    (1, 1, F32, 1, 1.0, 0, 0, 0, F32),
    (3, 2, BF16, 1, 2.0, 1, 1, 0, F32),
    (16, 10, F32, 3, 4.0, 0, 0, 0, F32),
    (5, 64, F16, 64, 1.0, 0, 0, 1, F16),       # every class listed
    (7, 65, BF16, 64, 1.0, 0, 3, 0, BF16),     # all but one
    (128, 1000, F32, 10, 4.0, 0, 0, 0, F32),
    (9, 1001, F16, 128, 0.5, 2, 0, 0, F32),
    (3, 2049, BF16, 17, 1.0, 0, 1, 3, F16),
    (700, 3001, F32, 5, 1.0, 0, 0, 0, F32),
    (3, 8193, F16, 64, 2.0, 1, 0, 0, F32),
    (300, 20011, BF16, 9, 1.0, 0, 0, 0, BF16),
    (2, 50021, F32, 128, 1.0, 0, 0, 1, F32),
    (2, 40000, BF16, 33, 3.0, 0, 0, 0, F32),   # rows in parts, at other temperatures
    (5, 20000, F32, 7, 4.0, 0, 0, 0, F32),
    (300, 30011, F32, 12, 1.0, 0, 0, 0, F32),  # more than the caches hold
    (1, 131072, BF16, 64, 1.0, 0, 0, 0, F32),
    (3, 131073, F32, 64, 2.0, 0, 1, 0, F32),
    (2, 200001, F16, 20, 1.0, 3, 1, 0, F32),
]


@pytest.mark.parametrize("rows,n,kind,k,t,pad,shift,dpad,vkind", DISTILL)
@pytest.mark.parametrize("mode", [DISTILL_RENORM, DISTILL_TAIL])
@pytest.mark.parametrize("hard", [0.0, 0.5])
def test_distill(gpu, rows, n, kind, k, t, pad, shift, dpad, vkind, mode, hard):
    rng = np.random.default_rng(rows + n + k)
    x = Rows(sample(rng, rows, n), kind, pad, shift)
    ids, values = teacher(rng, x.x, k, mode == DISTILL_TAIL, t)
    labels = np.where(rng.random(rows) < 0.5, ids[:, 0], rng.integers(0, n, rows))
    labels[rng.random(rows) < 0.2] = -1
    weights = rng.uniform(0.2, 2, rows)
    weights[rng.random(rows) < 0.2] = 0
    d = Distill(gpu, x, ids, values, labels if hard else None, weights, t, mode, 1 - hard / 2,
                hard, like(x, dpad, shift), vkind)
    d.call()
    d.check()
    x.read()


@pytest.mark.parametrize("n,kind", [(10, F32), (300, BF16), (5000, F32), (131072, F16)])
@pytest.mark.parametrize("mode", [DISTILL_RENORM, DISTILL_TAIL])
def test_distill_odd_teachers(gpu, n, kind, mode):
    """entries that are none or repeated, log probabilities of -inf, more
    probability than 1, no teacher at all, labels in and out of the list,
    masked students, rows of no weight with anything in them"""
    rng = np.random.default_rng(n)
    k = 8
    x = sample(rng, 14, n)
    x[6, rng.random(n) < 0.5] = -np.inf
    x[7] = -np.inf
    x[8] = np.nan
    x[9, n // 2] = np.inf
    rows = Rows(x, kind)
    ids, values = teacher(rng, np.where(np.isfinite(rows.x), rows.x, -9.0), k, mode == DISTILL_TAIL, 1.0)
    ids[0, 2:5] = ids[0, 1]                     # repeated
    ids[1, ::2] = (-1, n, 2 ** 31 - 1, -2 ** 31)
    ids[2] = -1                                 # no teacher
    values[3, 4:] = -np.inf
    values[4] = -np.inf
    values[5] += 0.5                            # sums to more than 1
    ids[6] = np.argsort(-rows.x[6])[:k]         # classes that are not masked
    ids[10] = ids[10, ::-1].copy()
    values[11] = np.log(1e-6)                   # nearly all in the rest
    labels = ids[:, 0].copy()
    labels[0], labels[2], labels[10], labels[12] = ids[0, 1], n - 1, -1, n
    labels[6] = ids[6, 1]
    weights = np.ones(14)
    weights[8] = weights[9] = 0
    for soft, hard in ((1.0, 0.0), (0.5, 0.25), (0.0, 1.0)):
        d = Distill(gpu, rows, ids, values, labels, weights, 1.0, mode, soft, hard)
        d.call()
        d.check()
        got = d.out.read()
        assert not got[[7, 8, 9]].any()


def test_distill_not_finite(gpu):
    """a NaN or +inf among the logits or the teacher's values of a row with a
    weight: its loss and delta are NaN, those of other rows are not"""
    rng = np.random.default_rng(3)
    for n, kind in ((10, F32), (1000, BF16), (9000, F32), (131072, BF16)):
        x = sample(rng, 5, n)
        x[1, n - 1] = np.nan
        x[2, 4] = np.inf
        rows = Rows(x, kind)
        for mode in (DISTILL_RENORM, DISTILL_TAIL):
            ids, values = teacher(rng, np.zeros((5, n)), 4, mode == DISTILL_TAIL, 1.0)
            values[3, 1] = np.nan
            d = Distill(gpu, rows, ids, values, None, None, 1.0, mode, 1.0, 0.0)
            d.call()
            loss, got = d.loss.numpy(), d.out.read()
            assert np.isnan(loss[1:4]).all() and np.isfinite(loss[[0, 4]]).all()
            assert np.isnan(got[1:4]).all() and np.isfinite(got[[0, 4]]).all()
            assert np.isnan(d.cost.numpy()[0])


def test_distill_masked_by_the_student(gpu):
    """the teacher gives probability to a class that the student has masked:
    the loss is +inf, the delta finite; a rest without a class of finite logit
    is left out"""
    for n in (12, 3000, 131072):
        x = np.full((2, n), -np.inf)
        x[:, :6] = np.arange(6)
        rows = Rows(x, F32)
        ids = np.array([[5, 7], [5, 4]])
        values = np.log([[0.5, 0.25], [0.5, 0.25]])
        d = Distill(gpu, rows, ids, values, None, None, 1.0, DISTILL_RENORM, 1.0, 0.0)
        d.call()
        assert np.isposinf(d.loss.numpy()[0]) and np.isfinite(d.loss.numpy()[1])
        near(d.out.read(), d.want()[2:], "delta")
        ids6, v6 = np.array([[0, 1, 2, 3, 4, 5]] * 2), np.log(np.full((2, 6), 0.15))
        d = Distill(gpu, rows, ids6, v6, None, None, 1.0, DISTILL_TAIL, 1.0, 0.0)
        d.call()
        d.check()


@pytest.mark.parametrize("n", [12, 3000, 131072])
def test_labels_of_masked_classes(gpu, n):
    """the loss of a label that the student has masked is +inf, its delta finite"""
    rng = np.random.default_rng(n)
    x = sample(rng, 3, n)
    x[0, n - 1] = -np.inf
    x[1, :-1] = -np.inf
    rows = Rows(x, F32)
    ids, values = teacher(rng, rows.x, 4, True, 1.0)
    labels = np.array([n - 1, 0, 5])
    for soft in (0.0, 0.5):
        d = Distill(gpu, rows, ids, values, labels, None, 1.0, DISTILL_TAIL, soft, 0.5)
        d.call()
        loss, got = d.loss.numpy(), d.out.read()
        assert np.isposinf(loss[:2]).all() and np.isfinite(loss[2]) and np.isfinite(got).all()
        assert np.isposinf(d.cost.numpy()[0])
        near(got, d.want()[2:], "delta")


@pytest.mark.parametrize("n", [12, 3000, 131072])
@pytest.mark.parametrize("kind", [F32, BF16])
def test_largest_numbers(gpu, n, kind):
    """logits at both ends of the type, whose differences overflow"""
    rng = np.random.default_rng(n)
    big = 3.3895313892515355e38
    x = sample(rng, 4, n)
    x[0, 3], x[0, 5] = big, -big
    x[1] = rng.choice([big, -big], n)
    x[2, ::2] = -big
    x[3] = -big
    x[3, n // 2] = big
    rows = Rows(x, kind)
    ids = np.array([3, 5, n - 1, n // 2])
    for t in (1.0, 0.25):
        f = Forward(gpu, rows, ids, 4, t)
        f.call()
        got = f.read()
        with np.errstate(over="ignore"):
            want = ref.logprobs(rows.x, ids, 4, t)
        for name, v in got.items():
            value, bound = want[name]  # beyond the largest number: -inf
            if value.dtype == np.float64:
                value = np.where(np.abs(value) > 3.5e38, np.copysign(np.inf, value), value)
            near(v, (value, bound), name)
    d = Distill(gpu, rows, np.array([[3, 1]] * 4), np.log(np.full((4, 2), 0.25)), None,
                [1.0, 1, 1, 1], 1.0, DISTILL_TAIL, 1.0, 0.0)
    d.call()
    got = d.out.read()
    # a row's deltas add up to 0; their sizes to 2 at most, each rounded by up to 2^-8
    assert np.isfinite(got).all() and np.abs(got.sum(1)).max() < 2 * 2.0 ** -8 + 1e-3


@pytest.mark.parametrize("outputs", [("loss",), ("delta",), ("cost",), ("loss", "cost"),
                                     ("delta", "cost")])
@pytest.mark.parametrize("n", [100, 4000, 131072])
def test_distill_each_output(gpu, outputs, n):
    rng = np.random.default_rng(n)
    x = Rows(sample(rng, 5, n), BF16)
    ids, values = teacher(rng, x.x, 12, True, 1.0)
    d = Distill(gpu, x, ids, values, ids[:, 1].copy(), None, 1.0, DISTILL_TAIL, 0.5, 0.5,
                outputs=outputs)
    d.call()
    d.check()


@pytest.mark.parametrize("rows,n", [(4, 33), (6, 2000), (5, 70000), (600, 6000)])
def test_distill_in_place(gpu, rows, n):
    rng = np.random.default_rng(n)
    x = Rows(sample(rng, rows, n), F32, pad=1)
    ids, values = teacher(rng, x.x, 16, True, 1.0)
    d = Distill(gpu, x, ids, values, ids[:, 3].copy(), None, 1.0, DISTILL_TAIL, 0.5, 0.5, out=x)
    want = d.want()
    d.call()
    d.check(want)


def test_distill_gradient_against_differences(gpu):
    """central differences of the kernel's own losses, h = 2^-5: truncation
    h^2/6 |f'''| with |f'''| <= 6 (soft T^2/T^3 + hard), rounding 2^-23 |f| / h"""
    rng = np.random.default_rng(9)
    n, t, h = 20, 2.0, 2.0 ** -5
    base = rng.standard_normal(n).astype(np.float32)
    ids, values = teacher(rng, base[None].astype(np.float64), 5, True, t)
    x = np.repeat(base[None], 2 * n, 0)
    x[np.arange(n), np.arange(n)] += h
    x[n + np.arange(n), np.arange(n)] -= h
    rows = Rows(x, F32)
    for mode in (DISTILL_RENORM, DISTILL_TAIL):
        d = Distill(gpu, rows, np.repeat(ids, 2 * n, 0), np.repeat(values, 2 * n, 0),
                    np.full(2 * n, 7), None, t, mode, 0.75, 0.5)
        d.call()
        loss = d.loss.numpy().astype(np.float64)
        step = rows.x[np.arange(n), np.arange(n)] - rows.x[n + np.arange(n), np.arange(n)]
        diff = (loss[:n] - loss[n:]) / step
        one = Rows(base[None], F32)
        e = Distill(gpu, one, ids, values, np.array([7]), None, t, mode, 0.75, 0.5)
        e.call()
        tol = h * h * (0.75 / t + 0.5) + 2.0 ** -23 * np.abs(loss).max() / h * 4
        assert np.abs(-e.out.read()[0] - diff).max() < tol


def test_offsets_past_32_bits(gpu):
    """rows 2^31 and more elements apart"""
    rng = np.random.default_rng(4)
    n, stride = 5003, (1 << 31) + 77
    x = sample(rng, 2, n)
    bits = ref.to_bits(x, BF16)
    xs = ref.from_bits(bits, BF16)
    big = aetcnn.DeviceArray(((stride + n) * 2,), np.uint8)
    out = aetcnn.DeviceArray(((stride + n) * 2,), np.uint8)

    class Far:
        rows, kind = 2, BF16

    far = Far()
    far.n, far.stride, far.ptr, far.x = n, stride, big.ptr, xs
    for r in range(2):
        check(gpu.ach_memcpy_h2d(big.ptr + r * stride * 2, bits[r].ctypes.data, n * 2, None))
    ids = np.array([3, int(xs[1].argmax())])
    _, got = check_forward(gpu, far, ids, 20, 1.0)

    def read():
        a = np.empty((2, n), np.uint16)
        for r in range(2):
            check(gpu.ach_memcpy_d2h(a[r].ctypes.data, out.ptr + r * stride * 2, n * 2, None))
        return ref.from_bits(a, BF16)

    far_out = Far()
    far_out.n, far_out.stride, far_out.ptr, far_out.read = n, stride, out.ptr, read
    b = Backward(gpu, far, ids, 1.0, [1.0, -0.5], [0.1, 0.2], far_out)
    b.call()
    near(read(), b.want(), "dlogits")
    tids, values = teacher(rng, xs, 8, True, 1.0)
    d = Distill(gpu, far, tids, values, ids, None, 1.0, DISTILL_TAIL, 0.5, 0.5, out=far_out)
    d.call()
    d.check()


def test_more_rows_than_workgroups(gpu):
    """over 2^20 rows: a workgroup takes several"""
    rows, n, period = (1 << 20) + 1000, 3, 1003
    rng = np.random.default_rng(2)
    some = sample(rng, period, n)
    some[5, 1] = -np.inf
    some[6] = -np.inf
    x = Rows(np.resize(some, (rows, n)), BF16)
    few = Rows(some, BF16)
    ids = np.resize(rng.integers(-1, n, period), rows)
    f, got = check_forward(gpu, x, ids, 2, 1.0)
    b = Backward(gpu, x, ids, 1.0, np.ones(rows), np.ones(rows), like(x))
    b.call()
    near(b.out.read(), b.want(), "dlogits")
    tids, values = teacher(rng, few.x, 2, True, 1.0)
    w = rng.uniform(0, 1, period)
    w[9] = 0
    args = [np.resize(a, (rows,) + a.shape[1:]) for a in (tids, values, ids[:period], w)]
    d = Distill(gpu, x, *args, 1.0, DISTILL_TAIL, 0.5, 0.5)
    e = Distill(gpu, few, tids, values, ids[:period], w, 1.0, DISTILL_TAIL, 0.5, 0.5)
    d.call()
    e.call()
    e.check()
    assert np.array_equal(d.out.read(), np.resize(e.out.read(), (rows, n)))
    loss = d.loss.numpy()
    assert np.array_equal(loss, np.resize(e.loss.numpy(), rows))
    total = loss.astype(np.float64).sum()
    assert abs(d.cost.numpy()[0] - total) <= 2 * ref.U * abs(total)


class Hip:
    """Graph capture through the HIP runtime that the library uses."""

    def __init__(self):
        self.lib = C.CDLL("libamdhip64.so")

    def do(self, name, *args):
        rc = getattr(self.lib, name)(*args)
        assert rc == 0, (name, rc)

    def capture(self, stream, work):
        graph, ex = C.c_void_p(), C.c_void_p()
        self.do("hipStreamBeginCapture", C.c_void_p(stream), 0)
        work()
        self.do("hipStreamEndCapture", C.c_void_p(stream), C.byref(graph))
        self.do("hipGraphInstantiate", C.byref(ex), graph, None, None, C.c_size_t(0))
        return ex

    def launch(self, ex, stream):
        self.do("hipGraphLaunch", ex, C.c_void_p(stream))


@pytest.fixture
def stream(gpu):
    s = C.c_void_p()
    check(gpu.ach_stream_create(C.byref(s)))
    yield s.value
    check(gpu.ach_stream_destroy(s.value))


def bits(f, d):
    """the bits of all outputs of a forward call and a distillation"""
    return b"".join([v.tobytes() for _, v in sorted(f.read().items())] +
                    [a.tobytes() for a in (d.loss.numpy(), d.out.read(), d.cost.numpy())])


def test_graph_replays(gpu, stream):
    """captured, then replayed with other inputs, with eager calls between;
    two graphs share a workspace"""
    hip = Hip()
    rng = np.random.default_rng(12)
    x = [Rows(sample(rng, r, n), kind) for r, n, kind in ((2, 100003, F32), (40, 1000, BF16))]
    calls, graphs = [], []
    for rows in x:
        ids, values = teacher(rng, rows.x, 16, True, 1.0)
        d = Distill(gpu, rows, ids, values, ids[:, 0].copy(), None, 1.0, DISTILL_TAIL, 0.5, 0.5)
        f = Forward(gpu, rows, ids[:, 0], 16, 1.0)
        calls.append((d, f))
    ws = D(max(max(d.nb, f.nb) for d, f in calls), np.uint8)
    for d, f in calls:
        d.ws = f.ws = ws
        graphs.append(hip.capture(stream, lambda: (f.call(stream), d.call(stream))))
    for replay in range(4):
        for i, (d, f) in enumerate(calls):
            rows = x[i]
            new = Rows(sample(rng, rows.rows, rows.n), rows.kind)
            rows.dev.upload(new.raw)
            rows.bits, rows.x, rows.raw = new.bits, new.x, new.raw
        for g in graphs:
            hip.launch(g, stream)
        check(gpu.ach_stream_sync(stream))
        for d, f in calls:
            d.check()
            want = ref.logprobs(f.rows.x, d.h_ids[:, 0], 16, 1.0)
            got = f.read()
            for name, v in got.items():
                near(v, want[name], name)
            graph = bits(f, d)
            f.call(stream)   # eager, between the replays
            d.call(stream)
            check(gpu.ach_stream_sync(stream))
            assert graph == bits(f, d)


def test_two_streams_at_once(gpu, stream):
    """calls on two streams with a workspace each, in flight together"""
    rng = np.random.default_rng(13)
    other = C.c_void_p()
    check(gpu.ach_stream_create(C.byref(other)))
    jobs = []
    for s in (stream, other.value):
        x = Rows(sample(rng, 3, 131072), BF16)
        ids, values = teacher(rng, x.x, 32, True, 1.0)
        jobs.append((s, Distill(gpu, x, ids, values, None, None, 1.0, DISTILL_TAIL, 1.0, 0.0),
                     Forward(gpu, x, ids[:, 2], 32, 1.0)))
    for _ in range(5):
        for s, d, f in jobs:
            f.call(s)
            d.call(s)
    for s, d, f in jobs:
        check(gpu.ach_stream_sync(s))
        d.check()
        want = ref.logprobs(f.rows.x, d.h_ids[:, 2], 32, 1.0)
        for name, v in f.read().items():
            near(v, want[name], name)
    check(gpu.ach_stream_destroy(other.value))


@pytest.mark.parametrize("n,kind", [(1000, F32), (13000, BF16), (20000, BF16), (131072, F32)])
def test_runs_are_equal(gpu, n, kind):
    """no result depends on the order in which anything ran"""
    rng = np.random.default_rng(n)
    x = Rows(np.round(sample(rng, 20, n) * 4) / 4, kind)  # many equal logits
    ids, values = teacher(rng, x.x, 128, True, 1.0)
    d = Distill(gpu, x, ids, values, ids[:, 1].copy(), None, 1.0, DISTILL_TAIL, 0.5, 0.5)
    f = Forward(gpu, x, ids[:, 0], 64, 1.0)
    seen = set()
    for _ in range(12):
        f.call()
        d.call()
        seen.add(bits(f, d))
    assert len(seen) == 1


@pytest.mark.parametrize("classes", [10, 1000, 40000])
def test_teacher_to_student(gpu, classes):
    """As they are used together: a teacher's top alternatives are the entries
    of a student's distillation, whose delta moves the student, whose log
    probabilities of the teacher's best classes then rise; and a student equal
    to its teacher has no loss and no delta beyond rounding."""
    rng = np.random.default_rng(classes)
    rows, k, t = 32, min(classes // 2, 32), 2.0
    ty = Rows(sample(rng, rows, classes, 2.0), F32)
    f = Forward(gpu, ty, None, k, t, outputs=())
    f.call()
    top = f.read()
    same = Distill(gpu, ty, top["top_ids"], top["top_logprobs"], None, None, t, DISTILL_TAIL, 1.0, 0.0)
    # the entries and workspace stay on the device in use; here they are the call's own buffers
    same.bufs[0], same.bufs[1] = f.out["top_ids"], f.out["top_logprobs"]
    same.call()
    same.check()
    assert np.abs(same.loss.numpy()).max() < t * t * 64 * 2.0 ** -23 * (8 + np.log(classes))
    sx = Rows(rng.standard_normal((rows, classes)) * 0.1, F32)
    last = None
    for _ in range(3):
        d = Distill(gpu, sx, top["top_ids"], top["top_logprobs"], None, None, t, DISTILL_TAIL, 1.0, 0.0)
        d.bufs[0], d.bufs[1] = f.out["top_ids"], f.out["top_logprobs"]
        d.call()
        d.check()
        a = Forward(gpu, sx, top["top_ids"][:, 0], 0, t)
        a.call()
        sx = Rows(sx.x + 0.5 * d.out.read(), F32)
        b = Forward(gpu, sx, top["top_ids"][:, 0], 0, t)
        b.call()
        assert (b.read()["logprobs"] > a.read()["logprobs"]).all()
