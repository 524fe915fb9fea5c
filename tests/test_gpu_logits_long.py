"""Long rows, to the last logit.  A lost or doubled logit among a hundred thousand
moves a sum by less than the error bound of ordinary rows: here the finite logits
are equal, so that sums are counts, exact in 32 bits, and one logit more or
less shows.  The rows reach what only long ones do: groups of several turns in
the search for the best, a second and a third segment of 32 turns in distillation,
parts of more than one segment.  Rows repeat: every copy has the first one's
result, bit by bit."""
import ctypes as C

import numpy as np
import pytest

import aetcnn
import logits_ref as ref
from aetcnn import BF16, F16, F32, DISTILL_RENORM, DISTILL_TAIL, check
from aetcnn import DeviceArray as D
from test_gpu_logits import Distill, Forward, Rows, near, sample, teacher

pytestmark = pytest.mark.gpu

U = ref.U
SIZE = {F32: 4, BF16: 2, F16: 2}


class Repeated:
    """the given rows over and over, `rows` in all, on the device"""

    def __init__(self, gpu, few, rows):
        self.kind, self.rows, self.n, self.stride, self.few = few.kind, rows, few.n, few.n, few
        self.period = few.rows
        row = few.n * SIZE[few.kind]
        self.dev = D(rows * row, np.uint8)
        self.ptr = self.dev.ptr
        for r in range(0, rows, few.rows):
            check(gpu.ach_memcpy_d2d(self.ptr + r * row, few.ptr, min(few.rows, rows - r) * row,
                                     None))

    def first(self):
        """the first rows as numbers, after a look at the others"""
        kind = {F32: np.float32, BF16: np.uint16, F16: np.float16}[self.kind]
        a = self.dev.numpy().view(kind).reshape(self.rows, self.n)
        return ref.from_bits(copies(a, self.period), self.kind)


def copies(a, period):
    for r in range(period, len(a), period):
        part = a[r:r + period]
        assert np.array_equal(part, a[:len(part)]), r
    return a[:period].copy()


def blank(gpu, x):
    """an output like x, of NaN"""
    return Repeated(gpu, Rows(np.full((1, x.n), np.nan), x.kind), x.rows)


def repeat(a, rows):
    return np.resize(a, (rows,) + a.shape[1:])


ROWS = 8


@pytest.mark.parametrize("rows,n,kind,k", [
    (264, 140001, F32, 20),     # two turns a group, of workgroups of 512 threads
    (264, 290003, BF16, 128),
    (1032, 70001, F32, 64),     # two, of 256
    (1032, 139999, F16, 20),
    (1032, 150001, F32, 33),    # four
])
def test_best_of_long_rows(gpu, rows, n, kind, k):
    rng = np.random.default_rng(n)
    j = np.arange(n)
    x = sample(rng, ROWS, n)
    x[1] = j / 1024                                  # ascending: every group has larger ones
    x[2] = -j / 1024
    x[3, rng.random(n) < 0.7] = -np.inf
    x[4] = np.where(rng.random(n) < 1e-3, 1.0, -np.inf)
    x[5, n - k - 3:] = 40 + np.arange(k + 3) % 5     # the best behind the last turn
    at = rng.permutation(n // 4096)[:k] * 4096 + 4095
    x[6, at] = 50 - np.arange(len(at)) / 8           # at the ends of turns
    x[7] = 1.0                                       # equal
    few = Rows(x, kind)
    ids = few.x.argmax(1)
    ids[::2] = n - 1
    f = Forward(gpu, Repeated(gpu, few, rows), repeat(ids, rows), k, 1.0)
    f.call()
    want = ref.logprobs(few.x, ids, k, 1.0)
    for name, v in f.read().items():
        near(copies(v, ROWS), want[name], name)


def equal_rows(n, lists):
    """Rows of equal finite logits: all; those at both sides of every multiple
    of 64 (a chunk, a wave's turn, a turn, a part and a segment end at such
    places); at every 61st place; the last two; two at a segment's end; and the
    listed classes alone.  Others are masked."""
    j = np.arange(n)
    on = np.stack([np.ones(n, bool), (j % 64 == 63) | (j % 64 == 0), j % 61 == 7, j >= n - 2,
                   (j == n // 2) | (j == n // 2 - 1), np.isin(j, lists)])
    return np.where(on, 0.75, -np.inf), on


EQUAL = [
    # rows in all, classes, type
    (6, 12, F32), (6, 1000, F16), (1500, 2051, BF16), (1500, 8192, BF16), (600, 9001, F32),
    (600, 33003, BF16), (1032, 33003, F32), (264, 70001, F32), (1032, 70001, F32),
    (264, 140001, F32), (264, 282003, F16), (264, 270005, F32),
    (1, 131072, BF16), (6, 131071, F32), (6, 200001, F16), (60, 100003, BF16), (200, 70001, F32),
    (198, 280001, F32),
]


def close(got, value, parts):
    """value formed from terms of the sizes `parts`: a function of log's kind is
    within 2 steps (4 U), the sums and products of them within 4 U more"""
    assert np.isfinite(got).all()
    assert (np.abs(got - value) <= 8 * U * parts + 2.0 ** -126).all(), (got, value)


@pytest.mark.parametrize("rows,n,kind", EQUAL)
def test_equal_logits_forward(gpu, rows, n, kind):
    lists = [n - 1, n // 3]
    x, on = equal_rows(n, lists)
    x, on = x[:rows], on[:rows]
    few, count = Rows(x, kind), on.sum(1)
    k = min(n, 7)
    last = np.array([np.flatnonzero(o)[-1] for o in on])
    f = Forward(gpu, Repeated(gpu, few, rows), repeat(last, rows), k, 1.0)
    f.call()
    got = {name: copies(v, len(x)) for name, v in f.read().items()}
    log = np.log(count)
    assert (got["stats"][:, 0] == 0.75).all() and not got["ranks"].any()
    # log1p of an exact count is within 2 steps: one logit in 300000 is 3.3e-6,
    # more than these 4 U log(n) = 3.0e-6
    assert (np.abs(got["stats"][:, 1] - log) <= 4 * U * log).all()
    assert (np.abs(got["logprobs"] + log) <= 4 * U * log).all()
    assert (np.abs(got["entropy"] - log) <= 4 * U * log).all()
    for r, o in enumerate(on):
        best = np.flatnonzero(o)[:k]
        rest = np.flatnonzero(~o)[:k - len(best)]
        assert np.array_equal(got["top_ids"][r], np.concatenate((best, rest)))
        assert (np.abs(got["top_logprobs"][r, :len(best)] + log[r]) <= 4 * U * log[r]).all()
        assert np.isneginf(got["top_logprobs"][r, len(best):]).all()


@pytest.mark.parametrize("rows,n,kind", EQUAL)
@pytest.mark.parametrize("soft,hard,t,mode", [(0.0, 1.0, 1.0, DISTILL_RENORM),
                                              (1.0, 0.0, 1.0, DISTILL_RENORM),
                                              (0.5, 0.5, 1.0, DISTILL_TAIL),
                                              (0.5, 0.25, 2.0, DISTILL_TAIL),
                                              (0.5, 0.25, 3.0, DISTILL_RENORM)])
def test_equal_logits_distilled(gpu, rows, n, kind, soft, hard, t, mode):
    """c equal logits, the teacher with 1/8 for each of four of them: KD is
    log c - log 4 (the four made to sum to 1), or 1/2 (log c - log 8) and for
    the c - 4 others 1/2 (log(1/2) - log((c - 4)/c)).  The deltas are
    -soft T (1/c - p) and -hard (1/c - [label])."""
    lists = np.array([0, 131072 % n, n - 1, n // 2 + 1])
    if len(set(lists)) < 4:
        lists = np.arange(4) * (n // 4)
    x, on = equal_rows(n, lists)
    x[:, lists], on[:, lists] = 0.75, True   # every row has finite logits there
    x, on = x[:rows], on[:rows]
    few, c = Rows(x, kind), on.sum(1).astype(np.float64)
    label = int(lists[2])
    big = Repeated(gpu, few, rows)
    d = Distill(gpu, big, repeat(lists[None], rows), np.full((rows, 4), np.log(0.125)),
                np.full(rows, label), None, t, mode, soft, hard, out=blank(gpu, big))
    d.call()
    loss = copies(d.loss.numpy(), len(x)).astype(np.float64)
    tail = mode == DISTILL_TAIL
    with np.errstate(divide="ignore", invalid="ignore"):
        rest = np.where(c > 4, 0.5 * (np.log(0.5) - np.log((c - 4) / c)), 0) if tail else 0
        per_rest = np.where(c > 4, 0.5 / (c - 4), 0) if tail else 0
    kd = 0.5 * (np.log(c) - np.log(8)) + rest if tail else np.log(c) - np.log(4)
    sizes = np.log(c) + np.log(8) + (np.abs(rest) + np.log(2) if tail else 0)
    close(loss, soft * t * t * kd + hard * np.log(c), soft * t * t * sizes + hard * np.log(c))
    total = repeat(loss, rows).sum()
    assert abs(d.cost.numpy()[0] - total) <= 2 * U * np.abs(repeat(loss, rows)).sum()
    out = d.out
    out.period = len(x)
    delta = out.first()
    p = 0.25 if not tail else 0.125
    P = np.where(c > 4, 1.0, 0.5) if tail else 1.0
    dense = soft * t * (P / c - per_rest) + hard / c
    off = soft * t * (P / c - p) + hard / c
    half = ref.EPS[kind] / 2
    for r, o in enumerate(on):
        unlisted = o.copy()
        unlisted[lists] = False
        assert not delta[r, ~o].any()
        got = np.unique(delta[r, unlisted])
        assert len(got) == min(1, unlisted.sum())
        for v, value, size in [(g, -dense[r], soft * t / (c[r] - 4) + hard / c[r]) for g in got] + \
                [(delta[r, lists[i]], -(off[r] - (hard if i == 2 else 0)), soft * t + hard)
                 for i in range(4)]:
            tol = 16 * U * size + half * max(abs(value), ref.TINY[kind])
            assert abs(v - value) <= tol, (r, v, value)


@pytest.mark.parametrize("rows,n,kind,k,t,mode", [
    (264, 140001, F32, 64, 1.0, DISTILL_TAIL),      # a second segment
    (264, 282003, BF16, 17, 2.0, DISTILL_RENORM),
    (264, 270005, F32, 128, 3.0, DISTILL_RENORM),   # a third
    (198, 280001, F32, 20, 4.0, DISTILL_TAIL),      # parts of two segments
])
def test_distillation_of_long_rows(gpu, rows, n, kind, k, t, mode):
    rng = np.random.default_rng(n)
    few = Rows(sample(rng, 6, n), kind)
    ids, values = teacher(rng, few.x, k, mode == DISTILL_TAIL, t)
    # listed classes on both sides of where segments and turns end, and at the end
    ids[0, :6] = (131071, 131072, 4095, 4096, n - 1, n - 2)
    ids[1, :4] = (262143 % n, 262144 % n, 139999, 140000)
    for r in range(2):  # entries that repeat these are dropped
        assert len(set(ids[r])) >= k - 6
    labels = np.array([131073, 131071, n - 1, int(ids[3, 0]), -1, 0])
    weights = np.array([1.0, 0.5, 1, 2, 1, 1])
    big = Repeated(gpu, few, rows)
    d = Distill(gpu, big, repeat(ids, rows), repeat(values, rows), repeat(labels, rows),
                repeat(weights, rows), t, mode, 0.5, 0.5, out=blank(gpu, big))
    d.call()
    one = ref.distill(few.x, ids, values, labels, weights, t, mode == DISTILL_TAIL, 0.5, 0.5, kind)
    near(copies(d.loss.numpy(), 6), one[:2], "loss")
    out = d.out
    out.period = 6
    near(out.first(), one[2:], "delta")


def test_gradient_of_long_rows(gpu):
    """the gradient of equal logits: p (a + b log p) of each, to the last"""
    for rows, n, kind in ((264, 140001, F32), (6, 200001, F16), (1, 131072, BF16)):
        x, on = equal_rows(n, [n - 1, n // 3])
        x, on = x[:rows], on[:rows]
        few, c = Rows(x, kind), on.sum(1).astype(np.float64)
        last = np.array([np.flatnonzero(o)[-1] for o in on])
        big = Repeated(gpu, few, rows)
        out = blank(gpu, big)
        out.period = len(x)
        log = np.log(c).astype(np.float32)
        stats = np.stack((np.full(len(x), 0.75, np.float32), log), 1)
        held = [D.from_numpy(np.ascontiguousarray(repeat(a, rows))) for a in
                (last.astype(np.int32), stats, log, np.full(len(x), 0.5, np.float32),
                 np.full(len(x), -0.25, np.float32))]
        desc = aetcnn.LogitsDesc(rows, n, kind, 1.0, n)
        check(gpu.ach_logprobs_bwd(C.byref(desc), big.ptr, *[b.ptr for b in held], out.ptr, 0,
                                   None))
        got = out.first()
        half = ref.EPS[kind] / 2
        for r, o in enumerate(on):
            # log p + entropy is 0: what is left is g ([j == id] - p)
            want = np.where(o, -0.5 / c[r], 0)
            want[last[r]] += 0.5
            err = np.where(o, (0.5 + 0.25) / c[r], 0) * 8 * U * (1 + np.log(c[r])) + \
                half * np.maximum(np.abs(want), ref.TINY[kind])
            err[last[r]] += 4 * U
            assert (np.abs(got[r] - want) <= err).all(), (rows, n, r)
            assert not got[r, ~o].any()
