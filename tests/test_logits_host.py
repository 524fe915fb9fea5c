"""Operators on logits without a GPU: which calls are refused, before anything
is launched, and the 64-bit gradients that the kernels are tested against,
themselves against differences of the losses."""
import ctypes as C

import numpy as np
import pytest

import aetcnn
import logits_ref as ref
from aetcnn import ACH_EINVAL, ACH_EWORKSPACE, DistillDesc, LogitsDesc
from logits_launches import record

MEM = 4096  # an address that is never read: the calls are refused
BIG = 1 << 40


def fwd(ops, d, k=0, logits=MEM, ids=MEM, logprobs=MEM, ranks=None, entropy=None, stats=None,
        top_ids=None, top_logprobs=None, ws=MEM, nb=BIG):
    return ops.ach_logprobs_fwd(C.byref(d) if d else None, logits, ids, k, logprobs, ranks,
                                entropy, stats, top_ids, top_logprobs, ws, nb, None)


def bwd(ops, d, logits=MEM, ids=MEM, stats=MEM, entropy=MEM, g=MEM, h=MEM, out=2 * MEM, stride=0):
    return ops.ach_logprobs_bwd(C.byref(d) if d else None, logits, ids, stats, entropy, g, h, out,
                                stride, None)


def dis(ops, d, t, logits=MEM, ids=MEM, values=MEM, labels=MEM, weights=None, loss=MEM,
        delta=2 * MEM, stride=0, cost=MEM, ws=MEM, nb=BIG):
    return ops.ach_distill_xent(C.byref(d) if d else None, C.byref(t) if t else None, logits, ids,
                                values, labels, weights, loss, delta, stride, cost, ws, nb, None)


BAD_DESCS = [LogitsDesc(-1, 10, 0, 1.0), LogitsDesc(2, 0, 0, 1.0), LogitsDesc(2, -3, 0, 1.0),
             LogitsDesc(2, 10, 3, 1.0), LogitsDesc(2, 10, -1, 1.0), LogitsDesc(2, 10, 0, 0.0),
             LogitsDesc(2, 10, 0, -1.0), LogitsDesc(2, 10, 0, float("nan")),
             LogitsDesc(2, 10, 0, float("inf")), LogitsDesc(2, 10, 0, 1e-7),
             LogitsDesc(2, 10, 0, 1.0, 9), LogitsDesc(2, 10, 0, 1.0, -10), None]


@pytest.mark.parametrize("d", BAD_DESCS)
def test_bad_descriptors(d):
    ops = aetcnn.ops()
    assert fwd(ops, d) == bwd(ops, d) == dis(ops, d, DistillDesc(2, 0, 0, 1, 0)) == ACH_EINVAL
    ref_d = C.byref(d) if d else None
    assert ops.ach_logprobs_workspace(ref_d, 1) == 0
    assert ops.ach_distill_workspace(ref_d, C.byref(DistillDesc(2, 0, 0, 1, 0))) == 0


def test_logprobs_refusals():
    ops = aetcnn.ops()
    d, wide = LogitsDesc(2, 10, aetcnn.F32, 1.0), LogitsDesc(2, 1000, aetcnn.BF16, 1.0)
    top = dict(top_ids=MEM, top_logprobs=MEM)
    assert fwd(ops, d, logits=None) == ACH_EINVAL
    assert fwd(ops, d, logits=MEM + 2) == ACH_EINVAL     # not at an element's address
    assert fwd(ops, wide, logits=MEM + 1) == ACH_EINVAL
    assert fwd(ops, d, ids=None) == ACH_EINVAL           # log probabilities of which classes?
    assert fwd(ops, d, ids=None, logprobs=None, ranks=MEM) == ACH_EINVAL
    assert fwd(ops, d, logprobs=None) == ACH_EINVAL      # nothing asked
    assert fwd(ops, d, k=11, **top) == ACH_EINVAL        # more than there are
    assert fwd(ops, wide, k=129, **top) == ACH_EINVAL    # more than ACH_TOP_MAX
    assert fwd(ops, wide, k=-1, **top) == ACH_EINVAL
    assert fwd(ops, d, k=3, top_ids=MEM) == ACH_EINVAL
    assert fwd(ops, d, k=3, top_logprobs=MEM) == ACH_EINVAL
    few = LogitsDesc(1, 200001, aetcnn.F32, 1.0)         # one long row: in parts
    nb = ops.ach_logprobs_workspace(C.byref(few), 20)
    if nb:
        assert fwd(ops, few, k=20, ws=None, **top) == ACH_EWORKSPACE
        assert fwd(ops, few, k=20, nb=nb - 1, **top) == ACH_EWORKSPACE


def test_logprobs_bwd_refusals():
    ops = aetcnn.ops()
    d = LogitsDesc(2, 10, aetcnn.F16, 1.0, 12)
    assert bwd(ops, d, logits=None) == bwd(ops, d, stats=None) == bwd(ops, d, out=None) == ACH_EINVAL
    assert bwd(ops, d, logits=MEM + 1) == bwd(ops, d, out=MEM + 1) == ACH_EINVAL
    assert bwd(ops, d, g=None, h=None) == ACH_EINVAL
    assert bwd(ops, d, ids=None) == bwd(ops, d, entropy=None) == ACH_EINVAL
    assert bwd(ops, d, stride=9) == bwd(ops, d, stride=-1) == ACH_EINVAL
    assert bwd(ops, d, out=MEM) == bwd(ops, d, out=MEM, stride=10) == ACH_EINVAL  # in place, restrided


def test_distill_refusals():
    ops = aetcnn.ops()
    d = LogitsDesc(3, 1000, aetcnn.BF16, 2.0)
    t = DistillDesc(8, aetcnn.DISTILL_RENORM, aetcnn.F32, 0.5, 0.5)
    inf, nan = float("inf"), float("nan")
    for bad in (DistillDesc(-1, 0, 0, 1, 0), DistillDesc(129, 0, 0, 1, 0), DistillDesc(0, 0, 0, 1, 0),
                DistillDesc(8, 2, 0, 1, 0), DistillDesc(8, -1, 0, 1, 0), DistillDesc(8, 0, 3, 1, 0),
                DistillDesc(8, 0, 0, inf, 0), DistillDesc(8, 0, 0, 1, nan), None):
        assert dis(ops, d, bad) == ACH_EINVAL
        assert ops.ach_distill_workspace(C.byref(d), C.byref(bad) if bad else None) == 0
    assert dis(ops, d, t, logits=None) == dis(ops, d, t, logits=MEM + 1) == ACH_EINVAL
    assert dis(ops, d, t, ids=None) == dis(ops, d, t, values=None) == ACH_EINVAL
    assert dis(ops, d, t, values=MEM + 2) == dis(ops, d, t, labels=None) == ACH_EINVAL
    assert dis(ops, d, t, loss=None, delta=None, cost=None) == ACH_EINVAL
    assert dis(ops, d, t, delta=MEM + 1) == dis(ops, d, t, stride=999) == ACH_EINVAL
    assert dis(ops, d, t, delta=MEM, stride=1001) == ACH_EINVAL
    nb = ops.ach_distill_workspace(C.byref(d), C.byref(t))
    assert nb > 0
    assert dis(ops, d, t, ws=None) == dis(ops, d, t, nb=nb - 1) == ACH_EWORKSPACE


def test_no_rows_no_launch(tmp_path):
    """rows 0: nothing is launched but the sum of no losses"""
    d = {"logits": [0, 1000, 1, 1.0, 0]}
    t = {"distill": [8, 1, 0, 1.0, 0.0]}
    p = "p"
    calls = [["ach_logprobs_fwd", [d, p, p, 5, p, p, p, p, p, p, None, 0, None]],
             ["ach_logprobs_bwd", [d, p, p, p, p, p, p, p, 0, None]],
             ["ach_distill_xent", [d, t, p, p, p, None, None, p, p, 0, None, None, 0, None]],
             ["ach_distill_xent", [d, t, p, p, p, None, None, p, p, 0, p, None, 0, None]]]
    got = record(calls, tmp_path)
    assert [r["rc"] for r in got] == [0] * 4
    assert [len(r["launches"]) for r in got] == [0, 0, 0, 1]


def _differences(f, x, h=1e-5):
    g = np.zeros_like(x)
    for j in range(x.shape[1]):
        a, b = x.copy(), x.copy()
        a[:, j] += h
        b[:, j] -= h
        g[:, j] = (f(a) - f(b)) / (2 * h)
    return g


@pytest.mark.parametrize("tail,hard,t", [(False, 0.0, 1.0), (False, 0.4, 2.5), (True, 0.0, 1.0),
                                         (True, 0.7, 0.5)])
def test_reference_distillation_gradient(tail, hard, t):
    """central differences of the 64-bit loss: truncation h^2/6 |f'''| <= 1e-9,
    rounding 2^-52 |f| / h <= 1e-9"""
    rng = np.random.default_rng(5)
    rows, n, k = 6, 12, 4
    x = rng.standard_normal((rows, n))
    ids = np.stack([rng.permutation(n)[:k] for _ in range(rows)])
    ids[1, 2] = ids[1, 0]      # repeated: dropped
    ids[2, 1] = -1             # none
    ids[3] = -1                # no teacher
    values = np.log(rng.dirichlet(np.ones(k), rows) * 0.8)
    labels = rng.integers(0, n, rows)
    labels[4], labels[5] = ids[4, 0], -1
    w = rng.standard_normal(rows)

    def call(y):
        return ref.distill(y, ids, values, labels, w, t, tail, 0.6, hard, ref.F32)

    want = -_differences(lambda y: call(y)[0], x)
    assert np.abs(call(x)[2] - want).max() < 1e-8


def test_reference_logprobs_gradient():
    rng = np.random.default_rng(6)
    rows, n, t = 5, 9, 1.7
    x, ids = rng.standard_normal((rows, n)), rng.integers(0, n, rows)
    ids[2] = -1
    g, h = rng.standard_normal(rows), rng.standard_normal(rows)

    def value(y):
        o = ref.logprobs(y, ids, 0, t)
        return g * o["logprobs"][0] + h * o["entropy"][0]

    o = ref.logprobs(x, ids, 0, t)
    got, _ = ref.logprobs_bwd(x, ids, t, o["stats"][0], o["entropy"][0], g, h, ref.F32)
    assert np.abs(got - _differences(value, x)).max() < 1e-8


def test_launches(tmp_path):
    """One launch for a forward call but for few long rows, two for these; two
    for a distillation with its cost; dynamic LDS that needs no limit raised."""
    p = "p"
    fwd = [(1, 131072, 2), (64, 100003, 2), (1, 60000, 1), (128, 1000, 1), (1024, 131072, 1),
           (4096, 100, 1), (256, 65536, 2), (257, 65536, 1)]
    calls = [["ach_logprobs_fwd", [{"logits": [r, n, 1, 1.0, 0]}, p, p, 20, p, p, p, p, p, p, p, BIG,
                                   None]] for r, n, _ in fwd]
    dis = [(1, 200001, 2), (16, 131072, 2), (128, 1000, 2), (2048, 131072, 2), (100, 9000, 2)]
    calls += [["ach_distill_xent", [{"logits": [r, n, 0, 2.0, 0]}, {"distill": [64, 1, 0, 0.5, 0.5]},
                                    p, p, p, p, None, p, p, 0, p, p, BIG, None]] for r, n, _ in dis]
    for call, want, got in zip(calls, [w for *_, w in fwd + dis], record(calls, tmp_path)):
        assert got["rc"] == 0 and len(got["launches"]) == want, (call, got)
        for v in got["launches"]:
            assert v["lds"] <= 32768 and v["grid"][1:] == [1, 1]
            assert v["grid"][0] * v["block"][0] < 2 ** 32
