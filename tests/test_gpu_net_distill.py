"""A network's answers as log probabilities (an_predict_top) and its training
from a teacher's answers (an_set_distillation, an_set_teacher)."""
import numpy as np
import pytest

import aetcnn
import logits_ref as ref
from aetcnn import configs

pytestmark = pytest.mark.gpu
BATCH = 8


def network(seed, name="tiny", batch=BATCH):
    aetcnn.net_lib().an_rand_seed(seed)
    net = aetcnn.Network(*configs.dims(name, batch))
    configs.build(net, name)
    net.finalize()
    return net


def logits(net):
    n = net.n_layers()
    return net.buffer(n - 2, 0).reshape(net.batch, -1).astype(np.float64)


@pytest.mark.parametrize("temperature", [1.0, 2.5])
@pytest.mark.parametrize("k", [1, 5, 10])
def test_predict_top(gpu, k, temperature):
    net = network(3)
    x, _, _ = configs.synthetic_batch("tiny", 21, BATCH)
    ids, lp, ent = net.predict_top(x, k, temperature)
    want = ref.logprobs(logits(net), np.full(BATCH, -1), k, temperature)
    assert np.array_equal(ids, want["top_ids"][0])
    assert (np.abs(lp - want["top_logprobs"][0]) <= want["top_logprobs"][1]).all()
    assert (np.abs(ent - want["entropy"][0]) <= want["entropy"][1]).all()
    probs = net.predict(x)  # the same answers as probabilities
    if temperature == 1.0:  # many of them are 0 in 32 bits: these have no order
        for r in range(BATCH):
            assert np.allclose(np.exp(lp[r]), probs[r, ids[r]], rtol=1e-5, atol=1e-37)
            assert np.delete(probs[r], ids[r]).max(initial=0) <= probs[r, ids[r]].min()
    net.close()


@pytest.mark.parametrize("mode", [aetcnn.DISTILL_RENORM, aetcnn.DISTILL_TAIL])
@pytest.mark.parametrize("soft,hard,t", [(1.0, 0.0, 2.0), (0.5, 0.5, 1.0), (0.25, 0.75, 4.0)])
def test_distillation_step(gpu, mode, soft, hard, t):
    """One training step against another network's answers: the loss and the
    softmax layer's delta are the operator's, the output stays the softmax, and
    the weights' gradients are those that the delta gives in the layers below."""
    teacher, student, plain = network(5), network(9), network(9)
    x, _, _ = configs.synthetic_batch("tiny", 33, BATCH)
    labels = np.arange(BATCH) % 10
    labels[2] = -1
    tt = t if mode == aetcnn.DISTILL_TAIL else 1.0
    ids, lp, _ = teacher.predict_top(x, 4, tt)
    student.set_distillation(4, mode, t, soft, hard)
    student.set_teacher(ids, lp, labels if hard else None)
    student.set_input(x, None)
    student.forward(1)
    n = student.n_layers()
    z = logits(student)
    loss, lerr, delta, derr = ref.distill(z, ids, lp.astype(np.float64), labels, None, t,
                                          mode == aetcnn.DISTILL_TAIL, soft, hard, ref.F32)
    got = student.buffer(n - 1, 1).reshape(BATCH, -1)
    assert (np.abs(got - delta) <= derr).all()
    assert abs(student.loss() * BATCH - loss.sum()) <= lerr.sum() + 4 * ref.U * np.abs(loss).sum()
    assert (np.abs(student.buffer(n - 1, 15)[:BATCH] - loss) <= lerr).all()
    e = np.exp(z - z.max(1, keepdims=True))
    assert np.allclose(student.buffer(n - 1, 0).reshape(BATCH, -1), e / e.sum(1, keepdims=True),
                       rtol=1e-5)
    student.backward()
    plain.set_input(x, np.zeros((BATCH, 10), np.float32))
    plain.forward(1)
    plain.set_buffer(n - 1, 1, got)
    plain.backward()
    for i in range(n):
        a, b = student.buffer(i, 3), plain.buffer(i, 3)
        assert (a is None) == (b is None)
        if a is not None:
            assert np.array_equal(a, b), i
    for net in (teacher, student, plain):
        net.close()


def test_training_from_a_teacher_and_back(gpu):
    """Steps against changing teachers run and update; after
    an_end_distillation a step is that of a network that never had one."""
    teacher, student, plain = network(5), network(9), network(9)
    x, truth, _ = configs.synthetic_batch("tiny", 40, BATCH)
    student.set_distillation(3, aetcnn.DISTILL_TAIL, 1.0)
    student.set_distillation(4, aetcnn.DISTILL_TAIL, 2.0)  # anew: the first is forgotten
    student.end_distillation()
    assert student.train(x, truth) == plain.train(x, truth)
    w = student.buffer(0, 2)
    assert np.array_equal(w, plain.buffer(0, 2))
    student.set_distillation(4, aetcnn.DISTILL_TAIL, 2.0, 0.5, 0.5)
    for seed in (41, 42):
        xs, _, labels = configs.synthetic_batch("tiny", seed, BATCH)
        ids, lp, _ = teacher.predict_top(xs, 4, 2.0)
        student.set_teacher(ids, lp, np.asarray(labels).reshape(-1)[:BATCH])
        student.set_input(xs, None)
        student.train_step()
        assert np.isfinite(student.loss())
        assert not np.array_equal(student.buffer(0, 2), w)
        w = student.buffer(0, 2)
    # inference and answers do not depend on the teacher
    ids, _, _ = student.predict_top(x, 10)
    assert np.array_equal(np.sort(ids, 1), np.tile(np.arange(10), (BATCH, 1)))
    for net in (teacher, student, plain):
        net.close()


def test_refusals(gpu):
    lib = aetcnn.net_lib()
    net = network(1)
    x, truth, _ = configs.synthetic_batch("tiny", 2, BATCH)
    bad = [(0, 1, 1.0, 1.0, 0.0), (11, 1, 1.0, 1.0, 0.0), (4, 2, 1.0, 1.0, 0.0),
           (4, 1, 0.0, 1.0, 0.0), (4, 1, float("nan"), 1.0, 0.0), (4, 1, 1.0, float("inf"), 0.0)]
    for a in bad:
        assert lib.an_set_distillation(net.h, *a) == aetcnn.ACH_EINVAL
    assert np.isfinite(net.train(x, truth))      # none of these has taken hold
    net.set_distillation(4, aetcnn.DISTILL_TAIL, 1.0, 0.5, 0.5)
    with pytest.raises(aetcnn.HipError, match=f"code {aetcnn.ACH_EINVAL}"):
        net.train(x, truth)                      # no teacher yet
    ids, lp, _ = net.predict_top(x, 4)
    net.set_teacher(ids, lp)
    with pytest.raises(aetcnn.HipError, match=f"code {aetcnn.ACH_EINVAL}"):
        net.train(x, truth)                      # the label term has no labels
    with pytest.raises(ValueError):
        net.set_teacher(ids[:, :3], lp[:, :3])
    with pytest.raises(ValueError):
        net.predict_top(x[:1], 3)
    i, l = np.empty(BATCH * 11, np.int32), np.empty(BATCH * 11, np.float32)
    for k, t in ((0, 1.0), (11, 1.0), (3, 0.0), (3, -1.0), (3, float("nan"))):
        assert lib.an_predict_top(net.h, x.ctypes.data, k, t, i.ctypes.data, l.ctypes.data,
                                  None) == aetcnn.ACH_EINVAL
    net.close()
    # a network that does not end in a softmax over all its inputs
    aetcnn.net_lib().an_rand_seed(1)
    n2 = aetcnn.Network(4, 8, 8, 3)
    n2.conv(10, 3, 1, 1, aetcnn.LEAKY, 0)
    n2.avgpool()
    assert lib.an_set_distillation(n2.h, 4, 1, 1.0, 1.0, 0.0) == aetcnn.ACH_EINVAL  # not finalized
    n2.finalize()
    assert lib.an_set_distillation(n2.h, 4, 1, 1.0, 1.0, 0.0) == aetcnn.ACH_EINVAL
    assert lib.an_end_distillation(n2.h) == 0
    assert lib.an_set_teacher(n2.h, i.ctypes.data, l.ctypes.data, None) == aetcnn.ACH_EINVAL
    assert lib.an_predict_top(n2.h, l.ctypes.data, 3, 1.0, i.ctypes.data, l.ctypes.data,
                              None) == aetcnn.ACH_EINVAL
    n2.close()
