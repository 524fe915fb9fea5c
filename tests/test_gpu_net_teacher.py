"""Training from a teacher: a step that is refused leaves the network as it was,
and a feeder's new images need answers of their own."""
import numpy as np
import pytest

import aetcnn
from aetcnn import configs

pytestmark = pytest.mark.gpu
BATCH = 8
TRAINED = (2, 3, 4, 5, 6, 7, 8, 9)  # parameters, momenta, rolling statistics
REFUSED = f"code {aetcnn.ACH_EINVAL}"


def network(seed, name="tiny", batch=BATCH, subdivisions=1):
    aetcnn.net_lib().an_rand_seed(seed)
    net = aetcnn.Network(*configs.dims(name, batch))
    configs.build(net, name)
    net.subdivisions(subdivisions)
    net.finalize()
    return net


def state(net, codes=(0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11)):
    """counters, and outputs, deltas, parameters, momenta and statistics"""
    out = [np.array([net.seen(), net.iteration()])]
    for i in range(net.n_layers()):
        out += [net.buffer(i, code) for code in codes]
    return [a for a in out if a is not None]


def equal(a, b):
    assert len(a) == len(b)
    return all(np.array_equal(x, y, equal_nan=True) for x, y in zip(a, b))


@pytest.mark.parametrize("name,subdivisions", [("tiny", 1), ("fcnet", 2), ("fcnet", 3)])
def test_refused_steps_change_nothing(gpu, name, subdivisions):
    """without a teacher, or without the labels that the factor `hard` asks for,
    before the first step and between steps: what follows is what a network
    does that never made the call, dropout, rolling statistics and the
    minibatch of the update included"""
    net, twin = (network(7, name, subdivisions=subdivisions) for _ in range(2))
    other = network(8, name)
    calls = (net.train_step, lambda: net.forward(1),
             lambda: net.layer_forward(net.n_layers() - 1, 1),
             lambda: net.train(np.zeros_like(x), np.zeros((BATCH, 10))))
    for seed in range(4):
        x, _, labels = configs.synthetic_batch(name, seed, BATCH)
        labels = np.asarray(labels).reshape(-1)[:BATCH]
        ids, lp, _ = other.predict_top(x, 4, 2.0)
        for n in (net, twin):
            if seed != 1:  # the second step goes on with the teacher that is set
                n.set_distillation(4, aetcnn.DISTILL_TAIL, 2.0, 0.5, 0.5)
            n.set_input(x, None)
        before = state(net)
        if seed != 1:
            for call in calls:
                with pytest.raises(aetcnn.HipError, match=REFUSED):
                    call()
                assert equal(state(net), before)
            net.set_teacher(ids, lp)  # no labels
            for call in calls:
                with pytest.raises(aetcnn.HipError, match=REFUSED):
                    call()
                assert equal(state(net), before)
        for n in (net, twin):
            n.set_teacher(ids, lp, labels)
            n.train_step()
        assert net.loss() == twin.loss()
        assert equal(state(net, TRAINED), state(twin, TRAINED)), seed
    for n in (net, twin, other):
        n.close()


def test_inference_needs_no_teacher(gpu):
    net = network(3)
    x, _, _ = configs.synthetic_batch("tiny", 5, BATCH)
    before = net.predict(x)
    net.set_distillation(4, aetcnn.DISTILL_TAIL, 1.0)
    assert np.array_equal(net.predict(x), before)
    net.forward(0)
    net.end_distillation()
    net.close()


def fed(net):
    """the images that the feeder has made the network's input"""
    shape = (net.batch,) + tuple(net.shape(0)[4:7])
    return aetcnn.DeviceArray.wrap(net.lib.an_input(net.h), shape).numpy(net.stream)


def test_teacher_of_fed_images(gpu):
    """A feeder's images, read back, are what the teacher answers for.  The next
    batch needs answers of its own: a step with those that a step has used is
    refused, and answers set before the batch is fetched, or after, are taken."""
    net, twin, teacher = network(4), network(4), network(5)
    feeder = aetcnn.Feeder(net, threads=2, seed=11)
    for n in (net, twin):
        n.set_distillation(4, aetcnn.DISTILL_TAIL, 2.0)
    for step in range(4):
        feeder.next()
        x = fed(net)
        if step:
            before = state(net)
            with pytest.raises(aetcnn.HipError, match=REFUSED):
                net.train_step()
            assert equal(state(net), before)
        ids, lp, _ = teacher.predict_top(x, 4, 2.0)
        twin.set_input(x, None)
        for n in (net, twin):
            n.set_teacher(ids, lp)
            n.train_step()
        assert net.loss() == twin.loss()
        for i in range(net.n_layers()):
            a, b = net.buffer(i, 2), twin.buffer(i, 2)
            assert a is b is None or np.array_equal(a, b)
    net.set_teacher(ids, lp)   # known beforehand
    feeder.next()
    net.train_step()
    net.set_input(x, None)     # the caller's own batches: as the caller says
    net.set_teacher(ids, lp)
    net.train_step()
    net.train_step()
    net.end_distillation()     # the truth again
    feeder.next()
    net.train_step()
    assert np.isfinite(net.loss())
    feeder.close()
    for n in (net, twin, teacher):
        n.close()
