"""What the distillation and layer norm units leave behind, and what the
captured step goes by, on the numpy path (the GPU's lane:
test_distillation_answers_gpu.py)."""

import numpy
import pytest

from test_distillation import build, mlp, save, teacher_file
from veles import prng
from veles.backends import NumpyDevice
from veles.dummy import DummyWorkflow
from veles.memory import Array
from veles.znicz_amd.distillation import numpy_distill
from veles.znicz_amd.normalization import LayerNormForward


def student(tmp_path, device, **kw):
    for key in ("default", "loader"):
        prng.get(key)              # (streams that are there get the seed)
    path = teacher_file(tmp_path)
    prng.seed_all(7)
    return build(mlp(16), device, loss="distillation",
                 distill={"snapshot": path, "top": 4, "temperature": 2.0},
                 **kw)


def test_likeliest_class_of_a_distilled_head(tmp_path):
    """Who links max_idx has the class of the largest logit."""
    wf = student(tmp_path, NumpyDevice())
    head = wf.forwards[-1]
    for _ in range(2):
        wf.loader.run()
        for f in wf.forwards:
            f.run()
        numpy.testing.assert_array_equal(head.max_idx.mem,
                                         head.output.mem.argmax(axis=1))
        assert len(set(head.max_idx.mem.tolist())) > 1


def stepper(wf):
    from veles.znicz_amd.hipgraph import GraphStepper
    wf.comm_sync = None            # (what run() would have; not used here)
    return GraphStepper(wf, enabled=False)


@pytest.mark.parametrize("change", ["temperature", "eps"])
def test_signature_of_a_captured_step(tmp_path, change):
    """What the evaluator and the forwards pass to kernels by value."""
    wf = student(tmp_path, NumpyDevice())
    st = stepper(wf)
    before = st._signature()
    assert st._signature() == before
    if change == "temperature":
        wf.evaluator.temperature = 3.0
    else:
        wf.forwards[1].eps = 1e-3
    assert st._signature() != before


def test_statistics_are_not_written_in_forward_mode():
    rng = numpy.random.RandomState(3)
    fwd = LayerNormForward(DummyWorkflow())
    fwd.input = Array(rng.normal(0, 1.5, (6, 12)).astype(numpy.float32))
    assert fwd.initialize(device=NumpyDevice()) is not False
    fwd.run()
    y, mean = fwd.output.mem.copy(), fwd.mean.mem.copy()
    assert mean.any() and fwd.rstd.mem.all()
    fwd.forward_mode = True
    fwd.mean.mem[...] = 7
    fwd.rstd.mem[...] = 8
    fwd.run()
    assert (fwd.mean.mem == 7).all() and (fwd.rstd.mem == 8).all()
    numpy.testing.assert_array_equal(fwd.output.mem, y)


@pytest.mark.parametrize("tau", [1.0, 2.5])
def test_loss_of_a_class_that_is_named_twice(tau):
    """It has both shares, in the loss as in the gradient: as if it were
    named once, with the logit that has their sum."""
    rng = numpy.random.RandomState(1)
    x = rng.normal(0, 2, (3, 30))
    idx = numpy.array([[4, 7, 4, 9], [5, 5, 5, 5], [1, 2, 2, 1]])
    z = rng.normal(0, 2, (3, 4))
    loss, grad = numpy_distill(x, idx, z, tau)
    for i in range(3):
        at = sorted(set(idx[i].tolist()))
        one = [tau * numpy.logaddexp.reduce(z[i][idx[i] == a] / tau)
               for a in at]
        want_l, want_g = numpy_distill(x[i:i + 1], [at], [one], tau)
        # a few roundings of 64 bits, of numbers below 20
        assert abs(loss[i] - want_l[0]) < 1e-12
        numpy.testing.assert_allclose(grad[i], want_g[0], atol=1e-13)
    # (one sure class, of which the student is as sure)
    x = numpy.full((1, 4), -50.0)
    x[0, 2] = 0.0
    assert abs(numpy_distill(x, [[2, 2]], [[0.0, 0.0]], tau)[0][0]) < 1e-6


def test_a_softmax_within_the_teacher_stays_one(tmp_path):
    """Its last layer alone gives logits."""
    for key in ("default", "loader"):
        prng.get(key)
    prng.seed_all(5)
    wf = build([{"type": "softmax", "->": {"output_sample_shape": 12},
                 "<-": {}},
                {"type": "softmax", "->": {"output_sample_shape": 10},
                 "<-": {}}], NumpyDevice())
    wf.run()
    path = save(wf, tmp_path, "within")
    wf = build(mlp(), NumpyDevice(), loss="distillation",
               distill={"snapshot": path, "top": 4})
    wf.loader.run()
    wf.teacher.run()
    first, last = wf.teacher.forwards_
    numpy.testing.assert_allclose(first.output.mem.sum(axis=1), 1.0,
                                  rtol=1e-5)
    assert not numpy.allclose(last.output.mem.sum(axis=1), 1.0)
    # as the same model served: log probabilities in fp32 on both sides
    from veles.serving import InferenceEngine
    n = int(wf.loader.minibatch_size)
    ans = InferenceEngine(path, device=NumpyDevice()).predict_top(
        wf.loader.minibatch_data.mem[:n], 4)
    numpy.testing.assert_array_equal(wf.teacher.top_idx.mem[:n], ans["top"])
    numpy.testing.assert_array_equal(wf.teacher.top_logprob.mem[:n],
                                     ans["top_logprob"])
