"""What the distillation and layer norm units leave behind, and what the
captured step goes by, on the numpy path (the GPU's lane:
test_distillation_answers_gpu.py)."""

import numpy
import pytest

from test_distillation import build, mlp, teacher_file
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
