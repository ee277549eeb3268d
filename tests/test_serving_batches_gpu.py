"""The engine on more samples than one batch holds."""

import numpy
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

from veles import prng  # noqa: E402
from veles.backends import NumpyDevice, ROCmDevice  # noqa: E402
from veles.config import root  # noqa: E402
from veles.dummy import DummyLauncher  # noqa: E402


def test_predict_of_several_batches(tmp_path):
    """What predict() gave for one batch stays when the next one runs."""
    prng.seed_all(99)
    from veles.serving import InferenceEngine
    from veles.snapshotter import SnapshotterToFile
    from veles.znicz_amd.models.wine import WineWorkflow
    root.wine.decision.update({"max_epochs": 3, "fail_iterations": 50})
    root.wine.loader.update({"n_train": 90, "n_valid": 30,
                             "minibatch_size": 30})
    wf = WineWorkflow(DummyLauncher())
    wf.initialize(device=NumpyDevice())
    wf.run()
    snap = SnapshotterToFile(wf, prefix="srv", directory=str(tmp_path),
                             compression="")
    wf.del_ref(snap)
    eng = InferenceEngine(snap.export(), device=ROCmDevice(0))
    x = numpy.random.RandomState(2).normal(
        0, 1, (75,) + tuple(eng._in.shape[1:]))
    first = eng.predict(x[:30])
    kept = first.copy()
    parts = [first] + [eng.predict(x[i:i + 30]) for i in (30, 60)]
    numpy.testing.assert_array_equal(first, kept)
    numpy.testing.assert_array_equal(eng.predict(x),
                                     numpy.concatenate(parts))
