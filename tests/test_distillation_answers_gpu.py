"""What the distillation units and the engine leave behind on the GPU: the
likeliest class beside the logits, a captured step after a change of the
temperature, graphs and copies of the served answers."""

import numpy
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

from test_distillation import build, mlp, save, teacher_file  # noqa: E402
from test_distillation_answers import student  # noqa: E402
from veles.backends import ROCmDevice  # noqa: E402


def steps(tmp_path, graph, n=14):
    """n training steps, the temperature changed after the eighth."""
    from bench import _NullCtx
    from veles.znicz_amd.hipgraph import GraphStepper
    from veles.znicz_amd.parallel import GradientReducer
    dev = ROCmDevice(0)
    wf = student(tmp_path, dev, n_train=120, n_valid=0)
    wf.grad_reducer = GradientReducer(_NullCtx(), dev)
    st = GraphStepper(wf, warmup=2 if graph else 100)
    for i in range(n):
        if i == 8:
            wf.evaluator.temperature = 4.0
            wf.forwards[1].eps = 0.01
        st.step()
        if i % 3 == 0:             # eager work between the replays
            torch.cuda.synchronize()
            torch.ones(100, device="cuda").sum().item()
    torch.cuda.synchronize()
    return wf, st


def test_a_captured_step_follows_the_temperature(tmp_path):
    ends = []
    for graph in (False, True):
        wf, st = steps(tmp_path, graph)
        if graph:
            assert st._graph is not None, getattr(st, "capture_error", "")
        ends.append([f.weights.devmem.clone() for f in wf.forwards] +
                    [wf.evaluator.loss.devmem.clone(),
                     wf.evaluator.n_err.devmem.clone(),
                     wf.forwards[-1].max_idx.devmem.clone()])
    for a, b in zip(*ends):
        assert torch.equal(a, b)


@pytest.mark.parametrize("graph", [False, True])
def test_likeliest_class_of_a_distilled_head(tmp_path, graph):
    wf, _ = steps(tmp_path, graph, 6)
    head = wf.forwards[-1]
    want = head.output.devmem.argmax(1)
    assert len(set(want.tolist())) > 1
    head.max_idx.map_read()
    assert head.max_idx.mem.tolist() == want.tolist()


def test_likeliest_class_of_rows_that_have_none(tmp_path):
    """It stays a class where there is no largest logit."""
    dev = ROCmDevice(0)
    wf = student(tmp_path, dev, n_valid=0)
    wf.loader.run()
    head = wf.forwards[-1]
    for f in wf.forwards[:-1]:
        f.run()
    head.input.devmem[3].fill_(float("nan"))
    head.input.touch_device()
    head.run()
    idx = head.max_idx.devmem.tolist()
    want = head.output.devmem.argmax(1).tolist()
    assert 0 <= idx[3] < 10
    assert idx[:3] + idx[4:] == want[:3] + want[4:]


def test_graphs_of_top_answers_are_few(tmp_path):
    from veles.serving import InferenceEngine
    eng = InferenceEngine(teacher_file(tmp_path), device=ROCmDevice(0))
    rng = numpy.random.RandomState(2)
    x = rng.normal(0, 1, (45, 24)).astype(numpy.float32)
    labels = rng.randint(-1, 10, 45)
    most = eng.predict_top(x, 128, labels)
    assert most["top"].shape == most["top_logprob"].shape == (45, 128)
    for top in list(range(1, 129, 3)) + [8, 9, 16, 128, 5]:
        ans = eng.predict_top(x, top, labels)
        assert ans["top"].shape == (45, top)
        numpy.testing.assert_array_equal(ans["top"], most["top"][:, :top])
        numpy.testing.assert_array_equal(ans["top_logprob"],
                                         most["top_logprob"][:, :top])
        for k in ("logprob", "entropy"):
            numpy.testing.assert_array_equal(ans[k], most[k])
    graphs = {id(v[0]) for v in eng._top_graphs.values()}
    assert len(graphs) <= 5
    assert all(v[0] is not None for v in eng._top_graphs.values())


@pytest.mark.parametrize("head", ["softmax", "all2all"])
def test_predict_copies_an_answer_once(tmp_path, head):
    """Out of the pinned buffer, which the next batch overwrites; a bf16
    head's numbers are copied by their conversion."""
    from torch.utils._python_dispatch import TorchDispatchMode
    from veles.serving import InferenceEngine

    class Copies(TorchDispatchMode):
        n = 0

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if func in (torch.ops.aten._to_copy.default,
                        torch.ops.aten.clone.default):
                Copies.n += 1
            return func(*args, **(kwargs or {}))

    path = teacher_file(tmp_path)
    wf = build(mlp(head=head), ROCmDevice(0), loss="distillation",
               distill={"snapshot": path, "top": 4})
    eng = InferenceEngine(save(wf, tmp_path, "copied"),
                          device=ROCmDevice(0))
    x = numpy.random.RandomState(2).normal(0, 1, (20, 24))
    eng.predict(x)
    Copies.n = 0
    with Copies():
        a = eng.predict(x)
    assert Copies.n == 1
    b = a.copy()
    eng.predict(x * 2)
    numpy.testing.assert_array_equal(a, b)
