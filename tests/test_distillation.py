"""Layer norm, teacher and distillation units and the engine's top answers on
the numpy path (the GPU's lane: test_distillation_gpu.py)."""

import json
import os
import subprocess
import threading
import urllib.request

import numpy
import pytest

from veles import prng
from veles.backends import NumpyDevice
from veles.dummy import DummyLauncher, DummyWorkflow
from veles.memory import Array
from veles.znicz_amd.models.synthetic import SyntheticClassLoader
from veles.znicz_amd.normalization import (LayerNormBackward,
                                           LayerNormForward)
from veles.znicz_amd.standard_workflow import StandardWorkflow

GD = {"learning_rate": 0.05, "gradient_moment": 0.9}


def build(layers, device, batch=20, loss="softmax", distill=None,
          shape=(24,), classes=10, n_train=60, n_valid=20, dtype=None):
    return_wf = StandardWorkflow(
        DummyLauncher(), layers=layers,
        loader_factory=lambda w, **kw: SyntheticClassLoader(w, **kw),
        loader_config={"minibatch_size": batch, "n_train": n_train,
                       "n_valid": n_valid, "sample_shape": shape,
                       "n_classes": classes, "noise": 0.3},
        decision_config={"max_epochs": 2, "fail_iterations": 10 ** 9},
        snapshotter_config={"enabled": False}, loss_function=loss,
        distillation_config=distill or {})
    return_wf.initialize(device=device)
    return return_wf


def mlp(hidden=16, classes=10, head="softmax"):
    return [
        {"type": "all2all_tanh", "->": {"output_sample_shape": hidden},
         "<-": dict(GD)},
        {"type": "layer_norm", "->": {"eps": 1e-5}, "<-": dict(GD)},
        {"type": head, "->": {"output_sample_shape": classes},
         "<-": dict(GD)}]


def save(wf, path, name):
    from veles.snapshotter import SnapshotterToFile
    snap = SnapshotterToFile(wf, prefix=name, directory=str(path),
                             compression="")
    wf.del_ref(snap)
    return snap.export()


def teacher_file(path, device=None, **kw):
    prng.seed_all(5)
    wf = build(mlp(32), device or NumpyDevice(), **kw)
    wf.run()
    return save(wf, path, "teacher")


# -- layer norm unit ---------------------------------------------------------

@pytest.mark.parametrize("shape", [(6, 12), (2, 3, 4, 5)])
@pytest.mark.parametrize("bias", [True, False])
def test_layer_norm_unit_gradients_by_differences(shape, bias):
    rng = numpy.random.RandomState(3)
    wf = DummyWorkflow()
    fwd = LayerNormForward(wf, include_bias=bias, eps=1e-4)
    fwd.input = Array(rng.normal(0, 1.5, shape).astype(numpy.float64))
    assert fwd.initialize(device=NumpyDevice()) is not False
    C = shape[-1]
    fwd.weights.mem = rng.normal(1, 0.2, C)
    if bias:
        fwd.bias.mem = rng.normal(0, 0.2, C)
    for name in ("output", "mean", "rstd"):
        a = getattr(fwd, name)
        a.mem = a.mem.astype(numpy.float64)
    gd = LayerNormBackward(wf, apply_gradient=False)
    gd.input, gd.output = fwd.input, fwd.output
    gd.weights, gd.bias = fwd.weights, fwd.bias
    gd.include_bias = bias
    gd.mean, gd.rstd = fwd.mean, fwd.rstd
    gd.batch_size = shape[0]
    gd.err_output = Array(rng.normal(0, 1, shape).astype(numpy.float64))
    gd.err_input = Array(numpy.zeros(shape))
    assert gd.initialize(device=NumpyDevice()) is not False
    fwd.run()
    gd.run()

    def loss():
        fwd.run()
        return float((fwd.output.mem * gd.err_output.mem).sum())

    pairs = [(fwd.input, gd.err_input.mem, 1),
             (fwd.weights, gd.gradient_weights.mem, shape[0])]
    if bias:
        pairs.append((fwd.bias, gd.gradient_bias.mem, shape[0]))
    for arr, got, scale in pairs:
        flat, g = arr.mem.reshape(-1), got.reshape(-1) * scale
        for i in rng.choice(flat.size, min(8, flat.size), replace=False):
            old, h = flat[i], 1e-6
            flat[i] = old + h
            up = loss()
            flat[i] = old - h
            dn = loss()
            flat[i] = old
            # h^2, and 2^-52 |loss| / h
            assert abs(g[i] - (up - dn) / (2 * h)) < 1e-6


def test_layer_norm_unit_refusals():
    wf = DummyWorkflow()
    with pytest.raises(ValueError, match="eps"):
        LayerNormForward(wf, eps=-1.0)
    f = LayerNormForward(wf)
    f.input = Array(numpy.zeros(4, numpy.float32))
    with pytest.raises(ValueError, match="no features"):
        f.initialize(device=NumpyDevice())


# -- distillation workflow -----------------------------------------------------

@pytest.mark.parametrize("head", ["softmax", "all2all"])
def test_distillation_workflow_runs(tmp_path, head):
    path = teacher_file(tmp_path)
    prng.seed_all(7)
    wf = build(mlp(12, head=head), NumpyDevice(), loss="distillation",
               distill={"snapshot": path, "top": 4, "temperature": 2.0})
    before = [f.weights.mem.copy() for f in wf.forwards]
    wf.run()
    assert wf.teacher.top_idx.shape == (20, 4)
    assert wf.decision.epoch_n_err[2] <= 60
    for f, w in zip(wf.forwards, before):
        assert not numpy.array_equal(f.weights.mem, w)
    # what the evaluator has left of the last minibatch
    n = int(wf.loader.minibatch_size)
    from veles.znicz_amd.distillation import numpy_distill
    loss, grad = numpy_distill(wf.forwards[-1].output.mem[:n],
                               wf.teacher.top_idx.mem[:n],
                               wf.teacher.top_logprob.mem[:n], 2.0)
    numpy.testing.assert_allclose(wf.evaluator.loss.mem[:n], loss,
                                  rtol=1e-5, atol=1e-6)
    numpy.testing.assert_allclose(wf.evaluator.err_output.mem[:n], grad,
                                  rtol=1e-5, atol=1e-6)


def test_distilled_student_is_saved_resumed_and_served(tmp_path):
    path = teacher_file(tmp_path)
    prng.seed_all(8)
    wf = build(mlp(12), NumpyDevice(), loss="distillation",
               distill={"snapshot": path, "top": 4})
    wf.run()
    mine = save(wf, tmp_path, "student")
    from veles.serving import InferenceEngine
    eng = InferenceEngine(mine, device=NumpyDevice())
    x = numpy.random.RandomState(1).normal(0, 1, (7, 24))
    probs = eng.predict(x)
    # a softmax again, whatever the training took of it
    numpy.testing.assert_allclose(probs.sum(1), 1.0, rtol=1e-5)
    # the teacher is no part of the snapshot: it is read again
    from veles.snapshotter import SnapshotterBase
    again = SnapshotterBase.import_(mine)
    assert again.teacher.forwards_ is None
    again.workflow = DummyLauncher()
    again.initialize(device=NumpyDevice())
    assert again.teacher.forwards_
    again.loader.run()
    for f in again.forwards:
        f.run()
    again.teacher.run()
    again.evaluator.run()


def test_distillation_refusals(tmp_path):
    path = teacher_file(tmp_path)
    with pytest.raises(ValueError, match="no teacher"):
        build(mlp(), NumpyDevice(), loss="distillation")
    with pytest.raises(ValueError, match="teacher has 10 classes"):
        build(mlp(classes=9), NumpyDevice(), loss="distillation",
              distill={"snapshot": path})
    with pytest.raises(ValueError, match="samples of"):
        build(mlp(), NumpyDevice(), loss="distillation", shape=(25,),
              distill={"snapshot": path})
    with pytest.raises(ValueError, match="top is"):
        build(mlp(), NumpyDevice(), loss="distillation",
              distill={"snapshot": path, "top": 129})
    with pytest.raises(ValueError, match="temperature"):
        build(mlp(), NumpyDevice(), loss="distillation",
              distill={"snapshot": path, "temperature": 0.0})
    with pytest.raises(ValueError, match="loss_function"):
        build(mlp(), NumpyDevice(), loss="hinge")


# -- top answers of the engine ---------------------------------------------------

def test_predict_top_matches_predict(tmp_path):
    from veles.serving import InferenceEngine
    eng = InferenceEngine(teacher_file(tmp_path), device=NumpyDevice())
    x = numpy.random.RandomState(2).normal(0, 1, (45, 24))
    probs = eng.predict(x).astype(float)
    labels = numpy.arange(45) % 11 - 1
    ans = eng.predict_top(x, 3, labels)
    order = numpy.argsort(-probs, axis=1, kind="stable")[:, :3]
    assert (ans["top"] == order).all()
    # probabilities and log probabilities are in fp32
    numpy.testing.assert_allclose(
        ans["top_logprob"],
        numpy.log(numpy.take_along_axis(probs, order, 1)), rtol=1e-4,
        atol=1e-5)
    numpy.testing.assert_allclose(
        ans["entropy"], -(probs * numpy.log(probs)).sum(1), rtol=1e-4)
    want = numpy.where(labels < 0, 0, numpy.log(
        probs[numpy.arange(45), numpy.maximum(labels, 0)]))
    numpy.testing.assert_allclose(ans["logprob"], want, rtol=1e-4,
                                  atol=1e-5)
    # more alternatives than classes; then predict() is as it was
    more = eng.predict_top(x[:2], 12)
    assert "logprob" not in more
    assert (more["top"][:, 10:] == -1).all()
    assert (more["top_logprob"][:, 10:] == -numpy.inf).all()
    numpy.testing.assert_array_equal(eng.predict(x), probs)
    for bad in (0, 129):
        with pytest.raises(ValueError, match="top is"):
            eng.predict_top(x, bad)
    with pytest.raises(ValueError, match="labels for"):
        eng.predict_top(x, 3, [1, 2])
    with pytest.raises(ValueError, match="sample shape"):
        eng.predict_top(x[:, :5], 3)
    with pytest.raises(ValueError, match="no samples"):
        eng.predict_top(x[:0], 3)


def test_predict_top_labels_of_any_type(tmp_path):
    """Whole numbers beyond 32 bits do not come round to a class; others are
    refused."""
    from veles.serving import InferenceEngine
    eng = InferenceEngine(teacher_file(tmp_path), device=NumpyDevice())
    x = numpy.random.RandomState(2).normal(0, 1, (3, 24))
    want = eng.predict_top(x, 2, [3, 0, 9])["logprob"]
    for dtype in (numpy.int8, numpy.uint8, numpy.int64, numpy.uint64):
        got = eng.predict_top(x, 2, numpy.array([3, 0, 9], dtype))
        numpy.testing.assert_array_equal(got["logprob"], want)
    got = eng.predict_top(x, 2, numpy.array([1 << 32, -(1 << 32), 10]))
    assert numpy.isnan(got["logprob"][[0, 2]]).all()
    assert got["logprob"][1] == 0
    got = eng.predict_top(x, 2, numpy.array([1 << 63, 3, 0], numpy.uint64))
    assert numpy.isnan(got["logprob"][0])
    for bad in ([1.5, 0, 0], [True, False, True], ["1", "2", "3"]):
        with pytest.raises(ValueError, match="whole numbers"):
            eng.predict_top(x, 2, bad)
    for bad in (2.5, "3", None):
        with pytest.raises(ValueError, match="top is"):
            eng.predict_top(x, bad)


def test_top_answers_over_http(tmp_path):
    import socket
    from veles import serving
    eng = serving.InferenceEngine(teacher_file(tmp_path),
                                  device=NumpyDevice())
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    threading.Thread(target=serving.serve, args=(eng, port),
                     daemon=True).start()
    x = numpy.random.RandomState(2).normal(0, 1, (2, 24))
    body = json.dumps({"inputs": x.tolist(), "top": 11,
                       "labels": [3, -1]}).encode()
    for _ in range(50):
        try:
            r = urllib.request.urlopen(
                "http://127.0.0.1:%d/" % port, body, timeout=10)
            break
        except urllib.error.URLError:
            import time
            time.sleep(0.1)
    got = json.loads(r.read())
    want = eng.predict_top(x, 11, [3, -1])
    assert got["top"] == want["top"].tolist()
    assert got["top_logprob"][0][10] is None       # no eleventh class
    numpy.testing.assert_allclose(got["logprob"], want["logprob"],
                                  rtol=1e-6)


def test_export_flat_layer_norm(tmp_path):
    from veles.serving import InferenceEngine, export_flat
    eng = InferenceEngine(teacher_file(tmp_path), device=NumpyDevice())
    out = str(tmp_path / "flat")
    export_flat(eng, out)
    lines = open(os.path.join(out, "manifest.txt")).read().splitlines()
    ops = [l.split() for l in lines if l.startswith("op ")]
    assert [o[1] for o in ops] == ["fc", "layernorm", "fc", "softmax"]
    assert ops[1][2:] == ["w1", "b1", "32", "20", "1e-05", "640"]
    binary = os.path.join(os.path.dirname(os.path.dirname(
        os.path.abspath(__file__))), "veles", "znicz_amd", "serve",
        "mzserve")
    if not os.path.exists(binary):
        return

    def parse(text, *args):
        with open(os.path.join(out, "manifest.txt"), "w") as f:
            f.write(text)
        return subprocess.run([binary, out] + list(args),
                              capture_output=True, text=True, timeout=60)
    text = "\n".join(lines) + "\n"
    r = parse(text, "--parse-only")
    assert r.returncode == 0 and json.loads(r.stdout)["ops"] == 4
    r = parse(text.replace("layernorm w1 b1 32 20 1e-05 640",
                           "layernorm w1 b1 32 20 1e-05 639"),
              "--parse-only")
    assert r.returncode == 1 and "bad layernorm" in r.stderr
    # a gain of another length ends it before the GPU is asked for anything
    r = parse(text.replace("op layernorm w1", "op layernorm w0"))
    assert r.returncode == 1 and "bad tensor w0" in r.stderr
