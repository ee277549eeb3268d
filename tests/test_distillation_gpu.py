"""Layer norm, teacher and distillation units on the GPU: against the numpy
references on what the units hold, in captured steps, and served."""

import json
import os
import subprocess

import numpy
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

from test_distillation import build, mlp, save, teacher_file  # noqa: E402
from veles import prng  # noqa: E402
from veles.backends import ROCmDevice  # noqa: E402
from veles.dummy import DummyWorkflow  # noqa: E402
from veles.memory import Array  # noqa: E402
from veles.znicz_amd.distillation import (  # noqa: E402
    numpy_distill, numpy_logprobs)
from veles.znicz_amd.normalization import (  # noqa: E402
    LayerNormBackward, LayerNormForward)

E32 = 2.0 ** -24
BF16 = 2.0 ** -8           # half a step


def f64(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("shape", [(64, 100), (8, 5, 5, 96), (4, 4096)])
@pytest.mark.parametrize("bias,need", [(True, True), (False, True),
                                       (True, False)])
def test_layer_norm_units(shape, bias, need):
    rng = numpy.random.RandomState(1)
    dev, wf, C = ROCmDevice(0), DummyWorkflow(), shape[-1]
    fwd = LayerNormForward(wf, include_bias=bias)
    fwd.input = Array(rng.normal(0.2, 1.5, shape).astype(numpy.float32),
                      device_dtype="bf16")
    fwd.input.initialize(dev)
    fwd.weights.mem = rng.normal(1, 0.2, C).astype(numpy.float32)
    fwd.bias.mem = rng.normal(0, 0.2, C).astype(numpy.float32)
    assert fwd.initialize(device=dev) is not False
    gd = LayerNormBackward(wf, learning_rate=0.5, weights_decay=0.0)
    gd.input, gd.output = fwd.input, fwd.output
    gd.weights, gd.bias, gd.include_bias = fwd.weights, fwd.bias, bias
    gd.mean, gd.rstd, gd.need_err_input = fwd.mean, fwd.rstd, need
    gd.batch_size = shape[0]
    gd.err_output = Array(rng.normal(0, 1, shape).astype(numpy.float32),
                          device_dtype="bf16")
    gd.err_output.initialize(dev)
    assert gd.initialize(device=dev) is not False
    fwd.run()
    gd.run()
    x = f64(fwd.input.devmem).reshape(-1, C)
    dy = f64(gd.err_output.devmem).reshape(-1, C)
    mu = x.mean(1, keepdims=True)
    r = 1 / numpy.sqrt(((x - mu) ** 2).mean(1, keepdims=True) + 1e-5)
    h = (x - mu) * r
    # the gain before the update: 1.0 steps of it are undone
    gw, gb = (dy * h).sum(0), dy.sum(0)
    n = x.shape[0]
    got_gw = f64(gd.gradient_weights.devmem)
    tol = (n / 128 + 1100) * E32 * numpy.abs(dy * h).sum(0) + \
        numpy.abs(dy).sum(0) * 64 * E32 * (1 + numpy.abs(mu).max() * r.max())
    assert (numpy.abs(got_gw - gw) <= tol).all()
    fwd.weights.map_read()
    start = rng.__class__(1)
    start.normal(0.2, 1.5, shape)
    gain = start.normal(1, 0.2, C).astype(numpy.float32)
    want = gain - 0.5 * got_gw / shape[0]
    # scaled, multiplied and subtracted: three roundings
    assert (numpy.abs(fwd.weights.mem - want) <=
            4 * E32 * (numpy.abs(gain) +
                       numpy.abs(got_gw) / shape[0])).all()
    shift = start.normal(0, 0.2, C).astype(numpy.float32) if bias else 0.0
    y = h * gain + shift
    err = numpy.abs(f64(fwd.output.devmem).reshape(-1, C) - y)
    assert (err <= BF16 * numpy.abs(y) +
            (C / 256 + 64) * E32 * (numpy.abs(h * gain) + 2)).all()
    if bias:
        assert (numpy.abs(f64(gd.gradient_bias.devmem) - gb) <=
                (n / 128 + 1100) * E32 * numpy.abs(dy).sum(0)).all()
    if need:
        g = dy * gain
        dx = r * (g - g.mean(1, keepdims=True) -
                  h * (g * h).mean(1, keepdims=True))
        err = numpy.abs(f64(gd.err_input.devmem).reshape(-1, C) - dx)
        assert (err <= BF16 * numpy.abs(dx) + (C / 256 + 64) * 4 * E32 * r *
                (numpy.abs(g) + 1 + numpy.abs(h))).all()
    # a served forward pass writes no statistics and the same output
    fwd.forward_mode = True
    fwd.mean.devmem.fill_(7.0)
    fwd.weights.devmem.copy_(torch.from_numpy(gain))
    if bias:
        fwd.bias.devmem.copy_(torch.from_numpy(shift))
    before = fwd.output.devmem.clone()
    fwd.run()
    assert torch.equal(fwd.output.devmem, before)
    assert (fwd.mean.devmem == 7).all()


def student(tmp_path, device, head="softmax", batch=20, **kw):
    path = teacher_file(tmp_path)
    prng.seed_all(7)
    return build(mlp(16, head=head), device, loss="distillation",
                 batch=batch, distill={"snapshot": path, "top": 4,
                                       "temperature": 2.0}, **kw)


@pytest.mark.parametrize("head", ["softmax", "all2all"])
def test_distillation_chain(tmp_path, head):
    """One minibatch (not full) through all units, each against the numpy
    reference on what the one before it has left."""
    wf = student(tmp_path, ROCmDevice(0), head, n_train=33, n_valid=0)
    ld = wf.loader
    for _ in range(2):             # the second of them has 13 samples
        ld.run()
        for f in wf.forwards:
            f.run()
        wf.teacher.run()
        wf.evaluator.run()
        wf.decision.run()
        for g in reversed(wf.gds):
            g.run()
    n = int(ld.minibatch_size)
    assert n == 13
    t = wf.teacher
    logits = f64(t.forwards_[-1].output.devmem)
    lp, ent, idx, top = numpy_logprobs(logits[:n], top=4)
    assert (t.top_idx.devmem.cpu().numpy()[:n] == idx).all()
    assert (t.top_idx.devmem.cpu().numpy()[n:] == -1).all()
    numpy.testing.assert_allclose(f64(t.top_logprob.devmem)[:n], top,
                                  atol=64 * E32 * 8)
    x = f64(wf.forwards[-1].output.devmem)
    err = f64(wf.evaluator.err_output.devmem)
    loss, grad = numpy_distill(x[:n], idx, f64(t.top_logprob.devmem)[:n],
                               2.0)
    assert (numpy.abs(err[:n] - grad) <=
            BF16 * numpy.abs(grad) + 256 * E32).all()
    assert (err[n:] == 0).all()
    numpy.testing.assert_allclose(f64(wf.evaluator.loss.devmem)[:n], loss,
                                  rtol=1e-5, atol=1024 * E32)
    for g in wf.gds:
        assert torch.isfinite(g.gradient_weights.devmem).all()
        assert (g.gradient_weights.devmem != 0).any()


def test_distillation_workflow_runs_on_gpu(tmp_path):
    wf = student(tmp_path, ROCmDevice(0))
    wf.run()
    assert wf.decision.epoch_n_err[2] <= 60
    for f in wf.forwards:
        f.weights.map_read()
        assert numpy.isfinite(f.weights.mem).all()


def test_distillation_step_in_a_graph(tmp_path):
    """A captured training step, replayed with new minibatches, follows the
    eager one to the bit."""
    from bench import _NullCtx
    from veles.znicz_amd.hipgraph import GraphStepper
    from veles.znicz_amd.parallel import GradientReducer
    ends = []
    for graph in (False, True):
        dev = ROCmDevice(0)
        wf = student(tmp_path, dev, n_train=120, n_valid=0)
        wf.grad_reducer = GradientReducer(_NullCtx(), dev)
        # (the eager side: as many steps before it would capture)
        st = GraphStepper(wf, warmup=2 if graph else 100)
        for i in range(11):
            st.step()
            if i % 3 == 0:         # eager work between the replays
                torch.cuda.synchronize()
                torch.ones(100, device="cuda").sum().item()
        torch.cuda.synchronize()
        if graph:
            assert st._graph is not None, getattr(st, "capture_error", "")
        ends.append([f.weights.devmem.clone() for f in wf.forwards] +
                    [wf.evaluator.loss.devmem.clone(),
                     wf.teacher.top_idx.devmem.clone(),
                     wf.evaluator.n_err.devmem.clone()])
    for a, b in zip(*ends):
        assert torch.equal(a, b)


def test_predict_top_on_gpu(tmp_path):
    from veles.serving import InferenceEngine
    path = teacher_file(tmp_path)
    eng = InferenceEngine(path, device=ROCmDevice(0))
    rng = numpy.random.RandomState(2)
    for turn in range(3):
        x = rng.normal(0, 1, (45, 24)).astype(numpy.float32)
        labels = rng.randint(-1, 10, 45)
        ans = eng.predict_top(x, 3, labels)
        probs = eng.predict(x).astype(float)   # (another graph, in turn)
        again = eng.predict_top(x, 3)
        assert "logprob" not in again
        for k in again:
            numpy.testing.assert_array_equal(ans[k], again[k])
        for i in range(45):
            # an order of probabilities in fp32, which may be equal there
            p = probs[i][ans["top"][i]]
            assert (numpy.diff(p) <= 0).all()
            assert p[0] == probs[i].max()
        got = numpy.exp(ans["top_logprob"].astype(float))
        want = numpy.take_along_axis(probs, ans["top"], 1)
        numpy.testing.assert_allclose(got, want, rtol=64 * E32 * 16,
                                      atol=1e-30)
        numpy.testing.assert_allclose(
            ans["entropy"], -(probs * numpy.log(probs)).sum(1), rtol=1e-4,
            atol=1e-5)
        assert (ans["logprob"][labels < 0] == 0).all()
    assert eng._top_graphs[3][0] is not None, "capture failed"
    more = eng.predict_top(x[:2], 12)
    assert (more["top"][:, 10:] == -1).all()


def test_mzserve_layer_norm(tmp_path):
    binary = os.path.join(os.path.dirname(os.path.dirname(
        os.path.abspath(__file__))), "veles", "znicz_amd", "serve",
        "mzserve")
    if not os.path.exists(binary):
        pytest.skip("mzserve binary not built")
    from veles.serving import InferenceEngine, export_flat
    prng.seed_all(5)
    layers = [
        {"type": "conv_str", "->": {"n_kernels": 16, "kx": 3, "ky": 3,
                                    "padding": (1, 1, 1, 1)}, "<-": {}},
        {"type": "layer_norm", "<-": {}},
        {"type": "all2all_tanh", "->": {"output_sample_shape": 40},
         "<-": {}},
        {"type": "layer_norm", "->": {"include_bias": False}, "<-": {}},
        {"type": "softmax", "->": {"output_sample_shape": 10}, "<-": {}}]
    wf = build(layers, ROCmDevice(0), shape=(8, 8, 8), n_valid=0)
    wf.run()
    path = save(wf, tmp_path, "served")
    eng = InferenceEngine(path, device=ROCmDevice(0))
    out = str(tmp_path / "flat")
    export_flat(eng, out)
    x = numpy.random.RandomState(3).normal(0, 1, (20, 8, 8, 8)).astype("<f4")
    x.tofile(str(tmp_path / "in.bin"))
    r = subprocess.run(
        [binary, out, "--input", str(tmp_path / "in.bin"), "--out",
         str(tmp_path / "out.bin"), "--batches", "3", "--warmup", "2"],
        capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.stdout, r.stderr)
    stats = json.loads(r.stdout.strip().splitlines()[-1])
    assert stats["ops"] == 6 and stats["graph"] is True
    got = numpy.fromfile(str(tmp_path / "out.bin"), "<f4").reshape(20, 10)
    # the same kernels on the same weights
    numpy.testing.assert_allclose(got, eng.predict(x).reshape(20, 10),
                                  rtol=1e-5, atol=1e-6)
