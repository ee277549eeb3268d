"""Distillation: a student learns from a teacher's top answers.

No reference counterpart; built on the evaluator contract of reference
``znicz/evaluator.py`` (err_output for the last GD unit, ``n_err`` for the
Decision).  The teacher is a trained snapshot; each minibatch its forward
chain runs on the student's input and leaves its ``top`` likeliest classes
with their log probabilities (``ops.token_logprobs``), from which
:class:`EvaluatorDistillation` takes the student's loss and err_output in
one kernel (``ops.eval_distill``).  ``StandardWorkflow`` builds both for
``loss_function="distillation"``; the last layer is a softmax layer, whose
logits are taken, or one that gives logits itself.
"""

import numpy

from veles.accelerated_units import AcceleratedUnit
from veles.memory import Array
from veles.znicz_amd.evaluator import EvaluatorBase


# -- numpy reference ---------------------------------------------------------

def numpy_logprobs(logits, labels=None, top=0):
    """(logprob, entropy, top_idx, top_logprob) of rows of logits, in 64
    bits, as ``ops.token_logprobs`` defines them."""
    x = numpy.asarray(logits, numpy.float64)
    rows, cols = x.shape
    high = x.max(axis=1)
    bad = ~(high < numpy.inf) | numpy.isnan(x).any(axis=1)
    none = ~bad & (high == -numpy.inf)
    ref = numpy.where(bad | none, 0.0, high)[:, None]
    with numpy.errstate(over="ignore", invalid="ignore", divide="ignore"):
        t = x - ref
        e = numpy.exp(t)
        s = e.sum(axis=1)
        lp = t - numpy.log(s)[:, None]
        entropy = numpy.log(s) - (
            e * numpy.where(e > 0, t, 0.0)).sum(axis=1) / s
    lp[none] = -numpy.inf
    lp[bad] = numpy.nan
    entropy[none] = 0.0
    entropy[bad] = numpy.nan
    logprob = None
    if labels is not None:
        labels = numpy.asarray(labels)
        logprob = numpy.zeros(rows)
        for i, l in enumerate(labels):
            if l >= 0:
                logprob[i] = lp[i, l] if l < cols else numpy.nan
    idx = numpy.full((rows, top), -1, numpy.int32)
    top_lp = numpy.full((rows, top), -numpy.inf)
    top_lp[bad] = numpy.nan
    n = min(top, cols)
    for i in numpy.flatnonzero(~bad & ~none):
        order = numpy.argsort(-x[i], kind="stable")[:n]
        order = order[x[i, order] > -numpy.inf]
        idx[i, :len(order)] = order
        top_lp[i, :len(order)] = lp[i, order]
    return logprob, entropy, idx, top_lp


def numpy_distill(logits, top_idx, top_logit, temperature):
    """(loss, gradient) of rows of logits, in 64 bits, as
    ``ops.eval_distill`` defines them."""
    x = numpy.asarray(logits, numpy.float64)
    z = numpy.asarray(top_logit, numpy.float64)
    idx = numpy.asarray(top_idx)
    rows, cols = x.shape
    loss, grad = numpy.zeros(rows), numpy.zeros((rows, cols))
    tau = float(temperature)
    for i in range(rows):
        named = (idx[i] >= 0) & (z[i] != -numpy.inf)
        at, zi = idx[i][named], z[i][named]
        if not (x[i] < numpy.inf).all() or (idx[i] >= cols).any() or \
                not (zi < numpy.inf).all():
            loss[i], grad[i] = numpy.nan, numpy.nan
            continue
        high = x[i].max()
        if not len(at) or high == -numpy.inf:
            continue
        lnp = (x[i] - high) / tau
        lnp -= numpy.log(numpy.exp(lnp).sum())
        lnq = (zi - zi.max()) / tau
        lnq -= numpy.log(numpy.exp(lnq).sum())
        # (all places of a class together)
        at, place = numpy.unique(at, return_inverse=True)
        joined = numpy.full(len(at), -numpy.inf)
        numpy.logaddexp.at(joined, place, lnq)
        q = numpy.exp(joined)
        some = q > 0
        loss[i] = tau * tau * (q[some] * (joined[some] -
                                          lnp[at[some]])).sum()
        grad[i] = numpy.exp(lnp)
        grad[i, at] -= q
        grad[i] *= tau
    return loss, grad


# -- units -------------------------------------------------------------------

class TeacherAnswers(AcceleratedUnit):
    """The ``top`` likeliest classes of a trained snapshot's forward chain
    for each sample of ``input``, with their log probabilities.

    The chain's last layer gives the logits: a softmax layer those before
    its softmax, another one its output.  It is read from the file at
    ``initialize`` and is no part of this workflow's own snapshots."""

    def __init__(self, workflow, **kwargs):
        super(TeacherAnswers, self).__init__(workflow, **kwargs)
        self.snapshot = kwargs.get("snapshot")
        self.top = int(kwargs.get("top", 16))
        if not 1 <= self.top <= 128:
            raise ValueError("TeacherAnswers: top is %d, not 1 to 128" %
                             self.top)
        self.input = None            # linked: loader.minibatch_data
        self.batch_size = None       # linked: loader.minibatch_size
        self.classes = 0
        self.top_idx = Array()
        self.top_logprob = Array()
        self.forwards_ = None

    def __getstate__(self):
        state = super(TeacherAnswers, self).__getstate__()
        state["forwards_"] = None
        return state

    def _load(self):
        from veles.snapshotter import SnapshotterBase
        if not self.snapshot:
            raise ValueError("TeacherAnswers: no teacher's snapshot")
        wf = SnapshotterBase.import_(self.snapshot)
        forwards = list(getattr(wf, "forwards", None) or ())
        if not forwards:
            raise ValueError("snapshot has no forward chain (%r)" %
                             self.snapshot)
        first = forwards[0]
        want = tuple(first.input.shape[1:])
        if want != tuple(self.input.shape[1:]):
            raise ValueError("teacher takes samples of %s, not %s" %
                             (want, tuple(self.input.shape[1:])))
        first.unlink_attrs("input")
        first.input = self.input
        return forwards

    def initialize(self, device=None, **kwargs):
        if self.input is None or not self.input:
            return False
        super(TeacherAnswers, self).initialize(device=device, **kwargs)
        if self.forwards_ is None:
            self.forwards_ = self._load()
        for f in self.forwards_:
            f.forward_mode = True
            if hasattr(f, "logits_only"):
                f.logits_only = f is self.forwards_[-1]
            f.initialize(device=device)
        batch = self.input.shape[0]
        out = self.forwards_[-1].output
        self.classes = out.sample_size
        shape = (batch, min(self.top, self.classes))
        if not self.top_idx or self.top_idx.shape != shape:
            self.top_idx.reset(numpy.full(shape, -1, numpy.int32))
            self.top_logprob.reset(numpy.zeros(shape, numpy.float32))
        self.init_array(self.top_idx, device_dtype="i32")
        self.init_array(self.top_logprob, device_dtype="f32")

    def run(self):
        for f in self.forwards_:
            f.run()
        super(TeacherAnswers, self).run()

    def numpy_run(self):
        out = self.forwards_[-1].output
        out.map_read()
        self.top_idx.map_invalidate()
        self.top_logprob.map_invalidate()
        n = int(self.batch_size)
        self.top_idx.mem[n:] = -1
        self.top_logprob.mem[n:] = 0
        _, _, idx, lp = numpy_logprobs(
            out.mem[:n].reshape(n, -1), top=self.top_idx.shape[1])
        self.top_idx.mem[:n] = idx
        self.top_logprob.mem[:n] = lp

    def hip_run(self):
        from veles.znicz_amd import ops
        ops.token_logprobs(ops.as2d(self.forwards_[-1].output),
                           top_idx=self.top_idx.devmem,
                           top_logprob=self.top_logprob.devmem,
                           batch=int(self.batch_size))
        self.top_idx.touch_device()
        self.top_logprob.touch_device()


class EvaluatorDistillation(EvaluatorBase):
    """loss = t² KL(teacher ‖ student) at temperature t over the teacher's
    top classes; err_output = t (p − q).  With labels it counts ``n_err`` by
    the student's likeliest class, as EvaluatorSoftmax does."""

    def __init__(self, workflow, **kwargs):
        super(EvaluatorDistillation, self).__init__(workflow, **kwargs)
        self.temperature = float(kwargs.get("temperature", 1.0))
        if not 1e-3 <= self.temperature <= 1e3:
            raise ValueError("EvaluatorDistillation: temperature is %r, not "
                             "within 0.001 and 1000" % self.temperature)
        self.top_idx = None          # linked: teacher.top_idx
        self.top_logit = None        # linked: teacher.top_logprob
        self.labels = None           # linked: loader.minibatch_labels
        self.teacher = None
        self.loss = Array()          # of each sample of the minibatch
        self.n_err = Array()

    def initialize(self, device=None, **kwargs):
        if self.top_idx is None or not self.top_idx:
            return False
        r = super(EvaluatorDistillation, self).initialize(device=device,
                                                          **kwargs)
        if r is False:
            return False
        if self.teacher is not None and \
                self.teacher.classes != self.input.sample_size:
            raise ValueError("teacher has %d classes, the student %d" %
                             (self.teacher.classes, self.input.sample_size))
        batch = self.input.shape[0]
        if not self.loss or self.loss.shape != (batch,):
            self.loss.reset(numpy.zeros(batch, numpy.float32))
        if not self.n_err:
            self.n_err.reset(numpy.zeros(2, dtype=numpy.int32))
        self.init_array(self.loss, device_dtype="f32")
        self.init_array(self.n_err, device_dtype="i32")

    def numpy_run(self):
        for arr in (self.input, self.top_idx, self.top_logit, self.labels):
            if arr is not None:
                arr.map_read()
        self.err_output.map_invalidate()
        self.loss.map_invalidate()
        n = int(self.batch_size)
        x = self.input.mem[:n].reshape(n, -1)
        loss, grad = numpy_distill(x, self.top_idx.mem[:n],
                                   self.top_logit.mem[:n],
                                   self.temperature)
        self.loss.mem[...] = 0
        self.loss.mem[:n] = loss
        self.err_output.mem[...] = 0
        self.err_output.mem[:n] = grad.reshape(
            self.err_output.mem[:n].shape)
        if self.labels is not None:
            self.n_err.map_write()
            labels = self.labels.mem[:n]
            none = ~(x < numpy.inf).all(axis=1) | \
                (x == -numpy.inf).all(axis=1)
            wrong = none | (x.argmax(axis=1) != labels)
            self.n_err.mem[0] += int((wrong & (labels >= 0)).sum())

    def hip_run(self):
        from veles.znicz_amd import ops
        labels = None if self.labels is None else \
            ops.labels_on_device(self.labels, self.device)
        ops.eval_distill(
            ops.as2d(self.input), self.top_idx.devmem,
            self.top_logit.devmem, ops.as2d(self.err_output),
            self.loss.devmem, int(self.batch_size), self.temperature,
            labels, None if labels is None else self.n_err.devmem)
        self.err_output.touch_device()
        self.loss.touch_device()
        if labels is not None:
            self.n_err.touch_device()
