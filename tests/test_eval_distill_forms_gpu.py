"""eval_distill on the GPU in the form in which the evaluator calls it (fp32
logits, a bf16 gradient, labels and n_err), its count of errors beside what
is wrong with the teacher, and classes that are named more than once."""

import math

import numpy
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

from test_row_ops_gpu import (  # noqa: E402
    E32, INF, TYPES, check_distill, cuda, f64, logits_case, rows_of,
    teacher_case)
from veles.znicz_amd import ops  # noqa: E402


def counted(tx, idx, z, err, labels, batch=None, tau=1.0):
    """(loss, n_err) of a call that counts from 10 on"""
    loss = torch.full((tx.shape[0],), 55.0, device="cuda")
    n = torch.tensor([10, 3], dtype=torch.int32).cuda()
    ops.eval_distill(tx, cuda(idx), cuda(z), err, loss, batch, tau,
                     torch.as_tensor(labels, dtype=torch.int32).cuda(), n)
    assert n[1].item() == 3
    return loss, n[0].item() - 10


# (up to 16384 classes of fp32 a row of 256 threads, to 32768 one of 512, to
# 65536 one of 1024, longer ones read twice; 64 rows or fewer may be cut)
@pytest.mark.parametrize("R", [9, 65, 97])
@pytest.mark.parametrize("C", [10, 1000, 5003, 16384, 20001, 50001, 140007])
@pytest.mark.parametrize("xpad,epad", [(0, 0), (1, 3)])
def test_form_of_the_evaluator(R, C, xpad, epad):
    rng = numpy.random.RandomState(C)
    x = logits_case(9, C, C)[numpy.arange(R) % 9]
    x[R // 2] = -INF
    x[R // 3, C // 2] = numpy.nan
    x[3, C - 2:] = 30.0                       # the first of two
    x[5] = -2.0 ** 15                         # far below 0, as one
    tx = rows_of(x, torch.float32, xpad)
    k = min(C, 16)
    idx, z = teacher_case(R, C, k, 5)
    idx[1] = -1
    z[2, k // 2:] = -INF
    err = rows_of(numpy.full((R, C), 55.0), torch.bfloat16, epad)
    xs = f64(tx)
    none = numpy.isnan(xs).any(1) | (xs == -INF).all(1)
    labels = numpy.where(none, 0, xs.argmax(1))
    labels[::4] = rng.randint(0, C, len(labels[::4]))
    labels[7] = -1
    live = R - 1
    loss, n = counted(tx, idx, z, err, labels, live, 2.0)
    check_distill(tx, xs, idx, z, 2.0, err, loss, live)
    wrong = none | (xs.argmax(1) != labels)
    assert n == (wrong & (labels >= 0))[:live].sum()
    if epad:
        buf = err.as_strided((R * (C + epad),), (1,), 0)
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep.as_strided((R, C), (C + epad, 1), 0).fill_(False)
        assert torch.isnan(buf[keep]).all()


@pytest.mark.parametrize("R", [6, 66])
@pytest.mark.parametrize("C", [12, 1000, 50001])
@pytest.mark.parametrize("name", sorted(TYPES))
def test_errors_are_the_students_alone(R, C, name):
    """A teacher's class that does not exist, or a logit of it that is no
    number, leaves the student's likeliest class what it is."""
    tx = rows_of(logits_case(R, C, 2), TYPES[name])
    idx, z = teacher_case(R, C, 4)
    z[0::6, 1] = numpy.nan
    z[1::6, 3] = INF
    idx[2::6, 0] = C
    idx[3::6, 2] = 2 ** 31 - 1
    z[4::6] = -INF
    labels = f64(tx).argmax(1)
    loss, n = counted(tx, idx, z, torch.empty_like(tx), labels)
    assert n == 0
    bad = numpy.isin(numpy.arange(R) % 6, (0, 1, 2, 3))
    assert (numpy.isnan(f64(loss)) == bad).all()
    labels[::2] = (labels[::2] + 1) % C
    assert counted(tx, idx, z, torch.empty_like(tx), labels)[1] == R // 2


@pytest.mark.parametrize("R", [5, 70])
@pytest.mark.parametrize("C", [40, 1000, 50001, 140007])
@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("tau", [0.7, 4.0])
def test_a_class_that_is_named_twice(R, C, name, tau):
    """Loss and gradient are those of the class named once, with the logit
    that has the sum of its shares."""
    rng = numpy.random.RandomState(C + R)
    tx = rows_of(logits_case(R, C, 6), TYPES[name])
    at, once = teacher_case(R, C, 6, 3)
    once -= numpy.float32(500.0)              # (a shift has no effect)
    # each of them again and again, 128 places in all, out of order
    part = rng.normal(0, 2, (R, 6, 21))
    part -= numpy.logaddexp.reduce(part / tau, axis=2)[:, :, None] * tau
    idx = numpy.repeat(at[:, :, None], 21, 2).reshape(R, 126)
    z = (once[:, :, None] + part).reshape(R, 126)
    order = rng.permutation(126)
    idx, z = idx[:, order], z[:, order].astype(numpy.float32, "C")
    idx = numpy.ascontiguousarray(idx)
    err = torch.empty_like(tx)
    loss, _ = counted(tx, idx, z, err, numpy.zeros(R, int), tau=tau)
    joined = numpy.zeros((R, 6))
    for i in range(R):
        for j in range(6):
            same = idx[i] == at[i, j]
            joined[i, j] = tau * numpy.logaddexp.reduce(
                z[i, same].astype(float) / tau)
    check_distill(tx, f64(tx), at, joined, tau, err, loss)


@pytest.mark.parametrize("C", [50, 50001])
@pytest.mark.parametrize("R", [3, 80])
def test_a_divergence_is_not_below_zero(R, C):
    """A student that is as sure as a teacher whose only class is named four
    times."""
    x = numpy.full((R, C), -60.0)
    x[:, C // 2] = 0.0
    tx = rows_of(x, torch.float32)
    idx = numpy.full((R, 4), C // 2, numpy.int32)
    z = numpy.tile(numpy.float32([0.0, 1.0, -3.0, 2.0]), (R, 1))
    loss, _ = counted(tx, idx, z, torch.empty_like(tx),
                      numpy.full(R, C // 2))
    # four shares and their four logarithms, a few steps of fp32 each
    assert (numpy.abs(f64(loss)) <= 4 * 16 * E32).all()
    assert not any(math.isnan(v) for v in f64(loss))
