"""Layer norm, token log probabilities and distillation without a GPU: the
numpy references against other forms, and what the operators refuse."""

import math

import numpy
import pytest

torch = pytest.importorskip("torch")

from veles.znicz_amd import ops  # noqa: E402
from veles.znicz_amd.distillation import (  # noqa: E402
    numpy_distill, numpy_logprobs)

if not ops.available():
    pytest.skip("_mzk is not built", allow_module_level=True)


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


f4 = torch.float32
i4 = torch.int32


def test_numpy_logprobs_matches_log_softmax():
    x = numpy.random.RandomState(0).normal(0, 3, (5, 40))
    x[1, 3:] = -numpy.inf
    labels = [3, 1, -1, 0, 39]
    lp, ent, idx, top = numpy_logprobs(x, labels, 6)
    want = torch.log_softmax(torch.from_numpy(x), 1)
    for i, l in enumerate(labels):
        assert lp[i] == (0 if l < 0 else pytest.approx(want[i, l].item(),
                                                       abs=1e-12))
    p = want.exp()
    h = -torch.special.xlogy(p, p).sum(1)
    numpy.testing.assert_allclose(ent, h.numpy(), atol=1e-12)
    v, i = want.topk(6, dim=1)
    keep = v > -math.inf
    assert (idx == torch.where(keep, i, -1).numpy()).all()
    numpy.testing.assert_allclose(top, v.numpy(), atol=1e-12)


def test_numpy_distill_matches_autograd():
    rng = numpy.random.RandomState(1)
    x = torch.from_numpy(rng.normal(0, 2, (4, 30))).requires_grad_()
    idx = numpy.stack([rng.choice(30, 6, replace=False) for _ in range(4)])
    z = rng.normal(0, 2, (4, 6))
    idx[2, 4:] = -1
    for tau in (1.0, 2.5):
        zz = torch.from_numpy(z) / tau
        zz = zz.masked_fill(torch.from_numpy(idx) < 0, -math.inf)
        lnq = torch.log_softmax(zz, 1)
        q = lnq.exp()
        lnp = torch.log_softmax(x / tau, 1).gather(
            1, torch.from_numpy(idx).clamp(min=0))
        part = torch.where(q > 0, q * (lnq - lnp), torch.zeros_like(q))
        loss = tau * tau * part.sum(1)
        grad, = torch.autograd.grad(loss.sum(), x)
        got_l, got_g = numpy_distill(x.detach().numpy(), idx, z, tau)
        numpy.testing.assert_allclose(got_l, loss.detach().numpy(),
                                      atol=1e-12)
        numpy.testing.assert_allclose(got_g, grad.numpy(), atol=1e-12)


# -- refusals ----------------------------------------------------------------

def refused(match, f, *a, **k):
    with pytest.raises(RuntimeError, match=match):
        f(*a, **k)


def test_operators_need_a_gpu():
    x, y = t(2, 8), t(2, 8)
    refused("not on a GPU", ops.layer_norm_fwd, x, y, None, None, None, None)
    refused("not on a GPU", ops.layer_norm_bwd, x, y, None, t(2, dtype=f4),
            t(2, dtype=f4), t(2, 8))
    refused("not on a GPU", ops.token_logprobs, x, entropy=t(2, dtype=f4))
    refused("not on a GPU", ops.eval_distill, x, t(2, 3, dtype=i4),
            t(2, 3, dtype=f4), y)


def test_layer_norm_refusals():
    x, y = t(4, 8), t(4, 8)
    f = ops.layer_norm_fwd
    refused("bf16, fp16 or fp32", f, t(4, 8, dtype=torch.float64),
            t(4, 8, dtype=torch.float64), None, None, None, None)
    refused("out is", f, x, t(4, 8, dtype=f4), None, None, None, None)
    refused("out is", f, x, t(4, 9), None, None, None, None)
    refused("out is", f, x, t(3, 8), None, None, None, None)
    refused("no columns", f, t(4, 0), t(4, 0), None, None, None, None)
    refused("contiguous", f, t(8, 4).t(), y, None, None, None, None)
    refused("contiguous", f, x, t(8, 4).t(), None, None, None, None)
    refused("overlap", f, x, t(1, 8).expand(4, 8), None, None, None, None)
    refused("weights has", f, x, y, t(7, dtype=f4), None, None, None)
    refused("bias is", f, x, y, None, t(8), None, None)
    refused("mean has", f, x, y, None, None, t(5, dtype=f4), None)
    refused("rstd must be contiguous", f, x, y, None, None, None,
            t(8, dtype=f4)[::2])
    refused("eps", f, x, y, None, None, None, None, -1.0)
    refused("eps", f, x, y, None, None, None, None, math.nan)
    m = t(4, dtype=f4)
    g = ops.layer_norm_bwd
    refused("err_output is", g, t(4, 7), x, None, m, m, y)
    refused("err_input is", g, x, y, None, m, m, t(4, 8, dtype=f4))
    refused("grad_w has", g, x, y, None, m, m, None, t(9, dtype=f4))
    refused("grad_b is", g, x, y, None, m, m, None, None, t(8))
    refused("mean has", g, x, y, None, t(3, dtype=f4), m, None)


def test_partial_overlaps_are_refused():
    buf = t(4, 24)
    f = ops.layer_norm_fwd
    a = buf[:, :8]
    refused("in part", f, a, buf[:, 4:12], None, None, None, None)
    refused("in part", f, buf[:, 4:12], a, None, None, None, None)
    refused("in part", f, a, buf.view(-1).as_strided((4, 8), (23, 1)), None,
            None, None, None)
    refused("in part", f, buf.view(-1)[:32].view(4, 8),
            buf.view(-1)[8:40].view(4, 8), None, None, None, None)
    # the last column of a row beside the next row's first
    refused("in part", f, buf[:, :8].as_strided((3, 8), (24, 1), 20),
            buf[:3, :8], None, None, None, None)
    # beside each other, or one and the same: allowed as far as that
    refused("not on a GPU", f, a, buf[:, 8:16], None, None, None, None)
    refused("not on a GPU", f, a, a, None, None, None, None)
    refused("in part", ops.layer_norm_bwd, a, t(4, 8), None,
            t(4, dtype=f4), t(4, dtype=f4), buf[:, 4:12])
    refused("in part", ops.layer_norm_bwd, t(4, 8), a, None,
            t(4, dtype=f4), t(4, dtype=f4), buf[:, 4:12])
    x = t(4, 8, dtype=f4)
    refused("in part", ops.eval_distill, x, t(4, 2, dtype=i4),
            t(4, 2, dtype=f4), x.view(torch.bfloat16)[:, :8])


def test_outputs_over_other_arrays_are_refused():
    """No output may lie over another one, nor over what is read."""
    x, y, w = t(4, 8), t(4, 8), t(8, dtype=f4)
    m, r = t(4, dtype=f4), t(4, dtype=f4)
    one = "mean and rstd overlap|rstd and mean overlap"
    refused(one, ops.layer_norm_fwd, x, y, w, None, m, m)
    refused("weights", ops.layer_norm_fwd, x, y, w, None, w[:4], r)
    z = t(4, 8, dtype=f4)
    refused("bias", ops.layer_norm_fwd, z, t(4, 8, dtype=f4), None, w, w[4:],
            r)
    refused("out and mean", ops.layer_norm_fwd, t(4, 8, dtype=f4), z, w,
            None, z.view(-1)[8:12], r)
    refused("grad_w and grad_b", ops.layer_norm_bwd, x, y, None, m, r, None,
            w, w)
    refused("weights", ops.layer_norm_bwd, x, y, w, m, r, None, w)
    refused("mean", ops.layer_norm_bwd, z[:4, :4], t(4, 4, dtype=f4), None,
            m, r, None, m)
    e, i, p = t(4, dtype=f4), t(4, 2, dtype=i4), t(4, 2, dtype=f4)
    lab = t(4, dtype=i4)
    f = ops.token_logprobs
    refused("logprob and entropy", f, x, lab, e, e)
    refused("labels", f, x, lab, lab.view(f4))
    refused("top_idx and top_logprob", f, x, top_idx=i,
            top_logprob=i.view(f4))
    refused("logits", f, z, entropy=z[1, :4])
    d = ops.eval_distill
    refused("top_logit", d, x, i, p, y, p.view(-1)[:4])
    refused("labels", d, x, i, p, y, None, labels=lab, n_err=lab)
    refused("top_idx", d, x, i, p, y, None, labels=lab, n_err=i)
    refused("loss", d, z, i, p, z, z[3, 4:])
    # beside each other, or between a matrix's rows
    both = t(12, dtype=f4)
    refused("not on a GPU", f, x, lab, both[:4], both[4:8])
    wide = t(4, 16, dtype=f4)
    refused("not on a GPU", f, wide[:, :8], entropy=wide[0, 8:12])
    refused("overlap", f, wide[:, :8], entropy=wide[0, 7:11])
    refused("overlap", f, wide[:, :8],
            entropy=wide.view(-1)[14:18])


def test_token_logprobs_class_limit():
    refused("at most 2.24", ops.token_logprobs, t(1, (1 << 24) + 1),
            entropy=t(1, dtype=f4))


def test_token_logprobs_refusals():
    x = t(4, 50)
    f = ops.token_logprobs
    e = t(4, dtype=f4)
    refused("labels and logprob", f, x, labels=t(4, dtype=i4))
    refused("labels and logprob", f, x, logprob=e)
    refused("labels is", f, x, labels=t(4, dtype=torch.int64), logprob=e)
    refused("labels has", f, x, labels=t(3, dtype=i4), logprob=e)
    refused("entropy is", f, x, entropy=t(4))
    refused("come together", f, x, top_idx=t(4, 3, dtype=i4))
    refused("top_logprob is", f, x, top_idx=t(4, 3, dtype=i4),
            top_logprob=t(4, 2, dtype=f4))
    refused("top_idx must be", f, x, top_idx=t(3, 3, dtype=i4),
            top_logprob=t(3, 3, dtype=f4))
    refused("alternatives", f, x, top_idx=t(4, 129, dtype=i4),
            top_logprob=t(4, 129, dtype=f4))
    refused("batch", f, x, entropy=e, batch=5)
    refused("batch", f, x, entropy=e, batch=-1)
    refused("bf16, fp16 or fp32", f, t(4, 50, dtype=torch.int32), entropy=e)
    refused("contiguous", f, t(50, 4).t(), entropy=e)


def test_eval_distill_refusals():
    x, err = t(4, 50), t(4, 50)
    idx, z = t(4, 3, dtype=i4), t(4, 3, dtype=f4)
    f = ops.eval_distill
    refused("err_output is", f, x, idx, z, t(4, 49))
    refused("err_output is", f, x, idx, z, t(4, 50, dtype=f4))
    refused("err_output is", f, t(4, 50, dtype=f4), idx, z,
            t(4, 50, dtype=torch.float16))
    refused("top_logit is", f, x, idx, t(4, 2, dtype=f4), err)
    refused("top_idx is", f, x, idx.long(), z, err)
    refused("top_idx must be", f, x, t(3, 3, dtype=i4), z, err)
    refused("teacher's classes", f, x, t(4, 0, dtype=i4),
            t(4, 0, dtype=f4), err)
    refused("teacher's classes", f, x, t(4, 129, dtype=i4),
            t(4, 129, dtype=f4), err)
    refused("loss has", f, x, idx, z, err, t(3, dtype=f4))
    for tau in (0.0, -1.0, math.nan, math.inf, 1e-4, 2e3):
        refused("temperature", f, x, idx, z, err, None, None, tau)
    refused("batch", f, x, idx, z, err, None, 9)
    refused("come together", f, x, idx, z, err, labels=t(4, dtype=i4))
    refused("n_err is empty", f, x, idx, z, err, labels=t(4, dtype=i4),
            n_err=t(0, dtype=i4))
    refused("contiguous", f, x, t(3, 4, dtype=i4).t(), z, err)
