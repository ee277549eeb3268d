"""Layer norm, token log probabilities and distillation on the GPU against
plain 64-bit forms.

Tolerances count roundings.  e32 = 2^-24 is half a step of fp32, e(t) half a
step of the stored type.  A sum of n terms in chains of n/256 (a workgroup's
share) plus a tree is off by at most (n/256 + 32) e32 of the sum of the
terms' magnitudes; powers are off by their exponent's rounding, |u| e32.
"""

import math

import numpy
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no GPU", allow_module_level=True)

from veles.znicz_amd import ops  # noqa: E402
from veles.znicz_amd.distillation import (  # noqa: E402
    numpy_distill, numpy_logprobs)

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
E32 = 2.0 ** -24
INF = math.inf


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of the smallest step (16-bit values below the normal range)."""
    return {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134,
            torch.float32: 2.0 ** -126}[dtype]


def rows_of(values, dtype, pad=0, shift=0):
    """values [R, C] on the GPU as rows of C + pad, `shift` elements into
    their buffer; what lies between the rows is NaN."""
    v = torch.as_tensor(values)
    R, C = v.shape
    buf = torch.full((R * (C + pad) + shift,), math.nan, dtype=dtype,
                     device="cuda")
    t = buf.as_strided((R, C), (C + pad, 1), shift)
    t.copy_(v.to(dtype))
    return t


def f64(t):
    return t.detach().double().cpu().numpy()


def near(got, want, tol):
    got, want = numpy.asarray(got, float), numpy.asarray(want, float)
    assert got.shape == want.shape
    nan = numpy.isnan(want)
    assert (numpy.isnan(got) == nan).all()
    inf = numpy.isinf(want)
    assert (got[inf] == want[inf]).all()
    ok = ~nan & ~inf
    d = numpy.abs(got[ok] - want[ok])
    tol = numpy.broadcast_to(tol, want.shape)[ok]
    assert (d <= tol).all(), (d / numpy.maximum(tol, 1e-300)).max()


# ---------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------

NORM_SIZES = [(1, 1), (3, 1), (5, 2), (4, 7), (9, 8), (1, 64), (4, 65),
              (77, 96), (33, 200), (130, 512), (6, 1000), (5, 1021),
              (2, 2048), (37, 2049), (19, 4096), (3, 8192), (5, 8200),
              (3, 16384), (2, 20001), (2, 33000), (1, 70001), (700, 24)]


def norm_case(R, C, dtype, seed=0):
    rng = numpy.random.RandomState(seed)
    x = rng.normal(0.5, 2.0, (R, C))
    dy = rng.normal(0, 1.0, (R, C))
    w = rng.normal(1, 0.3, C).astype(numpy.float32)
    b = rng.normal(0, 0.3, C).astype(numpy.float32)
    return x, dy, w, b


def cuda(a):
    return None if a is None else torch.from_numpy(a).cuda()


def check_norm_fwd(x, w, b, y, mean, rstd, eps, dtype):
    R, C = x.shape
    xd = f64(x)
    mu = xd.mean(1, keepdims=True)
    var = ((xd - mu) ** 2).mean(1, keepdims=True)
    r = 1 / numpy.sqrt(var + eps)
    h = (xd - mu) * r
    wd = 1.0 if w is None else w.astype(float)
    bd = 0.0 if b is None else b.astype(float)
    want = h * wd + bd
    n = (C / 256 + 32) * E32
    emu = n * numpy.abs(xd).mean(1, keepdims=True)
    # the mean's error shifts all of a row; the deviation's is relative
    tol = numpy.abs(wd) * r * (emu + E32 * (numpy.abs(xd) + numpy.abs(mu))) \
        + numpy.abs(wd * h) * (2 * n + r * emu) + numpy.abs(bd) * 2 * E32
    near(f64(y), want, tol + numpy.abs(want) * half_step(dtype) +
         tiny(dtype))
    if mean is not None:
        near(f64(mean), mu[:, 0], (emu + numpy.abs(mu) * E32)[:, 0])
        # (the variance is off by the square of the mean's error too)
        near(f64(rstd), r[:, 0],
             (r * (n + (r * emu) ** 2 + 4 * E32))[:, 0])


def check_norm_bwd(dy, x, w, mean, rstd, dx, dw, db, dtype):
    R, C = x.shape
    xd, g0 = f64(x), f64(dy)
    mu, r = f64(mean)[:, None], f64(rstd)[:, None]
    h = (xd - mu) * r
    wd = 1.0 if w is None else w.astype(float)
    g = g0 * wd
    s1 = g.mean(1, keepdims=True)
    s2 = (g * h).mean(1, keepdims=True)
    n = (C / 256 + 32) * E32
    eh = 2 * E32 * r * (numpy.abs(xd) + numpy.abs(mu))
    a1 = numpy.abs(g).mean(1, keepdims=True)
    a2 = numpy.abs(g * h).mean(1, keepdims=True)
    if dx is not None:
        want = r * (g - s1 - h * s2)
        tol = r * (n * (numpy.abs(g) + a1 + numpy.abs(h) * a2) +
                   eh * a2 + numpy.abs(h) *
                   (numpy.abs(g) * eh).mean(1, keepdims=True))
        near(f64(dx), want, tol + numpy.abs(want) * half_step(dtype) +
             tiny(dtype))
    # rows in chains of at most rows/128, and at most 1100 partial sums
    n = (R / 128 + 1100) * E32
    if dw is not None:
        near(f64(dw), (g0 * h).sum(0), (n * numpy.abs(g0 * h) +
                                        numpy.abs(g0) * eh).sum(0))
    if db is not None:
        near(f64(db), g0.sum(0), n * numpy.abs(g0).sum(0))


@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 0), (8, 8), (3, 1)])
@pytest.mark.parametrize("name", sorted(TYPES))
@pytest.mark.parametrize("R,C", NORM_SIZES)
def test_layer_norm(R, C, name, pad, shift):
    dtype = TYPES[name]
    x, dy, w, b = norm_case(R, C, dtype)
    tx, tdy = (rows_of(v, dtype, pad, shift) for v in (x, dy))
    y = rows_of(numpy.zeros((R, C)), dtype, pad, shift)
    mean = torch.empty(R, device="cuda")
    rstd = torch.empty(R, device="cuda")
    ops.layer_norm_fwd(tx, y, cuda(w), cuda(b), mean, rstd, 1e-5)
    check_norm_fwd(tx, w, b, y, mean, rstd, 1e-5, dtype)
    dx = rows_of(numpy.zeros((R, C)), dtype, pad, shift)
    dw, db = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
    ops.layer_norm_bwd(tdy, tx, cuda(w), mean, rstd, dx, dw, db)
    check_norm_bwd(tdy, tx, w, mean, rstd, dx, dw, db, dtype)
    # what lies between and before the rows is left as it was
    if pad or shift:
        buf = dx.as_strided((R * (C + pad) + shift,), (1,), 0)
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep.as_strided((R, C), (C + pad, 1), shift).fill_(False)
        assert torch.isnan(buf[keep]).all()


@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 3)])
@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("R,C", [
    (300001, 5), (200003, 24), (70001, 96), (20003, 300), (9001, 1000),
    (4099, 2048), (2500, 4097), (1501, 8000), (600, 16384), (601, 17000),
    (300, 33000)])
def test_layer_norm_many_rows(R, C, name, pad, shift):
    """Rows enough for several steps of every team, also over the inputs."""
    dtype = TYPES[name]
    x, dy, w, b = norm_case(R, C, dtype, 1)
    tx, tdy = (rows_of(v, dtype, pad, shift) for v in (x, dy))
    y, dx = torch.empty_like(tx), torch.empty_like(tx)
    mean = torch.empty(R, device="cuda")
    rstd = torch.empty(R, device="cuda")
    ops.layer_norm_fwd(tx, y, cuda(w), cuda(b), mean, rstd, 1e-5)
    check_norm_fwd(tx, w, b, y, mean, rstd, 1e-5, dtype)
    dw, db = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
    ops.layer_norm_bwd(tdy, tx, cuda(w), mean, rstd, dx, dw, db)
    check_norm_bwd(tdy, tx, w, mean, rstd, dx, dw, db, dtype)
    dw2, db2 = torch.empty_like(dw), torch.empty_like(db)
    ops.layer_norm_bwd(tdy, tx, cuda(w), mean, rstd, tdy, dw2, db2)
    assert torch.equal(tdy, dx)
    assert torch.equal(dw, dw2) and torch.equal(db, db2)
    ops.layer_norm_fwd(tx, tx, cuda(w), cuda(b), None, None, 1e-5)
    assert torch.equal(tx, y)


@pytest.mark.parametrize("R,C", [(3, 40), (600, 96), (5, 4096), (2, 20001)])
@pytest.mark.parametrize("what", ["no_w", "no_b", "no_dx", "no_dw", "no_db",
                                  "only_dx", "no_stats"])
def test_layer_norm_parts(R, C, what):
    dtype = torch.bfloat16
    x, dy, w, b = norm_case(R, C, dtype, 3)
    tx, tdy = rows_of(x, dtype), rows_of(dy, dtype)
    if what in ("no_w",):
        w = None
    if what == "no_b":
        b = None
    y = torch.empty_like(tx)
    mean = torch.empty(R, device="cuda")
    rstd = torch.empty(R, device="cuda")
    ops.layer_norm_fwd(tx, y, cuda(w), cuda(b), mean, rstd, 1e-3)
    check_norm_fwd(tx, w, b, y, mean, rstd, 1e-3, dtype)
    if what == "no_stats":
        y2 = torch.empty_like(tx)
        ops.layer_norm_fwd(tx, y2, cuda(w), cuda(b), None, None, 1e-3)
        assert torch.equal(y, y2)
        return
    dx = torch.empty_like(tx) if what != "no_dx" else None
    dw = torch.empty(C, device="cuda") \
        if what not in ("no_dw", "only_dx") else None
    db = torch.empty(C, device="cuda") \
        if what not in ("no_db", "only_dx") else None
    ops.layer_norm_bwd(tdy, tx, cuda(w), mean, rstd, dx, dw, db)
    check_norm_bwd(tdy, tx, w, mean, rstd, dx, dw, db, dtype)


def test_layer_norm_accumulates_and_repeats_to_the_bit():
    R, C = 4000, 96
    x, dy, w, b = norm_case(R, C, torch.bfloat16, 5)
    tx, tdy = rows_of(x, torch.bfloat16), rows_of(dy, torch.bfloat16)
    y, dx = torch.empty_like(tx), torch.empty_like(tx)
    mean, rstd = torch.empty(R).cuda(), torch.empty(R).cuda()
    ops.layer_norm_fwd(tx, y, cuda(w), cuda(b), mean, rstd)
    dw, db = torch.empty(C).cuda(), torch.empty(C).cuda()
    ops.layer_norm_bwd(tdy, tx, cuda(w), mean, rstd, dx, dw, db)
    dw2, db2 = torch.ones(C).cuda(), torch.full((C,), 2.0).cuda()
    ops.layer_norm_bwd(tdy, tx, cuda(w), mean, rstd, dx, dw2, db2,
                       accumulate=True)
    assert torch.equal(dw2, dw + 1) and torch.equal(db2, db + 2)


@pytest.mark.parametrize("C", [1, 100, 4096, 20001])
def test_layer_norm_of_no_rows(C):
    x = torch.empty(0, C, dtype=torch.bfloat16, device="cuda")
    e = torch.empty(0, device="cuda")
    dw = torch.full((C,), 7.0, device="cuda")
    db = torch.full((C,), 7.0, device="cuda")
    ops.layer_norm_fwd(x, torch.empty_like(x), None, None, e, e)
    ops.layer_norm_bwd(x, x, None, e, e, torch.empty_like(x), dw, db, True)
    assert (dw == 7).all() and (db == 7).all()
    ops.layer_norm_bwd(x, x, None, e, e, torch.empty_like(x), dw, db)
    assert (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("C", [96, 1000, 4096, 20001])
def test_layer_norm_in_place(C):
    R = 9
    x, dy, w, b = norm_case(R, C, torch.float32, 6)
    tx, tdy = rows_of(x, torch.float32), rows_of(dy, torch.float32)
    mean, rstd = torch.empty(R).cuda(), torch.empty(R).cuda()
    y = torch.empty_like(tx)
    ops.layer_norm_fwd(tx, y, cuda(w), cuda(b), mean, rstd)
    y2 = tx.clone()
    ops.layer_norm_fwd(y2, y2, cuda(w), cuda(b), None, None)
    assert torch.equal(y, y2)
    dx = torch.empty_like(tx)
    dw, db = torch.empty(C).cuda(), torch.empty(C).cuda()
    ops.layer_norm_bwd(tdy, tx, cuda(w), mean, rstd, dx, dw, db)
    for over in (0, 1):
        ins = [tdy.clone(), tx.clone()]
        dw2, db2 = torch.empty(C).cuda(), torch.empty(C).cuda()
        ops.layer_norm_bwd(ins[0], ins[1], cuda(w), mean, rstd, ins[over],
                           dw2, db2)
        assert torch.equal(ins[over], dx)
        assert torch.equal(dw, dw2) and torch.equal(db, db2)


@pytest.mark.parametrize("C", [8, 300, 4096, 20001])
def test_layer_norm_special_rows(C):
    """A row of equal values has no deviation; NaN and infinity stay in
    their row."""
    x = numpy.random.RandomState(1).normal(0, 1, (6, C))
    x[1] = 3.0
    x[2, C // 2] = numpy.nan
    x[3, C - 1] = numpy.inf
    x[4] = -1e30
    tx = rows_of(x, torch.float32)
    y = torch.empty_like(tx)
    mean, rstd = torch.empty(6).cuda(), torch.empty(6).cuda()
    ops.layer_norm_fwd(tx, y, None, None, mean, rstd, 1e-5)
    assert torch.isfinite(y[[0, 1, 5]]).all()
    assert (y[1] == 0).all()
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).any()
    assert abs(rstd[1].item() - 1e5 ** 0.5) <= 1e5 ** 0.5 * 4 * E32


def test_layer_norm_broadcast_rows():
    """Inputs whose rows are one row (stride 0)."""
    C, R = 1000, 50
    x, dy, w, b = norm_case(1, C, torch.bfloat16, 8)
    tx = rows_of(x, torch.bfloat16).expand(R, C)
    tdy = rows_of(dy, torch.bfloat16).expand(R, C)
    y = torch.empty(R, C, dtype=torch.bfloat16, device="cuda")
    mean, rstd = torch.empty(R).cuda(), torch.empty(R).cuda()
    ops.layer_norm_fwd(tx, y, cuda(w), cuda(b), mean, rstd)
    check_norm_fwd(tx, w, b, y, mean, rstd, 1e-5, torch.bfloat16)
    dx, dw, db = torch.empty_like(y), torch.empty(C).cuda(), \
        torch.empty(C).cuda()
    ops.layer_norm_bwd(tdy, tx, cuda(w), mean, rstd, dx, dw, db)
    check_norm_bwd(tdy, tx, w, mean, rstd, dx, dw, db, torch.bfloat16)


def test_layer_norm_gradient_by_differences():
    """The loss sum(y dy) moves as dx, dw and db say."""
    R, C = 3, 40
    x, dy, w, b = norm_case(R, C, torch.float32, 9)
    tx, tdy = rows_of(x, torch.float32), rows_of(dy, torch.float32)
    mean, rstd = torch.empty(R).cuda(), torch.empty(R).cuda()
    dx, dw, db = torch.empty_like(tx), torch.empty(C).cuda(), \
        torch.empty(C).cuda()
    ops.layer_norm_fwd(tx, torch.empty_like(tx), cuda(w), cuda(b), mean,
                       rstd)
    ops.layer_norm_bwd(tdy, tx, cuda(w), mean, rstd, dx, dw, db)

    def loss(x, w, b):
        m = x.mean(1, keepdims=True)
        v = ((x - m) ** 2).mean(1, keepdims=True)
        return (((x - m) / numpy.sqrt(v + 1e-5) * w + b) * f64(tdy)).sum()

    args = [f64(tx), w.astype(float), b.astype(float)]
    for k, got in ((0, f64(dx)), (1, f64(dw)), (2, f64(db))):
        rng = numpy.random.RandomState(k)
        for _ in range(4):
            d = rng.normal(0, 1, args[k].shape)
            h = 1e-5
            up = [a + h * d if i == k else a for i, a in enumerate(args)]
            dn = [a - h * d if i == k else a for i, a in enumerate(args)]
            want = (loss(*up) - loss(*dn)) / (2 * h)
            # differences: h^2 and 2^-52 |loss| / h; the kernel: 64 e32
            assert abs((got * d).sum() - want) <= \
                1e-6 + 64 * E32 * numpy.abs(got * d).sum()


# ---------------------------------------------------------------------------
# token log probabilities
# ---------------------------------------------------------------------------

PROB_SIZES = [(1, 1), (2, 2), (3, 5), (4, 64), (3, 65), (5, 257), (256, 10),
              (7, 1000), (3, 4095), (3, 4096), (2, 8193), (4, 20000),
              (2, 50001), (1, 131072), (2, 140007)]


def logits_case(R, C, seed=0, masked=0.0):
    rng = numpy.random.RandomState(seed)
    x = rng.normal(0, 3, (R, C))
    if masked:
        x[:, rng.rand(C) < masked] = -INF
    return x


def run_logprobs(tx, labels, top, batch=None):
    R = tx.shape[0]
    k = min(top, 128)
    out = (torch.full((R,), 55.0, device="cuda"),
           torch.full((R,), 55.0, device="cuda"),
           torch.full((R, k), 55, dtype=torch.int32, device="cuda"),
           torch.full((R, k), 55.0, device="cuda"))
    ops.token_logprobs(tx, torch.as_tensor(
        labels, dtype=torch.int32).cuda(), *out, batch=batch)
    return out


def check_logprobs(tx, labels, out, live=None):
    live = tx.shape[0] if live is None else live
    got = [f64(t) for t in out]
    C, k = tx.shape[1], out[2].shape[1]
    x = f64(tx)[:live]
    lp, ent, idx, top = numpy_logprobs(x, numpy.asarray(labels)[:live], k)
    m = x.max(1) if live else numpy.zeros(0)
    m = numpy.where(numpy.isfinite(m), m, 0)
    n = (C / 256 + 32) * E32
    ln = math.log(C) + 1

    def tol(v):
        v = numpy.where(numpy.isfinite(v), numpy.abs(v), 0)
        return n + 4 * E32 * (v + ln)
    near(got[0][:live], lp, tol(lp))
    near(got[1][:live], ent, (n + 64 * E32) * (2 + 2 * ln))
    assert (got[2][:live] == idx).all()
    near(got[3][:live], top, tol(top))
    assert (got[0][live:] == 0).all() and (got[1][live:] == 0).all()
    assert (got[2][live:] == -1).all() and (got[3][live:] == 0).all()


@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 0), (8, 8), (3, 1)])
@pytest.mark.parametrize("name", sorted(TYPES))
@pytest.mark.parametrize("R,C", PROB_SIZES)
def test_token_logprobs(R, C, name, pad, shift):
    x = logits_case(R, C, R + C)
    tx = rows_of(x, TYPES[name], pad, shift)
    labels = numpy.random.RandomState(2).randint(-1, C, R)
    check_logprobs(tx, labels, run_logprobs(tx, labels, 20))


@pytest.mark.parametrize("top", [1, 2, 5, 17, 63, 64, 65, 100, 127, 128])
@pytest.mark.parametrize("R,C", [(3, 70), (2, 1000), (3, 20000),
                                 (1, 140007)])
@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_token_logprobs_top(R, C, name, top):
    tx = rows_of(logits_case(R, C, top), TYPES[name])
    check_logprobs(tx, [C - 1] * R, run_logprobs(tx, [C - 1] * R, top))


@pytest.mark.parametrize("C", [129, 200, 255, 256, 257, 270, 400, 511, 513,
                               700, 1000, 1023, 1025, 1039, 1500])
@pytest.mark.parametrize("name", sorted(TYPES))
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 5)])
def test_token_logprobs_short_rows_of_many_alternatives(C, name, pad, shift):
    """Fewer packs than threads, and than alternatives."""
    rng = numpy.random.RandomState(C)
    x = rng.normal(0, 3, (9, C))
    x[1] = numpy.round(x[1])                    # equal values
    x[2, rng.rand(C) < 0.8] = -INF
    x[3, 130:] = -INF
    x[4] = 2.0
    x[5, :C // 2] += 100.0                      # all in the same packs
    x[6, ::9] += 100.0
    x[7, :] = -numpy.arange(C)
    tx = rows_of(x, TYPES[name], pad, shift)
    labels = numpy.arange(9) * 11 % C
    for top in (33, 66, 128):
        check_logprobs(tx, labels, run_logprobs(tx, labels, top))


@pytest.mark.parametrize("R,C,name", [
    (1, 600011, "bf16"),       # as many parts as there are, 128 of each
    (1, 300007, "f32"),
    (1, (1 << 24) - 3, "f16"),
    (600, (1 << 20) - 5, "bf16"),   # the longest parts, many rows
    (600, (1 << 19) - 3, "f32"),
    (600, (1 << 20) + 1, "f16")])
def test_token_logprobs_long_rows(R, C, name):
    """(one row again and again: a stride of 0)"""
    tx = rows_of(logits_case(1, C, 11), TYPES[name])
    for top in (128, 3):
        out = run_logprobs(tx.expand(R, C), [C - 1] * R, top)
        check_logprobs(tx, [C - 1], [t[:1] for t in out])
        for t in out:
            assert torch.equal(t, t[:1].expand_as(t))


@pytest.mark.parametrize("C", [1, 3, 64, 1000, 20000, 60000, 140007])
@pytest.mark.parametrize("name", sorted(TYPES))
def test_token_logprobs_orders(C, name):
    """Rows whose order is the worst for one way of looking or another:
    equal values, steps, rising, falling, both zeros, all at one end."""
    rows = [numpy.zeros(C), numpy.arange(C) % 7.0,
            numpy.arange(C) / 100.0, -numpy.arange(C) / 100.0,
            numpy.where(numpy.arange(C) % 2, 0.0, -0.0),
            numpy.where(numpy.arange(C) < C // 3, 5.0, -5.0),
            numpy.where(numpy.arange(C) % 512 < 8, 9.0, 1.0) +
            numpy.arange(C) % 8 * 0.5,
            numpy.where(numpy.arange(C) % 4096 < 64,
                        numpy.arange(C) % 64 * 1.0, -3.0)]
    tx = rows_of(numpy.stack(rows), TYPES[name])
    labels = numpy.arange(len(rows)) % C
    for top in (1, 40, 128):
        check_logprobs(tx, labels, run_logprobs(tx, labels, top))


@pytest.mark.parametrize("C", [5, 300, 4096, 50001, 140007])
@pytest.mark.parametrize("name", sorted(TYPES))
def test_token_logprobs_masks(C, name):
    dtype = TYPES[name]
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = logits_case(14, C, 4)
    x[0] = -INF
    x[1, 1:] = -INF
    x[2, :C - 1] = -INF
    x[3] = low
    x[4, :C // 2] = low
    x[5, C // 2] = numpy.nan
    x[6] = numpy.nan
    x[7, C - 1] = INF
    x[8] = INF
    x[9, ::2] = -INF
    x[10, C // 3] = high
    x[11] = -INF
    x[11, C // 2] = low
    x[12] = high
    labels = [0, 0, 0, 1, C - 1, 0, -1, 2, 1, 0, 1, C // 2, 3, C]
    tx = rows_of(x, dtype, 1)
    out = run_logprobs(tx, labels, 20)
    check_logprobs(tx, labels, out)
    assert torch.isnan(out[0][13])             # no such class


@pytest.mark.parametrize("C", [16390, 50001, 140007])
@pytest.mark.parametrize("name", sorted(TYPES))
@pytest.mark.parametrize("top", [7, 128])
def test_token_logprobs_many_long_rows(C, name, top):
    """Rows enough not to be cut into parts, masked, in the worst orders."""
    dtype = TYPES[name]
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    n = numpy.arange(C)
    x = logits_case(16, C, 4)
    x[0] = -INF
    x[1, 1:] = -INF
    x[2, :C - 1] = -INF
    x[3] = low
    x[4, C // 2] = numpy.nan
    x[5, C - 1] = INF
    x[6, ::2] = -INF
    x[7, C // 3] = high
    x[8] = 0.0
    x[9] = n % 7
    x[10] = n / 100.0
    x[11] = numpy.where(n % 2, 0.0, -0.0)
    x[12] = numpy.where(n % 4096 < 64, n % 64 * 1.0, -3.0)
    x[13] = numpy.where(n < 40, -n * 1.0, -INF)
    x[14] = -n / 100.0
    turns = 13
    tx = rows_of(numpy.tile(x, (turns, 1)), dtype, 0, 1)
    labels = numpy.arange(16 * turns) * 37 % C
    live = 16 * turns - 3
    out = run_logprobs(tx, labels, top, live)
    # (the first rows, at every place within 16 bytes, and the last ones)
    check_logprobs(tx[:48], labels[:48], [t[:48] for t in out])
    check_logprobs(tx[-20:], labels[-20:], [t[-20:] for t in out], 17)


def test_token_logprobs_huge_offset():
    """Shifted logits have the same answers, whatever the shift."""
    rng = numpy.random.RandomState(0)
    x = numpy.round(rng.normal(0, 3, (2, 5000)) * 8) / 8
    for shift in (0.0, 1e3, -1e5):
        tx = rows_of(x + shift, torch.float32)
        check_logprobs(tx, [3, 4], run_logprobs(tx, [3, 4], 10))


@pytest.mark.parametrize("batch", [0, 1, 6, 7])
def test_token_logprobs_padded_batch(batch):
    x = logits_case(7, 1000, 5)
    tx = rows_of(x, torch.bfloat16)
    tx[batch:] = math.nan
    labels = [4] * 7
    check_logprobs(tx, labels, run_logprobs(tx, labels, 5, batch), batch)


@pytest.mark.parametrize("C", [1000, 140007])
def test_token_logprobs_single_outputs(C):
    tx = rows_of(logits_case(3, C, 6), torch.bfloat16)
    labels = torch.tensor([1, 2, 3], dtype=torch.int32).cuda()
    lp, ent, idx, top = run_logprobs(tx, [1, 2, 3], 7)
    a = torch.empty_like(lp)
    ops.token_logprobs(tx, labels=labels, logprob=a)
    assert torch.equal(a, lp)
    ops.token_logprobs(tx, entropy=a)
    assert torch.equal(a, ent)
    i, t = torch.empty_like(idx), torch.empty_like(top)
    ops.token_logprobs(tx, top_idx=i, top_logprob=t)
    assert torch.equal(i, idx) and torch.equal(t, top)


def test_token_logprobs_of_no_rows():
    x = torch.empty(0, 50, dtype=torch.bfloat16, device="cuda")
    ops.token_logprobs(x, entropy=torch.empty(0, device="cuda"))


# ---------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------

def teacher_case(R, C, k, seed=0):
    rng = numpy.random.RandomState(seed)
    idx = numpy.stack([rng.choice(C, k, replace=k > C) for _ in range(R)])
    z = rng.normal(0, 2, (R, k))
    return idx.astype(numpy.int32), z.astype(numpy.float32)


def run_distill(tx, idx, z, tau, batch=None, err=None):
    R = tx.shape[0]
    err = torch.full_like(tx, 55.0) if err is None else err
    loss = torch.full((R,), 55.0, device="cuda")
    ops.eval_distill(tx, cuda(idx), cuda(z), err, loss, batch, tau)
    return err, loss


def check_distill(tx, x, idx, z, tau, err, loss, live=None):
    live = x.shape[0] if live is None else live
    C = x.shape[1]
    want_l, want_g = numpy_distill(x[:live], idx[:live], z[:live], tau)
    dtype = err.dtype
    n = (C / 256 + 64) * E32
    with numpy.errstate(all="ignore"):
        m = x[:live].max(1, keepdims=True)
        u = numpy.abs(x[:live] - m) / tau * 1.4427
        p = numpy.abs(want_g)                  # p and q where both are
        q = numpy.zeros_like(want_g)
        for i in range(live):
            ok = (idx[i] >= 0) & (idx[i] < C)
            numpy.add.at(q[i], idx[i][ok], 1.0)
        p = p + tau * q * 2
        u = numpy.where(numpy.isfinite(u), u, 0)
        # two constants' roundings move the exponent by 2 e32 |u| too
        tol = p * (n + 4 * u * E32) + \
            numpy.abs(want_g) * half_step(dtype) + tiny(dtype) + \
            tau * 2.0 ** -126
    got = f64(err)
    near(got[:live], want_g, numpy.nan_to_num(tol))
    assert (got[live:] == 0).all()
    with numpy.errstate(all="ignore"):
        zmax = numpy.abs(numpy.where(numpy.isfinite(z), z, 0)).max(1)
        xs = numpy.where(numpy.isfinite(x), numpy.abs(x), 0).max(1)
    tol = tau * tau * (n + 8 * E32 * (
        2 * (zmax[:live] + xs[:live]) / tau + math.log(C) + 6))
    got = f64(loss)
    # a loss beyond fp32's range (a teacher's class at the type's lowest
    # value) is infinity in fp32
    want_l[want_l >= 2.0 ** 128 * (1 - 2.0 ** -25)] = INF
    near(got[:live], want_l, numpy.minimum(tol, 1e300))
    assert (got[live:] == 0).all()


@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 0), (8, 8), (3, 1)])
@pytest.mark.parametrize("name", sorted(TYPES))
@pytest.mark.parametrize("R,C", PROB_SIZES)
def test_eval_distill(R, C, name, pad, shift):
    dtype = TYPES[name]
    tx = rows_of(logits_case(R, C, R + C), dtype, pad, shift)
    idx, z = teacher_case(R, C, min(C, 20))
    tau = 2.0 if C % 2 else 0.7
    err = rows_of(numpy.full((R, C), 55.0), dtype, pad, shift)
    err, loss = run_distill(tx, idx, z, tau, err=err)
    check_distill(tx, f64(tx), idx, z, tau, err, loss)
    if pad or shift:
        buf = err.as_strided((R * (C + pad) + shift,), (1,), 0)
        keep = torch.ones_like(buf, dtype=torch.bool)
        keep.as_strided((R, C), (C + pad, 1), shift).fill_(False)
        assert torch.isnan(buf[keep]).all()


@pytest.mark.parametrize("R,C", [(3, 10), (5, 1001), (2, 50001),
                                 (1, 140007)])
@pytest.mark.parametrize("xpad,epad", [(0, 0), (0, 1), (3, 0), (8, 8)])
def test_eval_distill_bf16_gradient_of_fp32(R, C, xpad, epad):
    tx = rows_of(logits_case(R, C, 1), torch.float32, xpad)
    idx, z = teacher_case(R, C, 9)
    err = rows_of(numpy.zeros((R, C)), torch.bfloat16, epad)
    err, loss = run_distill(tx, idx, z, 2.0, err=err)
    check_distill(tx, f64(tx), idx, z, 2.0, err, loss)


@pytest.mark.parametrize("k", [1, 2, 63, 64, 65, 127, 128])
@pytest.mark.parametrize("C", [130, 5000, 140007])
def test_eval_distill_top(k, C):
    tx = rows_of(logits_case(3, C, k), torch.float32)
    idx, z = teacher_case(3, C, k, k)
    err, loss = run_distill(tx, idx, z, 1.0)
    check_distill(tx, f64(tx), idx, z, 1.0, err, loss)


@pytest.mark.parametrize("C", [12, 1000, 50001, 140007])
@pytest.mark.parametrize("name", sorted(TYPES))
def test_eval_distill_special_rows(C, name):
    dtype = TYPES[name]
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    R = 18
    x = logits_case(R, C, 3)
    idx, z = teacher_case(R, C, 6, 4)
    x[0] = -INF                       # nothing is allowed
    idx[1] = -1                       # no teacher
    z[2] = -INF                       # neither
    z[3, 2:] = -INF
    idx[4, 1:] = -1
    idx[5] = C - 1                    # one class six times
    idx[6, 3:] = idx[6, :3]           # three twice
    x[7, idx[7, 0]] = -INF            # forbidden to the student alone
    x[8, C // 2] = numpy.nan
    x[9, 3] = INF
    z[10, 1] = numpy.nan
    z[11, 1] = INF
    idx[12, 2] = C                    # no such class
    x[13] = low
    x[14, : C // 2] = low
    x[15, 1] = high
    z[16] = numpy.finfo(numpy.float32).min
    x[17, ::2] = -INF
    idx[17] = numpy.arange(6) * 2 + 1
    for tau in (1.0, 3.0):
        tx = rows_of(x, dtype, 1)
        err, loss = run_distill(tx, idx, z, tau)
        check_distill(tx, f64(tx), idx, z, tau, err, loss)
        assert loss[7] == INF


@pytest.mark.parametrize("C", [5001, 20001, 40000, 50001, 140007])
@pytest.mark.parametrize("name", sorted(TYPES))
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 3)])
def test_eval_distill_many_long_rows(C, name, pad, shift):
    """Rows enough not to be cut into parts, special ones among them, in
    turn."""
    R, turns, tau = 12, 7, 1.5
    x = logits_case(R, C, 13)
    idx, z = teacher_case(R, C, 100, 13)
    x[0] = -INF
    idx[1] = -1
    idx[2] = C - 1 - numpy.arange(100) % 3      # the last ones, again
    idx[3] = numpy.arange(100)                  # beside each other
    x[4, C // 2] = numpy.nan
    x[5] = -2.0 ** 15                           # far below 0, as one
    x[6] += 3e4                                 # far above
    x[7, :C // 2] = -INF
    idx[7] = C // 2 + numpy.arange(100)
    z[8, ::2] = -INF
    x[9, C - 1] = 40.0                          # at the row's end alone
    dtype = TYPES[name]
    tx = rows_of(numpy.tile(x, (turns, 1)), dtype, pad, shift)
    err = rows_of(numpy.full(tx.shape, 55.0), dtype, pad, shift)
    loss = torch.full((R * turns,), 55.0, device="cuda")
    labels = f64(tx).argmax(1)
    labels[1::2] = (labels[1::2] + 1) % C
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    live = R * turns - 2
    idx, z = numpy.tile(idx, (turns, 1)), numpy.tile(z, (turns, 1))
    ops.eval_distill(tx, cuda(idx), cuda(z), err, loss, live, tau,
                     torch.as_tensor(labels, dtype=torch.int32).cuda(), n)
    # (rows of an odd length start at other places within 16 bytes each time,
    # which is another order of their sums: equal to the bit they need not be)
    check_distill(tx, f64(tx), idx, z, tau, err, loss, live)
    rows = numpy.arange(live) % R
    wrong = (numpy.arange(live) % 2 == 1) | (rows == 0) | (rows == 4)
    assert n.item() == wrong.sum()


@pytest.mark.parametrize("batch", [0, 1, 5, 6])
@pytest.mark.parametrize("C", [100, 50001])
def test_eval_distill_padded_batch(batch, C):
    tx = rows_of(logits_case(6, C, 5), torch.bfloat16)
    idx, z = teacher_case(6, C, 4)
    x = f64(tx)
    tx[batch:] = math.nan
    err, loss = run_distill(tx, idx, z, 2.0, batch)
    check_distill(tx, x, idx, z, 2.0, err, loss, batch)


@pytest.mark.parametrize("name", sorted(TYPES))
@pytest.mark.parametrize("R,C", [(3, 100), (3, 20000), (2, 50001),
                                 (1, 131072), (300, 140007)])
def test_eval_distill_in_place(R, C, name):
    tx = rows_of(logits_case(1, C, 7).repeat(R, 0), TYPES[name])
    idx, z = teacher_case(R, C, 30)
    err, loss = run_distill(tx, idx, z, 2.0)
    over = tx.clone()
    err2, loss2 = run_distill(over, idx, z, 2.0, err=over)
    assert torch.equal(err, err2) and torch.equal(loss, loss2)


@pytest.mark.parametrize("C", [3, 1000, 50001, 140007])
@pytest.mark.parametrize("name", sorted(TYPES))
def test_eval_distill_counts_errors(C, name):
    rng = numpy.random.RandomState(1)
    R = 12
    x = logits_case(R, C, 2)
    x[3] = 1.0                        # all equal: the first class
    x[4] = -INF
    x[5, 1] = numpy.nan
    tx = rows_of(x, TYPES[name])
    labels = f64(tx).argmax(1)
    labels[::3] = rng.randint(0, C, len(labels[::3]))
    labels[3] = 0
    labels[6] = -1
    labels[7] = C + 3
    idx, z = teacher_case(R, C, 2)
    n = torch.tensor([10, 0], dtype=torch.int32).cuda()
    err, loss = torch.empty_like(tx), torch.empty(R).cuda()
    ops.eval_distill(tx, cuda(idx), cuda(z), err, loss, 11, 1.0,
                     torch.as_tensor(labels, dtype=torch.int32).cuda(), n)
    want = 10
    for i in range(11):
        if labels[i] >= 0:
            bad = i in (4, 5)
            want += bad or f64(tx)[i].argmax() != labels[i]
    assert n.tolist() == [want, 0]


def test_eval_distill_of_no_rows():
    x = torch.empty(0, 50, dtype=torch.bfloat16, device="cuda")
    n = torch.tensor([4], dtype=torch.int32, device="cuda")
    ops.eval_distill(x, torch.empty(0, 3, dtype=torch.int32, device="cuda"),
                     torch.empty(0, 3, device="cuda"), torch.empty_like(x),
                     torch.empty(0, device="cuda"), labels=torch.empty(
                         0, dtype=torch.int32, device="cuda"), n_err=n)
    assert n.item() == 4


def test_more_rows_than_a_grid_has_in_a_dimension():
    R, C = 70001, 6
    tx = rows_of(logits_case(R, C, 12), torch.float32)
    labels = numpy.arange(R) % 7 - 1
    check_logprobs(tx, labels, run_logprobs(tx, labels, 2, R - 9), R - 9)
    idx, z = teacher_case(2, C, 3)
    idx, z = idx[numpy.arange(R) % 2], z[numpy.arange(R) % 2]
    err, loss = run_distill(tx, idx, z, 2.0, R - 9)
    # (the first rows, those about each 32768, and the last ones)
    for lo, hi in ((0, 20), (32758, 32778), (65526, 65546), (R - 20, R)):
        check_distill(tx[lo:hi], f64(tx[lo:hi]), idx[lo:hi], z[lo:hi], 2.0,
                      err[lo:hi], loss[lo:hi], min(hi, R - 9) - lo)


def test_eval_distill_gradient_by_differences():
    R, C, tau = 2, 30, 1.7
    tx = rows_of(logits_case(R, C, 8), torch.float32)
    idx, z = teacher_case(R, C, 5)
    idx[1, 1] = idx[1, 0]
    err, _ = run_distill(tx, idx, z, tau)
    x, got = f64(tx), f64(err)
    rng = numpy.random.RandomState(3)
    for _ in range(5):
        d, h = rng.normal(0, 1, x.shape), 1e-5
        up = numpy_distill(x + h * d, idx, z, tau)[0].sum()
        dn = numpy_distill(x - h * d, idx, z, tau)[0].sum()
        assert abs((got * d).sum() - (up - dn) / (2 * h)) <= \
            1e-6 + 64 * E32 * numpy.abs(got * d).sum()


# ---------------------------------------------------------------------------
# streams, graphs, far rows
# ---------------------------------------------------------------------------

def _all_ops(seed, C=5000, R=40, V=40000):
    """A run of the operators on buffers of its own; returns (run, outputs,
    inputs)."""
    x, dy, w, b = norm_case(R, C, torch.bfloat16, seed)
    tx, tdy = rows_of(x, torch.bfloat16), rows_of(dy, torch.bfloat16)
    w, b = cuda(w), cuda(b)
    mean, rstd = torch.empty(R).cuda(), torch.empty(R).cuda()
    y, dx = torch.empty_like(tx), torch.empty_like(tx)
    dw, db = torch.empty(C).cuda(), torch.empty(C).cuda()
    logits = rows_of(logits_case(4, V, seed), torch.bfloat16)
    student = rows_of(logits_case(4, V, seed + 1), torch.bfloat16)
    idx = torch.empty(4, 8, dtype=torch.int32, device="cuda")
    lp, ent = torch.empty(4, 8).cuda(), torch.empty(4).cuda()
    err, loss = torch.empty_like(student), torch.empty(4).cuda()

    def run():
        ops.layer_norm_fwd(tx, y, w, b, mean, rstd)
        ops.layer_norm_bwd(tdy, tx, w, mean, rstd, dx, dw, db)
        ops.token_logprobs(logits, entropy=ent, top_idx=idx, top_logprob=lp)
        ops.eval_distill(student, idx, lp, err, loss, temperature=2.0)
    return run, [y, mean, rstd, dx, dw, db, idx, lp, ent, err, loss], \
        [tx, tdy, logits, student]


def test_row_ops_on_two_streams():
    a, b = _all_ops(1), _all_ops(2)
    for run, _, _ in (a, b):
        run()
    torch.cuda.synchronize()
    want = [[t.clone() for t in o[1]] for o in (a, b)]
    for o in (a, b):
        for t in o[1]:
            t.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for s, o in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                o[0]()
    torch.cuda.synchronize()
    for o, w in zip((a, b), want):
        for t, v in zip(o[1], w):
            assert torch.equal(t, v)


def test_row_ops_in_graphs():
    """Two captured graphs, replayed in turn with eager work between and new
    inputs each time."""
    sets = [_all_ops(3), _all_ops(4, C=96, R=3000, V=300000)]
    graphs = []
    for run, _, _ in sets:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run()
        graphs.append(g)
    for turn in range(4):
        for (run, outs, ins), g in zip(sets, graphs):
            for t in ins:
                t.copy_(t.roll(1, 0) * 0.75)
            run()
            want = [t.clone() for t in outs]
            for t in outs:
                t.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            for t, v in zip(outs, want):
                assert torch.equal(t, v)


def test_rows_beyond_32_bits():
    """Rows more than 2^31 elements apart."""
    C, R = 700, 3
    stride = (1 << 30) + 9
    buf = torch.empty(stride * (R - 1) + C, dtype=torch.bfloat16,
                      device="cuda")
    x, dy, w, b = norm_case(R, C, torch.bfloat16, 5)
    far = buf.as_strided((R, C), (stride, 1))
    far.copy_(torch.as_tensor(x).to(torch.bfloat16))
    near_x = far.contiguous()
    mean, rstd = torch.empty(R).cuda(), torch.empty(R).cuda()
    ya, yb = torch.empty_like(near_x), torch.empty_like(near_x)
    ops.layer_norm_fwd(near_x, ya, cuda(w), cuda(b), mean, rstd)
    ops.layer_norm_fwd(far, yb, cuda(w), cuda(b), None, None)
    assert torch.equal(ya, yb)
    assert [t.tolist() for t in run_logprobs(far, [1, 2, 3], 9)] == \
        [t.tolist() for t in run_logprobs(near_x, [1, 2, 3], 9)]
    idx, z = teacher_case(R, C, 4)
    ea, la = run_distill(near_x, idx, z, 2.0)
    eb, lb = run_distill(far, idx, z, 2.0, err=far)
    assert torch.equal(ea, eb) and torch.equal(la, lb)


# ---------------------------------------------------------------------------
# refusals that need tensors on the GPU
# ---------------------------------------------------------------------------

def test_row_ops_refuse_mixed_devices():
    x = torch.zeros(2, 8, device="cuda")
    with pytest.raises(RuntimeError, match="is on cpu"):
        ops.layer_norm_fwd(x, torch.zeros(2, 8), None, None, None, None)
    with pytest.raises(RuntimeError, match="is on cpu"):
        ops.layer_norm_fwd(x, x.clone(), torch.ones(8), None, None, None)
    with pytest.raises(RuntimeError, match="is on cpu"):
        ops.token_logprobs(x, entropy=torch.zeros(2))
