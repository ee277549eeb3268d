"""Cases, plain forms and 64-bit results of three operator families:

* ``layer_norm_fwd`` / ``layer_norm_bwd``: normalisation of rows by their own
  mean and deviation, with a gain and a shift for each column, and its
  backward pass with the gain's and the shift's gradients;
* ``token_logprobs``: for each row of logits the log probability of a given
  class, the distribution's entropy, and the classes of highest probability;
* ``eval_distill``: the loss of a student's logits against a teacher's top
  logits, and its gradient.

``run`` computes them by elementary torch operations, or, where ``own`` is
true, by the calls that a user makes of ``veles.znicz_amd.ops``.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16,
          "f32": torch.float32}
EPS = 1e-5


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one sample through a served network: a row as wide as a
        # fully-connected layer of the image classifiers; latency counts
        {"name": "norm_one_row", "op": "norm_fwd", "rows": 1, "cols": 4096,
         "pad": 0, "dtype": "bf16", "stats": False, "affine": True},
        # channels of the first convolution's map (55 x 55 x 96) over a
        # minibatch of 64, in training
        {"name": "norm_channels", "op": "norm_fwd", "rows": 193600,
         "cols": 96, "pad": 0, "dtype": "bf16", "stats": True,
         "affine": True},
        # a long batch of wide rows, in training
        {"name": "norm_wide", "op": "norm_fwd", "rows": 16384, "cols": 4096,
         "pad": 0, "dtype": "bf16", "stats": True, "affine": True},
        # the same layer's backward pass, with the parameters' gradients
        {"name": "norm_wide_bwd", "op": "norm_bwd", "rows": 16384,
         "cols": 4096, "pad": 0, "dtype": "bf16", "stats": True,
         "affine": True},
        # an odd width and an odd number of rows, in 32 bits, cut out of
        # wider rows
        {"name": "norm_odd_bwd", "op": "norm_bwd", "rows": 2731,
         "cols": 1021, "pad": 3, "dtype": "f32", "stats": True,
         "affine": True},
        # the answer of one position over a large vocabulary, with its top
        # alternatives, between two steps of a generator; latency counts
        {"name": "logprobs_one_row", "op": "logprobs", "rows": 1,
         "live": 1, "cols": 131072, "pad": 0, "dtype": "bf16", "top": 5,
         "masked": 0.0},
        # answers of the image classifiers: a minibatch of 256, 1000 classes
        {"name": "logprobs_classes", "op": "logprobs", "rows": 256,
         "live": 250, "cols": 1000, "pad": 0, "dtype": "f32", "top": 5,
         "masked": 0.0},
        # scoring of given texts, with an odd vocabulary, a part of it
        # forbidden
        {"name": "logprobs_scoring", "op": "logprobs", "rows": 4096,
         "live": 4001, "cols": 50001, "pad": 0, "dtype": "bf16", "top": 20,
         "masked": 0.3},
        # a teacher's answers, written down for distillation
        {"name": "logprobs_teacher", "op": "logprobs", "rows": 2048,
         "live": 2048, "cols": 131072, "pad": 0, "dtype": "bf16",
         "top": 64, "masked": 0.0},
        # a small classifier that learns from a large one
        {"name": "distill_classes", "op": "distill", "rows": 256,
         "live": 256, "cols": 1000, "pad": 0, "dtype": "bf16", "top": 16,
         "masked": 0.0, "temperature": 2.0},
        # a training step in 32 bits, an odd vocabulary in padded rows, the
        # minibatch not full
        {"name": "distill_odd", "op": "distill", "rows": 1023,
         "live": 1000, "cols": 50001, "pad": 47, "dtype": "f32", "top": 20,
         "masked": 0.1, "temperature": 1.0},
        # a training step over a large vocabulary
        {"name": "distill_large", "op": "distill", "rows": 2048,
         "live": 2048, "cols": 131072, "pad": 0, "dtype": "bf16",
         "top": 64, "masked": 0.0, "temperature": 2.0},
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, v))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "logprobs", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op.startswith("norm"):
        cols = _between(rng, 8, 30000)
        most = 40000000 if dtype == "f32" else 60000000
        rows = _between(rng, 1, max(1, min(200000, most // cols)))
        return {"op": op, "rows": rows, "cols": cols,
                "pad": rng.choice([0, 0, 1, 8, 40]), "dtype": dtype,
                "stats": op == "norm_bwd" or rng.random() < 0.5,
                "affine": rng.random() < 0.9}
    cols = _between(rng, 10, 150000)
    most = 120000000 if dtype == "f32" else 240000000
    rows = _between(rng, 1, max(1, min(8192, most // cols)))
    case = {"op": op, "rows": rows,
            "live": rows if rng.random() < 0.6 else rng.randint(0, rows),
            "cols": cols, "pad": rng.choice([0, 0, 1, 8, 47]),
            "dtype": dtype,
            "top": min(cols, rng.choice([1, 5, 20, 33, 64, 100, 128])),
            "masked": rng.choice([0.0, 0.0, 0.1, 0.6])}
    if op == "distill":
        case["temperature"] = rng.choice([1.0, 1.0, 2.0, 4.0, 0.7])
    return case


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _rows(case, g, scale, shift=0.0):
    """[rows, cols] normal values of the case's type, in rows of
    cols + pad."""
    buf = torch.empty(case["rows"], case["cols"] + case["pad"],
                      dtype=DTYPES[case["dtype"]], device="cuda")
    buf.normal_(shift, scale, generator=g)
    return buf[:, :case["cols"]]


def _like(case):
    buf = torch.empty(case["rows"], case["cols"] + case["pad"],
                      dtype=DTYPES[case["dtype"]], device="cuda")
    return buf[:, :case["cols"]]


def _logits(case, g):
    """Logits as a trained model gives them: a few classes stand out of each
    row, a share of the classes is forbidden (minus infinity), and now and
    then all of a row is."""
    rows, cols = case["rows"], case["cols"]
    x = _rows(case, g, 2.0)
    few = min(cols, 8)
    at = torch.randint(cols, (rows, few), generator=g, device="cuda")
    up = torch.rand(rows, few, generator=g, device="cuda") * 9 + 3
    x.scatter_(1, at, up.to(x.dtype))
    if case["masked"]:
        off = torch.rand(cols, generator=g, device="cuda") < case["masked"]
        x.masked_fill_(off[None, :], -math.inf)
        if rows > 2:
            x[rows // 3] = -math.inf
    return x


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, cols = case["rows"], case["cols"]
    dev = {"device": "cuda"}
    s = {"case": case, "op": case["op"]}
    if case["op"].startswith("norm"):
        s["x"] = _rows(case, g, 1.5, 0.3)
        s["weights"] = s["bias"] = None
        if case["affine"]:
            s["weights"] = torch.randn(cols, generator=g, **dev) * 0.2 + 1
            s["bias"] = torch.randn(cols, generator=g, **dev) * 0.1
        s["out"] = _like(case)
        s["mean"] = s["rstd"] = None
        if case["stats"]:
            s["mean"] = torch.empty(rows, **dev)
            s["rstd"] = torch.empty(rows, **dev)
        if case["op"] == "norm_bwd":
            s["err"] = _rows(case, g, 0.02)
            # what the forward pass has left behind
            for i in range(0, rows, 4096):
                x = s["x"][i:i + 4096].double()
                m = x.mean(1)
                v = (x - m[:, None]).square().mean(1)
                s["mean"][i:i + 4096] = m.float()
                s["rstd"][i:i + 4096] = (v + EPS).rsqrt().float()
            s["grad_w"] = torch.empty(cols, **dev)
            s["grad_b"] = torch.empty(cols, **dev)
        return s
    s["x"] = _logits(case, g)
    k = case["top"]
    if case["op"] == "logprobs":
        labels = torch.randint(cols, (rows,), generator=g, **dev)
        # a sample without a label now and then
        labels[torch.rand(rows, generator=g, **dev) < 0.05] = -1
        s["labels"] = labels.int()
        s["logprob"] = torch.empty(rows, **dev)
        s["entropy"] = torch.empty(rows, **dev)
        s["top_idx"] = torch.empty(rows, k, dtype=torch.int32, **dev)
        s["top_logprob"] = torch.empty(rows, k, **dev)
    else:
        # a teacher names k different classes, the likeliest first; the last
        # places of some rows are empty
        first = torch.randint(cols, (rows, 1), generator=g, **dev)
        if k <= cols // 2:
            gap = torch.randint(1, max(2, cols // k), (rows, k),
                                generator=g, **dev)
        else:
            gap = torch.ones(rows, k, dtype=torch.int64, **dev)
        idx = (first + gap.cumsum(1)) % cols
        z = torch.randn(rows, k, generator=g, **dev) * 2.5
        z = z.sort(1, descending=True).values
        kept = torch.randint(1, k + 1, (rows, 1), generator=g, **dev)
        some = torch.rand(rows, 1, generator=g, **dev) < 0.2
        gone = (torch.arange(k, **dev)[None, :] >= kept) & some
        # it has no answers outside the classes that are allowed
        gone |= s["x"].gather(1, idx) == -math.inf
        s["idx"] = idx.masked_fill(gone, -1).int()
        s["z"] = z.masked_fill(gone, -math.inf)
        s["err"] = _like(case)
        s["loss"] = torch.empty(rows, **dev)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    return _own_run(s) if own else _plain_run(s)


def _own_run(s):
    from veles.znicz_amd import ops
    if s["op"] == "norm_fwd":
        ops.layer_norm_fwd(s["x"], s["out"], s["weights"], s["bias"],
                           s["mean"], s["rstd"], EPS)
        return [s["out"]] if s["mean"] is None else \
            [s["out"], s["mean"], s["rstd"]]
    if s["op"] == "norm_bwd":
        ops.layer_norm_bwd(s["err"], s["x"], s["weights"], s["mean"],
                           s["rstd"], s["out"], s["grad_w"], s["grad_b"])
        return [s["out"], s["grad_w"], s["grad_b"]]
    if s["op"] == "logprobs":
        ops.token_logprobs(s["x"], s["labels"], s["logprob"], s["entropy"],
                           s["top_idx"], s["top_logprob"],
                           s["case"]["live"])
        return [s["logprob"], s["entropy"], s["top_idx"], s["top_logprob"]]
    ops.eval_distill(s["x"], s["idx"], s["z"], s["err"], s["loss"],
                     s["case"]["live"], s["case"]["temperature"])
    return [s["err"], s["loss"]]


def _plain_run(s):
    if s["op"] == "norm_fwd":
        return _plain_norm_fwd(s)
    if s["op"] == "norm_bwd":
        return _plain_norm_bwd(s)
    if s["op"] == "logprobs":
        return _plain_logprobs(s)
    return _plain_distill(s)


def _plain_norm_fwd(s):
    x = s["x"].float()
    mean = x.mean(1)
    xc = x - mean[:, None]
    rstd = 1 / (xc.square().mean(1) + EPS).sqrt()
    y = xc * rstd[:, None]
    if s["weights"] is not None:
        y = y * s["weights"] + s["bias"]
    y = y.to(s["x"].dtype)
    return [y] if s["mean"] is None else [y, mean, rstd]


def _plain_norm_bwd(s):
    dy = s["err"].float()
    rstd = s["rstd"][:, None]
    xh = (s["x"].float() - s["mean"][:, None]) * rstd
    gy = dy if s["weights"] is None else dy * s["weights"]
    dx = rstd * (gy - gy.mean(1, keepdim=True) -
                 xh * (gy * xh).mean(1, keepdim=True))
    return [dx.to(s["x"].dtype), (dy * xh).sum(0), dy.sum(0)]


def _plain_logprobs(s):
    case = s["case"]
    rows, cols, k, live = (case[n] for n in ("rows", "cols", "top", "live"))
    logprob = torch.zeros_like(s["logprob"])
    entropy = torch.zeros_like(s["entropy"])
    top_idx = torch.full_like(s["top_idx"], -1)
    top_logprob = torch.zeros_like(s["top_logprob"])
    out = [logprob, entropy, top_idx, top_logprob]
    if not live:
        return out
    x = s["x"][:live].float()
    high = x.amax(1, keepdim=True)
    none = (high == -math.inf)[:, 0]       # nothing is allowed there
    t = x - high.masked_fill(none[:, None], 0.0)
    e = t.exp()
    total = e.sum(1)
    ln = total.log()
    expected = (e * t.masked_fill(t == -math.inf, 0.0)).sum(1) / total
    entropy[:live] = (ln - expected).masked_fill(none, 0.0)
    labels = s["labels"][:live].long()
    given = t.gather(1, labels.clamp(min=0)[:, None])[:, 0] - ln
    given = given.masked_fill(none, -math.inf)
    logprob[:live] = given.masked_fill(labels < 0, 0.0)
    # the order of the values, and of the classes where values are equal, in
    # one whole number (adding zero makes one of the two zeros)
    bits = (x + 0.0).view(torch.int32)
    bits = torch.where(bits < 0, bits ^ 0x7fffffff, bits).long()
    back = torch.arange(cols - 1, -1, -1, device=x.device)
    keys = (bits * 4294967296 + back).topk(k, dim=1).values
    at = cols - 1 - (keys & 0xffffffff)
    lp = t.gather(1, at) - ln[:, None]
    off = lp.masked_fill(none[:, None], -math.inf) == -math.inf
    top_idx[:live] = at.masked_fill(off, -1).int()
    top_logprob[:live] = lp.masked_fill(off, -math.inf)
    return out


def _plain_distill(s):
    case = s["case"]
    live, tau = case["live"], case["temperature"]
    err, loss = torch.zeros_like(s["err"]), torch.zeros_like(s["loss"])
    if not live:
        return [err, loss]
    x = s["x"][:live].float() / tau
    high = x.amax(1, keepdim=True)
    high = high.masked_fill(high == -math.inf, 0.0)
    e = (x - high).exp()
    total = e.sum(1, keepdim=True)
    idx = s["idx"][:live].long()
    named = idx >= 0
    z = (s["z"][:live] / tau).masked_fill(~named, -math.inf)
    zh = z.amax(1, keepdim=True)
    some = (zh > -math.inf) & (total > 0)  # a row that teaches something
    w = (z - zh.masked_fill(~some, 0.0)).exp()
    wsum = w.sum(1, keepdim=True)
    q = w / wsum
    lnq = z - zh.masked_fill(~some, 0.0) - wsum.log()
    at = idx.clamp(min=0)
    lnp = x.gather(1, at) - high - total.log()
    part = torch.where(q > 0, q * (lnq - lnp), torch.zeros_like(q))
    loss[:live] = torch.where(some[:, 0], tau * tau * part.sum(1),
                              loss[:live])
    q = q.masked_fill(~(some & named), 0.0)
    d = (e / total).scatter_add_(1, at, -q) * tau
    err[:live] = d.masked_fill(~some, 0.0).to(err.dtype)
    return [err, loss]


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    rows, cols = case["rows"], case["cols"]
    size = 4 if case["dtype"] == "f32" else 2
    n = rows * cols
    if case["op"] == "norm_fwd":
        return {"bytes": 2 * n * size + (8 * cols if case["affine"] else 0) +
                (8 * rows if case["stats"] else 0), "flops": 7 * n}
    if case["op"] == "norm_bwd":
        return {"bytes": 3 * n * size + 8 * rows +
                (12 if case["affine"] else 8) * cols, "flops": 14 * n}
    live, k = case["live"], case["top"]
    m = live * cols
    if case["op"] == "logprobs":
        return {"bytes": m * size + rows * (8 + 8 * k) + 4 * live,
                "flops": 7 * m}
    return {"bytes": (m + n) * size + 8 * live * k + 4 * rows,
            "flops": 9 * m}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    rows, cols = case["rows"], case["cols"]
    f8 = {"dtype": torch.float64, "device": "cuda"}
    part = max(1, (1 << 25) // cols)       # rows at a time

    if case["op"] == "norm_fwd":
        y = torch.empty(rows, cols, **f8)
        mean, rstd = torch.empty(rows, **f8), torch.empty(rows, **f8)
        for i in range(0, rows, part):
            x = s["x"][i:i + part].double()
            var, mu = torch.var_mean(x, dim=1, correction=0)
            r = torch.rsqrt(var + EPS)
            h = (x - mu.unsqueeze(1)) * r.unsqueeze(1)
            if case["affine"]:
                h = torch.addcmul(s["bias"].double(), h,
                                  s["weights"].double())
            y[i:i + part], mean[i:i + part], rstd[i:i + part] = h, mu, r
        return [y, mean, rstd] if case["stats"] else [y]

    if case["op"] == "norm_bwd":
        dx = torch.empty(rows, cols, **f8)
        gw, gb = torch.zeros(cols, **f8), torch.zeros(cols, **f8)
        w = s["weights"].double() if case["affine"] else \
            torch.ones(cols, **f8)
        for i in range(0, rows, part):
            dy = s["err"][i:i + part].double()
            r = s["rstd"][i:i + part].double().unsqueeze(1)
            h = (s["x"][i:i + part].double() -
                 s["mean"][i:i + part].double().unsqueeze(1)) * r
            gw += torch.linalg.vecdot(dy, h, dim=0)
            gb += dy.sum(dim=0)
            a = (dy @ w).unsqueeze(1) / cols
            b = ((dy * h) @ w).unsqueeze(1) / cols
            dx[i:i + part] = (dy * w - a - b * h) * r
        return [dx, gw, gb]

    live, k = case["live"], case["top"]
    if case["op"] == "logprobs":
        logprob, entropy = torch.zeros(rows, **f8), torch.zeros(rows, **f8)
        top = torch.zeros(rows, k, **f8)
        for i in range(0, live, part):
            j = min(live, i + part)
            x = s["x"][i:j].double()
            lse = torch.logsumexp(x, dim=1, keepdim=True)
            lp = torch.where(lse == -math.inf, -math.inf, x - lse)
            p = lp.exp()
            entropy[i:j] = -torch.special.xlogy(p, p).sum(dim=1)
            label = s["labels"][i:j].long()
            had = label >= 0
            at = torch.nonzero(had)[:, 0]
            logprob[i + at] = lp[at, label[had]]
            top[i:j] = torch.topk(lp, k, dim=1).values
        return [logprob, entropy, None, top]

    tau = case["temperature"]
    err, loss = torch.zeros(rows, cols, **f8), torch.zeros(rows, **f8)
    for i in range(0, live, part):
        j = min(live, i + part)
        x = s["x"][i:j].double() / tau
        lse = torch.logsumexp(x, dim=1, keepdim=True)
        idx, z = s["idx"][i:j].long(), s["z"][i:j].double() / tau
        at = idx.clamp_min(0)
        # the teacher's distribution over all classes
        full = torch.full_like(x, -math.inf)
        full.scatter_reduce_(
            1, at, torch.where(idx < 0, -math.inf, z), "amax")
        lnq = full - torch.logsumexp(full, dim=1, keepdim=True)
        q = lnq.exp()
        d = torch.where(q > 0, q * (lnq - (x - lse)), 0.0).sum(dim=1)
        good = (torch.isfinite(full).any(dim=1) &
                torch.isfinite(lse[:, 0]))
        loss[i:j] = torch.where(good, d * tau ** 2, 0.0)
        g = ((x - lse).exp() - q) * tau
        err[i:j] = torch.where(good.unsqueeze(1), g, 0.0)
    return [err, loss]
