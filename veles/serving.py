"""Forward-only inference over trained snapshots (serving path).

The reference ecosystem shipped separate C++ engines (libVeles/libZnicz)
that loaded Veles snapshots for inference; SURVEY §2b scoped those out
of the training engine but kept the snapshot format loadable.  This
module is the MI355X-native serving analog: load a pickled Workflow,
keep only its forward chain, feed batches straight into the first
unit's input buffer (no Loader), and on a GPU replay the whole forward
pass as ONE captured hipGraph per batch — decode-style serving is
launch-bound, exactly the regime graph replay removes.

    from veles.serving import InferenceEngine
    eng = InferenceEngine("snap.4.pickle.gz")      # auto device
    probs = eng.predict(batch_ndarray)             # [n, n_classes]
    labels = probs.argmax(1)
    ans = eng.predict_top(batch_ndarray, 5)        # likeliest classes

    python -m veles.serving snap.pickle.gz --port 8080   # HTTP JSON
"""

import json
import numbers
import threading

import numpy


class InferenceEngine(object):
    """Snapshot → forward-only executor with fixed-batch graph replay."""

    #: alternatives of the passes that predict_top captures: requests of any
    #: other number take the first ones of the next larger list
    TOP_SIZES = (8, 16, 32, 64, 128)

    def __init__(self, snapshot_path, device=None, batch_size=None):
        from veles.snapshotter import SnapshotterBase
        wf = SnapshotterBase.import_(snapshot_path)
        if not getattr(wf, "forwards", None):
            raise ValueError("snapshot has no forward chain (%r)" %
                             snapshot_path)
        self.wf = wf
        self.forwards = list(wf.forwards)
        if device is None:
            from veles.backends import Device
            device = Device()
        self.device = device
        # initialize ONLY what the forward pass needs: the loader's
        # minibatch buffer (the first forward's input) plus the chain
        wf.loader.initialize(device=device)
        for f in self.forwards:
            f.forward_mode = True      # inference: dropout = identity
            if hasattr(f, "logits_only"):
                f.logits_only = False  # (a distilled head is a softmax)
            f.initialize(device=device)
        self.batch_size = batch_size or int(wf.loader.max_minibatch_size)
        self._in = wf.loader.minibatch_data
        self._graph = None
        #: alternatives -> (graph, run, outputs), which all that have the
        #: same of TOP_SIZES share
        self._top_graphs = {}
        self._lock = threading.Lock()

    # -- core ---------------------------------------------------------------
    def _forward(self):
        for f in self.forwards:
            f.run()

    def _forward_logits(self):
        """The forward pass up to the logits: those of a softmax head, or
        what another head gives."""
        head = self.forwards[-1]
        soft = hasattr(head, "logits_only")
        if soft:
            head.logits_only = True
        try:
            self._forward()
        finally:
            if soft:
                head.logits_only = False

    def _upload(self, x):
        import torch
        n = x.shape[0]
        dev = self._in.devmem
        # one pinned buffer in the DEVICE dtype: torch's cross-dtype
        # host copy converts multithreaded (~600 GB/s measured), then a
        # single H2D in the small dtype — the fp32-staging variant
        # cost ~40 ms/batch in host copies for AlexNet-sized inputs
        if getattr(self, "_pin", None) is None or \
                self._pin.dtype != dev.dtype:
            self._pin = torch.empty(dev.shape, dtype=dev.dtype,
                                    pin_memory=True)
        self._pin[:n].copy_(torch.from_numpy(
            numpy.ascontiguousarray(x, numpy.float32)))
        dev[:n].copy_(self._pin[:n], non_blocking=True)
        if n < dev.shape[0]:
            dev[n:] = 0

    def _run_device(self, x):
        import torch
        self._upload(x)
        n = x.shape[0]
        if self._graph is None:
            # warm up once eagerly, then capture the forward chain
            self._forward()
            try:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    self._forward()
                g.replay()             # capture records, doesn't run
                self._graph = g
            except Exception:
                self._graph = False    # eager fallback, permanently
                self._forward()
        elif self._graph is False:
            self._forward()
        else:
            self._graph.replay()
        out = self.forwards[-1].output
        out.touch_device()
        # pinned D2H + host fp32 view: Array.map_read's pageable
        # `.to("cpu")` measured ~39 ms/call on this ROCm build
        if getattr(self, "_out_pin", None) is None:
            self._out_pin = torch.empty(out.devmem.shape,
                                        dtype=out.devmem.dtype,
                                        pin_memory=True)
        self._out_pin.copy_(out.devmem)
        # (a copy of any head's numbers, once: those of an fp32 one would
        # else lie in the pinned buffer, which the next batch overwrites)
        return self._out_pin[:n].to(torch.float32, copy=True).numpy()

    def _run_numpy(self, x):
        self._in.map_invalidate()
        n = x.shape[0]
        self._in.mem[:n] = x
        if n < self._in.mem.shape[0]:
            self._in.mem[n:] = 0
        self._forward()
        out = self.forwards[-1].output
        out.map_read()
        return out.mem[:n].copy()

    def predict(self, x):
        """x: [n, ...sample shape] float array → [n, ...output] fp32.
        n may exceed the engine batch; inputs are chunked."""
        x = numpy.asarray(x, numpy.float32)
        if x.shape[1:] != tuple(self._in.shape[1:]):
            raise ValueError("sample shape %s != model input %s" %
                             (x.shape[1:], tuple(self._in.shape[1:])))
        outs = []
        with self._lock:
            on_gpu = self._in.devmem is not None and self._in.on_gpu
            for i in range(0, x.shape[0], self.batch_size):
                chunk = x[i:i + self.batch_size]
                outs.append(self._run_device(chunk) if on_gpu
                            else self._run_numpy(chunk))
        return numpy.concatenate(outs) if len(outs) > 1 else outs[0]

    def predict_labels(self, x):
        return self.predict(x).reshape(x.shape[0], -1).argmax(axis=1)

    # -- answers with their log probabilities --------------------------------
    def _top_device(self, x, labels, top):
        import torch
        from veles.znicz_amd import ops
        self._upload(x)
        out = self.forwards[-1].output
        size = min(s for s in self.TOP_SIZES if s >= top)
        if size not in self._top_graphs:
            batch, dev = out.devmem.shape[0], out.devmem.device
            outs = {
                "labels": torch.full((batch,), -1, dtype=torch.int32,
                                     device=dev),
                "logprob": torch.empty(batch, device=dev),
                "entropy": torch.empty(batch, device=dev),
                "top": torch.empty(batch, size, dtype=torch.int32,
                                   device=dev),
                "top_logprob": torch.empty(batch, size, device=dev)}

            def run():
                self._forward_logits()
                ops.token_logprobs(ops.as2d(out), outs["labels"],
                                   outs["logprob"], outs["entropy"],
                                   outs["top"], outs["top_logprob"])

            run()                      # warm up, then capture as predict()
            graph = None
            try:
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    run()
                graph = g
            except Exception:          # eager, permanently
                graph = None
            self._top_graphs[size] = (graph, run, outs)
        graph, run, outs = self._top_graphs.setdefault(
            top, self._top_graphs[size])
        given = numpy.full(outs["labels"].shape[0], -1, numpy.int32)
        if labels is not None:
            given[:len(labels)] = labels
        outs["labels"].copy_(torch.from_numpy(given))
        if graph is not None:
            graph.replay()
        else:
            run()
        out.touch_device()
        n = x.shape[0]
        ans = {k: v[:n].cpu().numpy() for k, v in outs.items()
               if k != "labels"}
        for k in ("top", "top_logprob"):
            ans[k] = ans[k][:, :top]   # (a list in order)
        return ans

    def _top_numpy(self, x, labels, top):
        from veles.znicz_amd.distillation import numpy_logprobs
        n = x.shape[0]
        self._in.map_invalidate()
        self._in.mem[:n] = x
        self._in.mem[n:] = 0
        self._forward_logits()
        out = self.forwards[-1].output
        out.map_read()
        lp, ent, idx, top_lp = numpy_logprobs(
            out.mem[:n].reshape(n, -1),
            numpy.full(n, -1) if labels is None else labels, top)
        return {"logprob": lp.astype(numpy.float32),
                "entropy": ent.astype(numpy.float32), "top": idx,
                "top_logprob": top_lp.astype(numpy.float32)}

    def predict_top(self, x, top=5, labels=None):
        """The likeliest classes of each sample with their log probabilities:
        {"top": int32[n, top], "top_logprob": fp32[n, top], "entropy":
        fp32[n]} and, for given ``labels``, "logprob": fp32[n] (0 for a
        label below 0, NaN for one beyond the classes).  ``top`` is 1 to 128;
        places beyond the number of classes hold -1 and minus infinity."""
        x = numpy.asarray(x, numpy.float32)
        if x.shape[1:] != tuple(self._in.shape[1:]):
            raise ValueError("sample shape %s != model input %s" %
                             (x.shape[1:], tuple(self._in.shape[1:])))
        if not isinstance(top, numbers.Integral) or not 1 <= top <= 128:
            raise ValueError("top is %r, not 1 to 128" % (top,))
        top = int(top)
        if not x.shape[0]:
            raise ValueError("no samples")
        if labels is not None:
            labels = numpy.asarray(labels).reshape(-1)
            if len(labels) != x.shape[0]:
                raise ValueError("%d labels for %d samples" %
                                 (len(labels), x.shape[0]))
            if labels.dtype.kind not in "iu":
                raise ValueError("labels are %s, not whole numbers" %
                                 labels.dtype)
            # (int32, of any type; beyond it there is no class either way)
            beyond = labels > (1 << 31) - 1
            labels = numpy.where(beyond, 0, labels).astype(numpy.int64)
            labels[beyond] = (1 << 31) - 1
            labels = numpy.maximum(labels, -1).astype(numpy.int32)
        parts = []
        with self._lock:
            on_gpu = self._in.devmem is not None and self._in.on_gpu
            run = self._top_device if on_gpu else self._top_numpy
            for i in range(0, x.shape[0], self.batch_size):
                some = None if labels is None else \
                    labels[i:i + self.batch_size]
                parts.append(run(x[i:i + self.batch_size], some, top))
        ans = {k: numpy.concatenate([p[k] for p in parts])
               for k in parts[0]}
        if labels is None:
            del ans["logprob"]
        return ans


# -- flat export for the standalone C++ engine (mzserve) --------------------
# The reference ecosystem's libVeles/libZnicz loaded snapshots in C++;
# pickles are a Python format, so the native engine consumes a flat
# manifest instead: a line-oriented text file + one raw weights blob,
# with every tensor already in the exact device layout the kernels
# take (FC forward image [N,K] bf16, conv image [K, KY*KW*C] bf16,
# fp32 biases).  veles/znicz_amd/serve/mzserve.cpp links the same
# kernel translation units the _mzk extension uses.

def export_flat(engine, outdir):
    """Export an InferenceEngine's forward chain for mzserve.

    Writes ``manifest.txt`` + ``weights.bin`` into *outdir*.  Works on
    any device (host copies are the source of truth).  Raises
    NotImplementedError for units mzserve does not implement
    (stochastic pooling, RBM/Kohonen forwards, cutter...).
    """
    import os
    import torch
    from veles.znicz_amd import all2all, conv as conv_mod, pooling, \
        normalization, dropout as dropout_mod, activation as act_mod

    os.makedirs(outdir, exist_ok=True)
    blob = bytearray()
    lines = ["mzserve 1"]

    def tensor(name, mem, dtype):
        a = numpy.ascontiguousarray(mem, numpy.float32)
        if dtype == "bf16":
            raw = torch.from_numpy(a).to(torch.bfloat16) \
                .view(torch.int16).numpy().tobytes()
        else:
            raw = a.tobytes()
        while len(blob) % 16:       # device pointers = base + offset
            blob.append(0)
        off = len(blob)
        blob.extend(raw)
        lines.append("tensor %s %s %d %d" % (name, dtype, a.size, off))
        return name

    inp = engine._in
    lines.append("batch %d" % engine.batch_size)
    lines.append("in_shape %s" % " ".join(str(s) for s in inp.shape))

    def host(arr):
        arr.map_read()
        return arr.mem

    for i, f in enumerate(engine.forwards):
        out_numel = int(numpy.prod(f.output.shape)) \
            if getattr(f, "output", None) else 0
        if isinstance(f, dropout_mod.DropoutForward):
            continue                     # identity at inference
        elif isinstance(f, all2all.All2AllSoftmax):
            w = host(f.weights)
            if f.weights_transposed:     # host [K,N] -> forward [N,K]
                w = w.T
            wn = tensor("w%d" % i, w, "bf16")
            bn = tensor("b%d" % i, host(f.bias), "f32") \
                if f.include_bias else "-"
            M, N = f.output.shape[0], f.output.shape[1]
            K = w.shape[1]
            lines.append("op fc %s %s 0 %d %d %d f32" % (wn, bn, M, N, K))
            lines.append("op softmax %d %d" % (M, N))
        elif isinstance(f, all2all.All2All):
            w = host(f.weights)
            if f.weights_transposed:
                w = w.T
            wn = tensor("w%d" % i, w, "bf16")
            bn = tensor("b%d" % i, host(f.bias), "f32") \
                if f.include_bias else "-"
            M = f.output.shape[0]
            N = int(numpy.prod(f.output.shape[1:]))
            K = w.shape[1]
            lines.append("op fc %s %s %d %d %d %d bf16" %
                         (wn, bn, f.ACTIVATION, M, N, K))
        elif isinstance(f, conv_mod.Conv):
            d = f.conv_desc()
            if d[3] % 4 != 0:
                raise NotImplementedError(
                    "mzserve conv needs C%%4==0 (got C=%d); train with "
                    "padded channels as the GPU path does" % d[3])
            w = host(f.weights).reshape(f.weights.shape[0], -1)
            wn = tensor("w%d" % i, w, "bf16")
            bn = tensor("b%d" % i, host(f.bias), "f32") \
                if f.include_bias else "-"
            lines.append("op conv %s %s %d %s %d" %
                         (wn, bn, f.ACTIVATION,
                          " ".join(str(x) for x in d), out_numel))
        elif isinstance(f, pooling.Pooling):
            from veles.znicz_amd.pooling import POOL_STOCHASTIC
            if f.MODE == POOL_STOCHASTIC:
                raise NotImplementedError("mzserve: stochastic pooling")
            lines.append("op pool %d %s %d" %
                         (f.MODE,
                          " ".join(str(x) for x in f.pool_desc()),
                          out_numel))
        elif isinstance(f, normalization.LRNormalizerForward):
            C = f.input.shape[-1]
            rows = int(numpy.prod(f.input.shape)) // C
            lines.append("op lrn %d %d %r %r %r %d %d" %
                         (C, rows, f.alpha, f.beta, f.k, f.n, out_numel))
        elif isinstance(f, normalization.LayerNormForward):
            C = f.input.shape[-1]
            rows = int(numpy.prod(f.input.shape)) // C
            wn = tensor("w%d" % i, host(f.weights), "f32")
            bn = tensor("b%d" % i, host(f.bias), "f32") \
                if f.include_bias else "-"
            lines.append("op layernorm %s %s %d %d %r %d" %
                         (wn, bn, C, rows, float(f.eps), out_numel))
        elif isinstance(f, act_mod.ActivationForward):
            lines.append("op act %d" % f.ACTIVATION)
        else:
            raise NotImplementedError(
                "mzserve: no export for unit %s" % type(f).__name__)
    lines.append("end")
    with open(os.path.join(outdir, "weights.bin"), "wb") as fo:
        fo.write(bytes(blob))
    with open(os.path.join(outdir, "manifest.txt"), "w") as fo:
        fo.write("\n".join(lines) + "\n")
    return outdir


# -- minimal HTTP JSON front end (same dependency-light style as
# web_status.py; fastapi/uvicorn exist in the image but add nothing
# here) ----------------------------------------------------------------------

def serve(engine, port=8080):
    from http.server import BaseHTTPRequestHandler, HTTPServer

    def finite(v):
        """JSON has no infinities: they become null."""
        if v.dtype.kind != "f":
            return v.tolist()
        return numpy.where(numpy.isfinite(v), v.astype(object),
                           None).tolist()

    class Handler(BaseHTTPRequestHandler):
        def do_POST(self):
            try:
                n = int(self.headers.get("Content-Length", 0))
                req = json.loads(self.rfile.read(n))
                x = numpy.asarray(req["inputs"], numpy.float32)
                want_labels = req.get("labels_only", False)
                if want_labels:
                    resp = {"labels":
                            engine.predict_labels(x).tolist()}
                elif "top" in req:
                    resp = {k: finite(v) for k, v in engine.predict_top(
                        x, req["top"], req.get("labels")).items()}
                else:
                    resp = {"outputs": engine.predict(x).tolist()}
                body = json.dumps(resp).encode()
                self.send_response(200)
            except Exception as e:
                body = json.dumps({"error": repr(e)}).encode()
                self.send_response(400)
            self.send_header("Content-Type", "application/json")
            self.send_header("Content-Length", str(len(body)))
            self.end_headers()
            self.wfile.write(body)

        def log_message(self, *a):
            pass

    srv = HTTPServer(("0.0.0.0", port), Handler)
    srv.serve_forever()


def main(argv=None):
    import argparse
    p = argparse.ArgumentParser(
        prog="veles.serving",
        description="serve a trained Veles snapshot over HTTP JSON")
    p.add_argument("snapshot")
    p.add_argument("--port", type=int, default=8080)
    p.add_argument("--batch", type=int, default=None)
    p.add_argument("--export", default=None, metavar="DIR",
                   help="write a flat manifest+weights export for the "
                        "standalone C++ engine (mzserve) and exit")
    args = p.parse_args(argv)
    eng = InferenceEngine(args.snapshot, batch_size=args.batch)
    if args.export:
        export_flat(eng, args.export)
        print("exported %s -> %s (run: veles/znicz_amd/serve/mzserve %s)"
              % (args.snapshot, args.export, args.export))
        return
    print("serving %s on :%d (batch %d)" % (args.snapshot, args.port,
                                            eng.batch_size))
    serve(eng, args.port)


if __name__ == "__main__":
    main()
