"""Local response normalization (cross-channel).

Parity target: reference ``znicz/normalization.py``
(``LRNormalizerForward``, ``LRNormalizerBackward``): AlexNet-style
y = x·(k + α·Σ_{j∈window} x_j²)^(−β), window n across adjacent channels;
closed-form backward.  Forward saves the denominators for backward.
"""

import numpy

from veles.memory import Array
from veles.znicz_amd.nn_units import Forward, GradientDescentBase


class LRNormalizerForward(Forward):
    MAPPING = "norm"

    def __init__(self, workflow, **kwargs):
        super(LRNormalizerForward, self).__init__(workflow, **kwargs)
        self.alpha = kwargs.get("alpha", 0.0001)
        self.beta = kwargs.get("beta", 0.75)
        self.k = kwargs.get("k", 2)
        self.n = kwargs.get("n", 5)
        self.denominators = Array()

    @property
    def has_weights(self):
        return False

    def initialize(self, device=None, **kwargs):
        super(LRNormalizerForward, self).initialize(device=device,
                                                    **kwargs)
        if self.input is None or not self.input:
            return False
        if not self.output or self.output.shape != self.input.shape:
            self.output.reset(numpy.zeros(self.input.shape,
                                          numpy.float32))
            self.output.device_dtype = "bf16"
        if not self.denominators or \
                self.denominators.shape != self.input.shape:
            self.denominators.reset(numpy.zeros(self.input.shape,
                                                numpy.float32))
        self.init_array(self.output)
        self.init_array(self.denominators, device_dtype="f32")

    def _win(self, c, C):
        half = self.n // 2
        return max(0, c - half), min(C - 1, c + half)

    def numpy_run(self):
        self.input.map_read()
        self.output.map_invalidate()
        self.denominators.map_invalidate()
        x = self.input.mem.reshape(-1, self.input.shape[-1])
        C = x.shape[1]
        d = numpy.empty_like(x)
        sq = x * x
        for c in range(C):
            j0, j1 = self._win(c, C)
            d[:, c] = self.k + self.alpha * sq[:, j0:j1 + 1].sum(axis=1)
        y = x * d ** (-self.beta)
        self.denominators.mem[...] = d.reshape(self.input.shape)
        self.output.mem[...] = y.reshape(self.input.shape)

    def hip_run(self):
        from veles.znicz_amd import ops
        # no denom store: the backward kernel recomputes it from its
        # own x halo — saves the fp32 round-trip (memory-wait bound)
        ops.lrn_fwd(self.input.devmem, self.output.devmem, None,
                    self.alpha, self.beta, self.k, self.n)
        self.output.touch_device()


class LRNormalizerBackward(GradientDescentBase):
    MAPPING = "norm"
    BACKWARD = True
    LINK_FROM_FORWARD = ("denominators",)

    def __init__(self, workflow, **kwargs):
        super(LRNormalizerBackward, self).__init__(workflow, **kwargs)
        self.include_bias = False
        self.alpha = kwargs.get("alpha", 0.0001)
        self.beta = kwargs.get("beta", 0.75)
        self.k = kwargs.get("k", 2)
        self.n = kwargs.get("n", 5)
        self.denominators = None    # linked
        self.forward_unit = None

    def initialize(self, device=None, **kwargs):
        if self.err_output is None or not self.err_output:
            return False
        if self.input is None or not self.input:
            return False
        if not self.err_input or \
                self.err_input.shape != self.input.shape:
            self.err_input.reset(numpy.zeros(self.input.shape,
                                             numpy.float32))
            self.err_input.device_dtype = "bf16"
        super(LRNormalizerBackward, self).initialize(device=device,
                                                     **kwargs)
        self.init_array(self.err_input)
        fwd = self.forward_unit
        if fwd is not None:
            self.alpha, self.beta = fwd.alpha, fwd.beta
            self.k, self.n = fwd.k, fwd.n

    def numpy_run(self):
        self.err_output.map_read()
        self.input.map_read()
        self.denominators.map_read()
        self.err_input.map_invalidate()
        C = self.input.shape[-1]
        x = self.input.mem.reshape(-1, C)
        dy = self.err_output.mem.reshape(-1, C)
        d = self.denominators.mem.reshape(-1, C)
        half = self.n // 2
        t = dy * x * d ** (-self.beta - 1.0)
        out = dy * d ** (-self.beta)
        for c in range(C):
            j0, j1 = max(0, c - half), min(C - 1, c + half)
            out[:, c] -= 2.0 * self.alpha * self.beta * x[:, c] * \
                t[:, j0:j1 + 1].sum(axis=1)
        self.err_input.mem[...] = out.reshape(self.input.shape)

    def hip_run(self):
        from veles.znicz_amd import ops
        ops.lrn_bwd(self.err_output.devmem, self.input.devmem, None,
                    None, self.err_input.devmem,
                    self.alpha, self.beta, self.k, self.n)
        self.err_input.touch_device()


class LayerNormForward(Forward):
    """Normalization over the last dimension (a sample's features, or the
    channels at each place of a map) by its own mean and deviation:

        y = (x − mean) / sqrt(var + eps) · weights + bias

    ``weights`` (the gain, 1 at the start) and ``bias`` have one value for
    each feature.  In training the row statistics are kept for the backward
    unit; in ``forward_mode`` they are not written.  No reference
    counterpart."""

    MAPPING = "layer_norm"

    def __init__(self, workflow, **kwargs):
        kwargs.setdefault("weights_filling", "constant")
        kwargs.setdefault("weights_stddev", 1.0)
        kwargs.setdefault("bias_stddev", 0.0)
        super(LayerNormForward, self).__init__(workflow, **kwargs)
        self.eps = kwargs.get("eps", 1e-5)
        if not 0 <= self.eps < 1e30:
            raise ValueError("layer_norm: eps is %r" % (self.eps,))
        self.mean = Array()
        self.rstd = Array()

    def initialize(self, device=None, **kwargs):
        super(LayerNormForward, self).initialize(device=device, **kwargs)
        if self.input is None or not self.input:
            return False
        if len(self.input.shape) < 2:
            raise ValueError("layer_norm: input shape %s has no features" %
                             (self.input.shape,))
        C = self.input.shape[-1]
        rows = self.input.size // C
        if not self.weights:
            self.weights.mem = numpy.zeros(C, numpy.float32)
            self.fill_array(self.weights_filling, self.weights,
                            self.weights_stddev)
        if self.include_bias and not self.bias:
            self.bias.mem = numpy.zeros(C, numpy.float32)
            self.fill_array(self.bias_filling, self.bias, self.bias_stddev)
        if not self.output or self.output.shape != self.input.shape:
            self.output.reset(numpy.zeros(self.input.shape,
                                          numpy.float32))
            self.output.device_dtype = "bf16"
        for arr in (self.mean, self.rstd):
            if not arr or arr.shape != (rows,):
                arr.reset(numpy.zeros(rows, numpy.float32))
            self.init_array(arr, device_dtype="f32")
        self.init_array(self.weights, device_dtype="f32")
        if self.include_bias:
            self.init_array(self.bias, device_dtype="f32")
        self.init_array(self.output)

    def numpy_run(self):
        self.input.map_read()
        self.output.map_invalidate()
        x = self.input.mem.reshape(-1, self.input.shape[-1])
        mean = x.mean(axis=1, keepdims=True)
        xc = x - mean
        rstd = 1.0 / numpy.sqrt((xc * xc).mean(axis=1, keepdims=True) +
                                self.eps)
        y = xc * rstd * self.weights.mem
        if self.include_bias:
            y = y + self.bias.mem
        if not self.forward_mode:
            self.mean.map_invalidate()
            self.rstd.map_invalidate()
            self.mean.mem[...] = mean[:, 0]
            self.rstd.mem[...] = rstd[:, 0]
        self.output.mem[...] = y.reshape(self.output.shape)

    def hip_run(self):
        from veles.znicz_amd import ops
        train = not self.forward_mode
        ops.layer_norm_fwd(
            self.input.devmem, self.output.devmem, self.weights.devmem,
            self.bias.devmem if self.include_bias else None,
            self.mean.devmem if train else None,
            self.rstd.devmem if train else None, self.eps)
        self.output.touch_device()
        if train:
            self.mean.touch_device()
            self.rstd.touch_device()


class LayerNormBackward(GradientDescentBase):
    """err_input and the gradients of the gain and the bias in one pass over
    err_output and input; the update is that of the fully-connected layers
    (batch mean, decay, momentum, the reducer's buckets)."""

    MAPPING = "layer_norm"
    BACKWARD = True
    LINK_FROM_FORWARD = ("mean", "rstd")

    def __init__(self, workflow, **kwargs):
        super(LayerNormBackward, self).__init__(workflow, **kwargs)
        self.mean = None            # linked
        self.rstd = None
        self.forward_unit = None

    def initialize(self, device=None, **kwargs):
        if self.err_output is None or not self.err_output:
            return False
        if self.input is None or not self.input:
            return False
        if self.need_err_input and (
                not self.err_input or
                self.err_input.shape != self.input.shape):
            self.err_input.reset(numpy.zeros(self.input.shape,
                                             numpy.float32))
            self.err_input.device_dtype = "bf16"
        super(LayerNormBackward, self).initialize(device=device, **kwargs)
        if self.need_err_input:
            self.init_array(self.err_input)

    def numpy_run(self):
        for arr in (self.err_output, self.input, self.mean, self.rstd):
            arr.map_read()
        C = self.input.shape[-1]
        x = self.input.mem.reshape(-1, C)
        dy = self.err_output.mem.reshape(-1, C)
        rstd = self.rstd.mem[:, None]
        xh = (x - self.mean.mem[:, None]) * rstd
        gw, gb = (dy * xh).sum(axis=0), dy.sum(axis=0)
        if self.need_err_input:
            self.err_input.map_invalidate()
            g = dy * self.weights.mem
            dx = rstd * (g - g.mean(axis=1, keepdims=True) -
                         xh * (g * xh).mean(axis=1, keepdims=True))
            self.err_input.mem[...] = dx.reshape(self.err_input.shape)
        self.numpy_update_weights(gw)
        self.numpy_update_bias(gb)

    def hip_run(self):
        from veles.znicz_amd import ops
        has_bias = self.include_bias and self.bias is not None and \
            bool(self.bias)
        shape = self.input.devmem.shape
        ops.layer_norm_bwd(
            self.err_output.devmem.view(shape), self.input.devmem,
            self.weights.devmem, self.mean.devmem, self.rstd.devmem,
            self.err_input.devmem if self.need_err_input else None,
            self.gradient_weights.devmem,
            self.gradient_bias.devmem if has_bias else None,
            accumulate=self.accumulate_gradient)
        if self.need_err_input:
            self.err_input.touch_device()
        self.gradient_weights.touch_device()
        if has_bias:
            self.gradient_bias.touch_device()
        self._hip_apply(self.err_output.shape[0])
