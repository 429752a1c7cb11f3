"""Dense weights in 4 bits (this package's extension; the layout is described in include/xsmi355.h)."""
import numpy as np

from ..backend import kernels as K, to_device
from ..core.base import is_device


class Weight4Bit:
    """The weight of a dense layer as whole numbers in -8 .. 7 with a float16 scale for each ``group`` inputs (32, 64 or 128) of
    an output, in device memory: ``codes`` uint8 and ``scales`` float16 arrays of the shapes that
    ``backend.kernels.dense_4bit_shapes`` gives.  ``Weight4Bit.quantize`` makes one from a float32 weight."""

    def __init__(self, codes, scales, in_features, out_features, group=128):
        shapes = K.dense_4bit_shapes(in_features, out_features, group)
        for name, a, shape, kind in (('codes', codes, shapes[0], np.uint8), ('scales', scales, shapes[1], np.float16)):
            if tuple(a.shape) != shape or a.dtype != kind:
                raise ValueError('Weight4Bit: %s of shape %s, %s, expected %s, %s' % (name, tuple(a.shape), a.dtype, shape, np.dtype(kind)))
        self.codes, self.scales = codes, scales
        self.in_features, self.out_features, self.group = int(in_features), int(out_features), int(group)

    @classmethod
    def quantize(cls, weight, group=128):
        """From an ``(in, out)`` weight, a Tensor or an array on the host or the device: in each group the value of largest magnitude
        becomes -8 times the scale, the others go to the nearest number.  Values of 5e5 and more are too large for
        the scale."""
        w = weight.eval if hasattr(weight, 'eval') else weight
        w = w if is_device(w) else to_device(np.ascontiguousarray(w), np.float32)
        if len(w.shape) != 2:
            raise ValueError('Weight4Bit: weight of shape %s' % (tuple(w.shape),))
        return cls(*K.quantize_4bit(w, group), *w.shape, group)

    def _on_device(self):
        """Both arrays on the device, where an unpickled weight may not be."""
        if not is_device(self.codes):
            self.codes, self.scales = to_device(self.codes), to_device(self.scales, np.float16)
        return self.codes, self.scales

    def dequantize(self):
        """The values that the codes stand for, an ``(in, out)`` float32 device array."""
        return K.dequantize_4bit(*self._on_device(), self.in_features, self.out_features, self.group)

    def product(self, x, bias=None, x_scale=None, out=None):
        return K.dense_4bit(x, *self._on_device(), self.in_features, self.out_features, self.group, bias, x_scale, out)
