"""Dense and Flatten (counterpart of xs/layers/linear.py), and Dense4Bit (this package's own)."""
import math

from .base import Layer, F, Parameter, Tensor
from .activators import Activation, FusedActivation
from ..nn.initializers import get_initializer
from ..nn.weight4 import Weight4Bit


class Dense(FusedActivation, Layer):
    """``y = act(x @ W + b)``, W ``(in, out)``, b ``(1, out)``; ``activation`` names 'relu', 'sigmoid' or
    'tanh' (a child activation layer on the product's output)."""

    def __init__(self, out_features, activation=None, use_bias=True, kernel_initializer='normal',
                 bias_initializer='zeros', **kwargs):
        self.out_features = out_features
        self.use_bias = use_bias
        self.kernel_initializer = get_initializer(kernel_initializer)
        self.bias_initializer = get_initializer(bias_initializer)
        self._set_activation(activation, fuse_relu=False)
        super().__init__(**kwargs)

    def compute_output_shape(self, input_shape=None):
        self._shape = (self.out_features,)
        return self._shape

    def init_params(self, input_shape=None, *args):
        if input_shape is not None:
            self._input_shape = tuple(input_shape)
        w_shape = tuple(self._input_shape) + (self.out_features,)
        self._parameters.append(Parameter(self.kernel_initializer(w_shape, requires_grad=True)))
        if self.use_bias:
            self._parameters.append(Parameter(self.bias_initializer((1, self.out_features), requires_grad=True)))

    def init_layer_out_tensor(self, x=None):
        super().init_layer_out_tensor(x)
        self._static_act_buffer()

    def call(self, x, *args, **kwargs):
        weight = self._parameters[0]
        if self.use_bias:
            self._data = F.addmm(self._parameters[1], x, weight, self._data)
        else:
            self._data = F.mm(x, weight, self._data)
        return self._activate(self._data)

    def backward(self, gradients=None):
        self._act_backward()
        super().backward(gradients)


class Dense4Bit(FusedActivation, Layer):
    """A trained ``Dense`` with its weight in 4 bits, for inference: ``Dense4Bit.from_dense(layer, group)`` packs the weight and
    takes over the bias and the activation.  It takes float32 rows, or, called as ``layer(q, scale=scale)``, the 8-bit rows of
    ``rms_norm_8bit``.  It has no parameters to train and no backward."""

    def __init__(self, weight, bias=None, activation=None, **kwargs):
        if not isinstance(weight, Weight4Bit):
            raise ValueError('Dense4Bit: weight must be a Weight4Bit')
        self.weight, self.bias, self.out_features = weight, bias, weight.out_features
        self._set_activation(activation, fuse_relu=False)
        kwargs.setdefault('trainable', False)
        kwargs.setdefault('input_shape', (weight.in_features,))
        super().__init__(**kwargs)

    @classmethod
    def from_dense(cls, dense, group=128):
        params = dense.parameters()
        if not params:
            raise ValueError('Dense4Bit: the layer has no weight yet')
        bias = None
        if dense.use_bias:
            b = params[1].eval
            bias = Tensor(F.to_device(b) if not F.is_device(b) else b.copy())
        act = dense._act_layer
        return cls(Weight4Bit.quantize(params[0], group), bias, act if isinstance(act, Activation) else act and type(act).__name__)

    def compute_output_shape(self, input_shape=None):
        self._shape = (self.out_features,)
        return self._shape

    def init_layer_out_tensor(self, x=None):
        super().init_layer_out_tensor(x)
        self._static_act_buffer()

    def call(self, x, scale=None, *args, **kwargs):
        out = None if x.is_dynamic else self._data       # a dynamic call may read what the one before it wrote
        if out is not None and (out.eval is None or tuple(out.shape) != tuple(x.shape[:-1]) + (self.out_features,)):
            out = None
        self._data = F.dense_4bit(x, self.weight, self.bias, scale, out)
        return self._activate(self._data)

    def backward(self, gradients=None):
        raise NotImplementedError('Dense4Bit has no backward')


class Flatten(Layer):
    def __init__(self, start_dim=1, **kwargs):
        if start_dim < 1:
            raise ValueError('start_dim must be > 0')
        self.start_dim = start_dim
        super().__init__(**kwargs)

    def compute_output_shape(self, input_shape=None):
        keep = self.start_dim - 1
        self._shape = tuple(input_shape[:keep]) + (math.prod(input_shape[keep:]),)
        return self._shape

    def call(self, x, *args, **kwargs):
        self._data = F.flatten(x, self.start_dim, self._data)
        return self._data
