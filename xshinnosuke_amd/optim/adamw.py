"""AdamW: Adam with decoupled weight decay, over all parameters in one launch, its moments in 32 or in 8 bits.

No counterpart in the reference, whose optimizers beside SGD do not run (they use an undefined ``np``).
"""
import ctypes

import numpy as np

from ..backend import XsmiError, kernels as K
from ..backend import array as dev

from ..nn import array_ops as A
from .base import Optimizer

_FULL = slice(None, None, None)


class _DeviceMoments:
    """The moments of the device parameters that the optimizer met together, and their count of steps.  Each moment is one
    flat array in which a parameter has a stretch that starts at a multiple of 256 elements (blocks of the 8-bit form
    never hold two parameters)."""

    def __init__(self, params, bits, steps=0, values=None):
        if dev._CAPTURE[0] is not None:
            raise XsmiError("AdamW's moments must exist before a step is recorded: run one step first")
        self.params, self.bits = list(params), bits
        self.sizes, self.starts, total = [p._data.size for p in self.params], [], 0
        for size in self.sizes:
            self.starts.append(total)
            total += -(-size // 256) * 256
        total = max(total, 256)
        kind = np.float32 if bits == 32 else np.uint8
        self.m, self.v = dev.zeros((total,), kind), dev.zeros((total,), kind)
        self.me = self.ve = None
        if bits == 8:
            self.me, self.ve = dev.zeros((total // 256,), np.uint8), dev.zeros((total // 256,), np.uint8)
        self.state = dev.to_device(np.array([steps, 0, 0], np.int64))
        for start, size, pair in zip(self.starts, self.sizes, values or ()):
            for flat, value in zip((self.m, self.v), pair):
                flat.leading(start, start + size).set(np.asarray(value, np.float32).reshape(-1))
        self.launch = None

    def __getstate__(self):
        return dict(self.__dict__, launch=None)      # it holds addresses

    def steps(self):
        return int(np.asarray(self.state)[0])

    def decoded(self):
        """(m, v) as flat float32 arrays; those that are held in 32 bits themselves."""
        return (self.m, self.v) if self.bits == 32 else K.adamw_moments(self.m, self.v, self.me, self.ve)


class _Launch:
    """The arguments of a step that stay the same while every parameter and gradient keeps its array."""

    def __init__(self, moments):
        self.of = []                                  # (parameter, its array, gradient tensor, its array)
        values, grads, starts = [], [], []
        self.lasting = True
        for p, start, size in zip(moments.params, moments.starts, moments.sizes):
            if p is None or p._grad is None or not p.requires_grad:
                self.lasting = False
                continue
            value, grad = p.eval, p.grad.eval
            if not A.is_device(grad) or value is not p._data or grad is not p._grad._data:
                self.lasting = False
            grad = A.same_place(value, grad)
            if value.size != grad.size or value.dtype != np.float32 or grad.dtype != np.float32:
                raise ValueError("AdamW: parameter %s %s and gradient %s %s: both must be float32, of one size"
                                 % (value.shape, value.dtype, grad.shape, grad.dtype))
            if value.size > size:
                raise ValueError("AdamW: parameter %s has moments of %d elements" % (value.shape, size))
            self.of.append((p, value, p._grad, grad))
            values.append(value)
            grads.append(grad)
            starts.append(start)
        self.values, self.grads = values, grads
        self.ids = {id(p) for p, _, _, _ in self.of}
        n = len(values)
        self.count = n
        self.pp = (ctypes.c_void_p * n)(*[a.address() for a in values])
        self.gp = (ctypes.c_void_p * n)(*[a.address() for a in grads])
        self.starts = (ctypes.c_size_t * n)(*starts)
        self.ns = (ctypes.c_size_t * n)(*[a.size for a in values])

    def holds(self):
        if not self.lasting:
            return False
        for p, value, grad_tensor, grad in self.of:
            if p._data is not value or p._grad is not grad_tensor or grad_tensor._data is not grad or p._slices != _FULL or not p.requires_grad:
                return False
        return True

    def run(self, moments, opt):
        if self.count:
            K.adamw_step(self, moments, opt)
        return self.values


class AdamW(Optimizer):
    """``p -= lr * (m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + epsilon) + weight_decay * p)`` with the moments
    ``m = beta1 m + (1 - beta1) g`` and ``v = beta2 v + (1 - beta2) g^2``.

    ``state_bits=8`` (device parameters) holds both moments in 8 bits with an exponent for each 256 elements, a quarter of
    the memory and four sevenths of a step's traffic; they are rounded stochastically, by noise that ``seed`` and the
    step decide, so that runs repeat.  ``t`` counts a parameter's own steps; on the device it is kept there, and a step recorded with
    ``StepGraph`` goes on counting when it is replayed (the recording freezes the rate, the betas, epsilon and the decay).
    A gradient that has become infinite or NaN makes its element NaN, with 8 bits the whole block of 256."""

    def __init__(self, parameters=None, lr=0.001, betas=(0.9, 0.999), epsilon=1e-8, weight_decay=0.01, state_bits=32, seed=0):
        super().__init__(parameters, lr, weight_decay)
        if len(betas) != 2 or not all(0 <= b < 1 for b in betas):
            raise ValueError('AdamW: betas must be two numbers in [0, 1), got %r' % (betas,))
        if not (lr >= 0 and epsilon >= 0 and weight_decay >= 0):
            raise ValueError('AdamW: lr, epsilon and weight_decay must not be negative')
        if state_bits not in (8, 32):
            raise ValueError('AdamW: state_bits must be 8 or 32, got %r' % (state_bits,))
        self.betas, self.epsilon, self.state_bits, self.seed = tuple(betas), epsilon, state_bits, int(seed) & 0xFFFFFFFF
        self._groups = []            # _DeviceMoments
        self._host = {}              # parameter -> [m, v, steps]

    def _settle(self):
        """Moments for every parameter that needs them, where the parameter is."""
        walk = self._parameters
        if isinstance(walk, (set, frozenset)):       # models hand over a set: in an order that repeats from run to run
            walk = sorted(walk, key=lambda p: getattr(p, 'serial', 0))
        at = {id(p): g for g in self._groups for p in g.params if p is not None}
        fresh, host, seen = [], [], set()
        for p in walk:
            if not p.requires_grad or p._grad is None or id(p) in seen:
                continue
            seen.add(id(p))
            if A.is_device(p._data):
                if id(p) not in at:
                    fresh.append(p)
            else:
                host.append(p)
                if id(p) in at:
                    self._fetch(p, at[id(p)])
                elif p not in self._host:
                    if self.state_bits == 8:
                        raise NotImplementedError('AdamW: 8-bit moments need device tensors')
                    self._host[p] = [np.zeros_like(p._data), np.zeros_like(p._data), 0]
        lots = {}                                     # by steps taken: those of a parameter that comes from the host go on
        for p in fresh:
            m, v, steps = self._host.pop(p, (np.zeros(p._data.size, np.float32),) * 2 + (0,))
            lots.setdefault(steps, []).append((p, (m, v)))
        for steps, lot in lots.items():
            self._groups.append(_DeviceMoments([p for p, _ in lot], self.state_bits, steps, [pair for _, pair in lot] if steps else None))
        return host

    def _fetch(self, p, group):
        """A parameter has moved to the host since its last step: so do its moments."""
        if group.bits == 8:
            raise NotImplementedError('AdamW: 8-bit moments need device tensors')
        i = [q is p for q in group.params].index(True)
        if p._data.size != group.sizes[i]:
            raise ValueError('AdamW: parameter %s has moments of %d elements' % (p._data.shape, group.sizes[i]))
        stretch = slice(group.starts[i], group.starts[i] + group.sizes[i])
        self._host[p] = [np.asarray(a)[stretch].reshape(p._data.shape).astype(p._data.dtype) for a in (group.m, group.v)] + [group.steps()]
        group.params[i] = group.launch = None

    def step(self):
        # the usual step: the parameters and gradients of the last one, all on the device
        launch = self._groups[0].launch if len(self._groups) == 1 and not self._host else None
        if launch is not None and launch.holds() and all(id(p) in launch.ids for p in self._parameters):
            updated = launch.run(self._groups[0], self)
        else:
            for p in self._settle():
                self._host_step(p)
            updated = []
            for g in self._groups:
                if g.launch is None or not g.launch.holds():
                    g.launch = _Launch(g)
                updated += g.launch.run(g, self)
        if updated:
            K.refresh_layouts(updated)
        super().step()

    def _host_step(self, p):
        (b1, b2), state = self.betas, self._host[p]
        m, v = state[0], state[1]
        state[2] = t = state[2] + 1
        value, g = p.eval, np.asarray(A.same_place(p._data, p.grad.eval)).reshape(p.eval.shape)
        if m.shape != value.shape:
            raise ValueError('AdamW: parameter %s has moments of shape %s' % (value.shape, m.shape))
        m *= b1
        m += (1 - b1) * g
        v *= b2
        v += (1 - b2) * g * g
        value *= 1 - self.lr * self.weight_decay
        value -= self.lr / (1 - b1 ** t) * m / (np.sqrt(v) / np.sqrt(1 - b2 ** t) + self.epsilon)

    def moments(self):
        """The moments of the device parameters as float32: a list of ``(parameters, m, v)``, one for each lot of parameters that got
        their first gradients together.  ``m`` and ``v`` are flat device arrays; in the order of ``parameters`` each has a
        stretch of its size there, and the next one starts at the next multiple of 256 elements.  Moments of 32 bits are
        the optimizer's own arrays, those of 8 bits are decoded into new ones."""
        return [(list(g.params),) + tuple(g.decoded()) for g in self._groups]
