"""Optimizers (counterpart of xs/optim).  Of the reference's only SGD demonstrably works (the others use an
undefined ``np``, e.g. xs/optim/sgd.py:21), so only SGD follows it; AdamW is this package's own."""
from ..nn import array_ops as A
from .base import Optimizer
from .adamw import AdamW


class SGD(Optimizer):
    def step(self):
        """v -= lr * v.grad for every trainable parameter (reference xs/optim/sgd.py:4-9)."""
        A.sgd_step_all([(v.eval, v.grad.eval) for v in self._parameters if v.requires_grad and v.grad is not None],
                       self.lr)
        super().step()


def get_optimizer(optimizer, **kwargs):
    if isinstance(optimizer, str):
        if optimizer.lower() in ('sgd',):
            return SGD(**kwargs)
        if optimizer.lower() in ('adamw',):
            return AdamW(**kwargs)
        raise ValueError('unknown optimizer %r (sgd and adamw are available)' % optimizer)
    if isinstance(optimizer, Optimizer):
        if kwargs.get('parameters') is not None:
            optimizer._parameters = kwargs['parameters']
        return optimizer
    raise ValueError('unknown optimizer type!')
