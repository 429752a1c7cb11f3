"""rms_norm on host tensors (gradients against differences), its graph wiring, and what it refuses."""
import numpy as np
import pytest

import xshinnosuke_amd as xs
from xshinnosuke_amd.backend import capi
from xshinnosuke_amd.layers import Dense, ReLU, RMSNormalization
from xshinnosuke_amd.nn import functional as F
from xshinnosuke_amd.nn.models import Module, Sequential


@pytest.fixture(autouse=True)
def _fresh_state():
    xs.GLOBAL.INPUTS = None
    yield
    xs.GLOBAL.INPUTS = None


def _tensors(rng, shape):
    x, r = (xs.Tensor(rng.standard_normal(shape), requires_grad=True) for _ in range(2))
    return x, r, xs.Parameter(xs.Tensor(rng.standard_normal(shape[-1:]), requires_grad=True))


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("shape", [(1, 1), (3, 5), (2, 3, 4)])
def test_gradients_equal_differences(shape, residual):
    rng = np.random.default_rng(0)
    x, r, gamma = _tensors(rng, shape)
    dy, ds = rng.standard_normal(shape), rng.standard_normal(shape)

    def value():
        with xs.no_grad():
            if residual:
                y, s = F.rms_norm(x, gamma, r, epsilon=0.1)
                return float((y.eval * dy + s.eval * ds).sum())
            return float((F.rms_norm(x, gamma, epsilon=0.1).eval * dy).sum())

    if residual:
        y, s = F.rms_norm(x, gamma, r, epsilon=0.1)
        s.grad = xs.Tensor(ds.copy())
    else:
        y = F.rms_norm(x, gamma, epsilon=0.1)
    y.backward(xs.Tensor(dy))
    for t in (x, gamma) + ((r,) if residual else ()):
        want = np.zeros(t.shape)
        for i in np.ndindex(*t.shape):
            at = t.eval[i]
            t.eval[i] = at + 1e-5
            up = value()
            t.eval[i] = at - 1e-5
            want[i] = (up - value()) / 2e-5
            t.eval[i] = at
        # second-order error of the difference: 1e-10 times a third derivative of a few; rounding: 1e-15 / 1e-5
        np.testing.assert_allclose(t.grad.eval, want, rtol=0, atol=1e-7)


def test_one_tensor_as_both_addends_and_a_sum_that_is_used_again():
    rng = np.random.default_rng(1)
    x, _, gamma = _tensors(rng, (3, 4))
    y, s = F.rms_norm(x, gamma, x)
    z = y + s
    z.backward(xs.Tensor(np.ones((3, 4))))
    twice = x.grad.eval.copy()
    x.zero_grad()
    gamma.zero_grad()
    xs.GLOBAL.INPUTS = None
    s = x + x
    z = F.rms_norm(s, gamma) + s
    z.backward(xs.Tensor(np.ones((3, 4))))
    np.testing.assert_allclose(twice, x.grad.eval, rtol=1e-12)


def test_layer_in_both_graph_styles():
    np.random.seed(3)
    x, y = np.random.randn(20, 6).astype(np.float32), np.random.randint(0, 3, (20,))
    net = Sequential(Dense(8, input_shape=(6,)), RMSNormalization(), ReLU(), Dense(3))
    net.compile('adamw', 'cross_entropy', lr=0.01)
    assert len(net.parameters()) == 5
    net.fit(x, y, batch_size=8, epochs=2, verbose=0)
    assert net.predict(x).shape == (20, 3)

    class Net(Module):
        def __init__(self):
            super().__init__()
            self.layers = [Dense(6), RMSNormalization(), Dense(3)]

        def forward(self, x):
            y, s = self.layers[1](self.layers[0](x), x)
            return self.layers[2](y)

    net = Net()
    t = xs.Tensor(x, requires_grad=True)
    loss = xs.nn.CrossEntropyLoss()(net(t), xs.Tensor(y))
    assert len(net.parameters()) == 5
    loss.backward()
    assert all(p.grad is not None and np.abs(p.grad.eval).max() > 0 for p in net.parameters())


def test_one_layer_twice_in_a_forward():
    rng = np.random.default_rng(3)
    x, w = xs.Tensor(rng.standard_normal((3, 4)), requires_grad=True), rng.standard_normal((3, 4))
    norm = RMSNormalization(epsilon=0.1)

    class Net(Module):
        def forward(self, x):
            a = norm(x)
            return norm(a * xs.Tensor(w)) + a

    Net()(x).backward(xs.Tensor(np.ones((3, 4))))
    grads = [t.grad.eval.copy() for t in (x, norm.parameters()[0])]
    xs.GLOBAL.INPUTS = None
    u, gamma = xs.Tensor(x.eval.copy(), requires_grad=True), xs.Parameter(xs.Tensor(np.ones(4), requires_grad=True))
    a = F.rms_norm(u, gamma, epsilon=0.1)
    z = F.rms_norm(a * xs.Tensor(w), gamma, epsilon=0.1) + a
    z.backward(xs.Tensor(np.ones((3, 4))))
    for got, want in zip(grads, (u.grad.eval, gamma.grad.eval)):
        np.testing.assert_allclose(got, want, rtol=1e-6, atol=1e-7)       # the layer's scales are float32


def test_refusals():
    rng = np.random.default_rng(2)
    x, r, gamma = _tensors(rng, (3, 4))
    for out in (x, r, gamma):
        with pytest.raises(ValueError):
            F.rms_norm(x, gamma, r, out=out)
    with pytest.raises(ValueError):
        F.rms_norm(x, xs.Parameter(xs.Tensor(np.ones(3))))
    with pytest.raises(ValueError):
        F.rms_norm(x, gamma, xs.Tensor(np.ones((1, 4))))
    with pytest.raises(ValueError):
        F.rms_norm(x, gamma, epsilon=-1)
    with pytest.raises(ValueError):
        F.rms_norm(x, gamma, epsilon=float('nan'))
    with pytest.raises(NotImplementedError):
        F.rms_norm_8bit(x, gamma)
    query = capi.lib.raw("xsmi_rms_norm_workspace_bytes")
    assert query(0, 5) == 0 and query(1 << 31, 5) == 0 and query(5, 0) == 0 and query(5, -1) == 0
    assert query(3, 100) == 0 and query(4096, 4096) >= 4 * 4096 and query(1 << 20, 16384) <= 1 << 28
