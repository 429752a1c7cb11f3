"""AdamW on host tensors, its 8-bit moments' definition, and what it refuses without a device."""
import ctypes
import pickle

import numpy as np
import pytest

import xshinnosuke_amd as xs
from xshinnosuke_amd.backend import capi
from xshinnosuke_amd.layers import Dense, ReLU
from xshinnosuke_amd.nn.models import Sequential
from xshinnosuke_amd.optim import AdamW, get_optimizer
from adamw_plain import Code, Plain, mix, noise


def _param(value, grad):
    p = xs.Parameter(xs.Tensor(value.copy(), requires_grad=True))
    p.grad = xs.Tensor(grad.copy())
    return p


def test_host_steps_follow_the_formula():
    rng = np.random.default_rng(0)
    shapes = [(3, 4), (1, 7), (5,)]
    params = [_param(rng.standard_normal(s), rng.standard_normal(s)) for s in shapes]
    plain = [Plain(p.numpy(), lr=0.01, betas=(0.8, 0.95), epsilon=1e-6, decay=0.1) for p in params]
    opt = AdamW(params, lr=0.01, betas=(0.8, 0.95), epsilon=1e-6, weight_decay=0.1)
    for _ in range(5):
        for p, q in zip(params, plain):
            g = rng.standard_normal(p.shape).astype(np.float32)
            p.grad.eval[...] = g
            q.step(g)
        opt.step()
    assert opt.iterations == 5
    for p, q in zip(params, plain):
        # float64: five steps of ten roundings of 2^-53 each, on values below 4
        assert np.abs(p.numpy().ravel() - q.p).max() < 5 * 10 * 2.0 ** -53 * 4


def test_parameters_without_gradients_and_repeated_ones():
    rng = np.random.default_rng(1)
    a, b = _param(rng.standard_normal(4), rng.standard_normal(4)), xs.Parameter(xs.Tensor(rng.standard_normal(3), requires_grad=True))
    frozen = _param(rng.standard_normal(2), rng.standard_normal(2))
    frozen.requires_grad = False
    before, plain = (b.numpy().copy(), frozen.numpy().copy()), Plain(a.numpy())
    opt = AdamW([a, b, a, frozen])
    plain.step(a.grad.numpy())
    opt.step()
    assert np.array_equal(b.numpy(), before[0]) and np.array_equal(frozen.numpy(), before[1])
    np.testing.assert_allclose(a.numpy(), plain.p, rtol=1e-6)     # the plain one takes the gradient in 32 bits
    b.grad = xs.Tensor(np.ones(3))                                  # its own first step: the corrections are those of t = 1
    opt.step()
    np.testing.assert_allclose(b.numpy(), before[0] * (1 - 1e-5) - 1e-3, rtol=0, atol=1e-8)


def test_fit_save_load_and_go_on(tmp_path):
    np.random.seed(0)
    x, y = np.random.randn(24, 6).astype(np.float32), np.random.randint(0, 3, (24,))
    net = Sequential(Dense(8, input_shape=(6,)), ReLU(), Dense(3))
    net.compile('adamw', 'cross_entropy', lr=0.01, weight_decay=0.1, betas=(0.9, 0.99))
    assert isinstance(net.optimizer, AdamW) and net.optimizer.betas == (0.9, 0.99)
    net.fit(x, y, batch_size=8, epochs=2, verbose=0)
    net.save(str(tmp_path / 'ck'))
    again = Sequential()
    again.load(str(tmp_path / 'ck.pkl'))
    a = net.fit(x, y, batch_size=8, epochs=2, verbose=0, shuffle=False)
    b = again.fit(x, y, batch_size=8, epochs=2, verbose=0, shuffle=False)
    assert a['train_loss'] == b['train_loss'] and again.optimizer.iterations == net.optimizer.iterations == 12


def test_a_parameter_of_another_size_is_refused():
    p = _param(np.ones(3), np.ones(3))
    opt = AdamW([p])
    opt.step()
    p._data, p.grad = np.ones(4), xs.Tensor(np.ones(4))
    with pytest.raises(ValueError):
        opt.step()


def test_refusals():
    p = _param(np.ones(3), np.ones(3))
    for bad in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(betas=(0.9,)), dict(lr=-1), dict(lr=float('nan')), dict(epsilon=-1e-8),
                dict(weight_decay=-1), dict(state_bits=16)):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    with pytest.raises(NotImplementedError):
        AdamW([p], state_bits=8).step()
    with pytest.raises(ValueError):
        get_optimizer('adamax')
    dll = ctypes.CDLL(capi.library_path())
    if not dll.xsmi_is_initialized():
        dll.xsmi_adamw_step.argtypes = capi.SIGNATURES["xsmi_adamw_step"][1]
        assert dll.xsmi_adamw_step(0, None, None, None, None, None, None, None, None, 0, 32, 0, 0, 0, 0, 0, 0, None) == 3


def test_pickled_optimizer_holds_no_addresses():
    p = _param(np.ones(3), np.ones(3))
    opt = AdamW([p])
    opt.step()
    again = pickle.loads(pickle.dumps(opt))
    (q,) = again._parameters
    again.step()
    opt.step()
    assert np.array_equal(q.numpy(), p.numpy())


def test_code_keeps_what_it_can_hold_and_is_unbiased():
    """Codes come back as themselves whatever the noise, the mean over all noise is the value, and the hash's halves are even."""
    rng = np.random.default_rng(2)
    for signed in (True, False):
        code = Code(1000, signed)
        x = (rng.standard_normal(1000) * np.exp(3 * rng.standard_normal(1000))).astype(np.float32)
        code.store(x if signed else np.abs(x), np.full(1000, 0x8000))
        kept = code.values()
        for n in (0, 0x7FFF, 0xFFFF):
            code.store(kept, np.full(1000, n))
            assert np.array_equal(code.values(), kept)
        most = 0.0
        for value in (1.0, 0.33, 1e-3, 2e-5):
            one = Code(65536, signed)
            v = np.full(65536, value, np.float32)
            v[::256] = 1.0                                           # every block's largest
            one.store(v, np.arange(65536))
            got = one.values()[v == np.float32(value)].astype(np.float64).mean()
            most = max(most, abs(got / value - 1))
        # all noise of a step but one 256th of it, spread evenly: off by less than an eighth times a 256th, or a 256th of the smallest code
        assert most < (1 / 8) / 256 if signed else most < 1 / 256
    of_m, of_v = noise(0, 1 << 16, 3, 7)
    for n in (of_m, of_v):
        # mean of 65536 even 16-bit numbers: 32767.5, five standard deviations of 18918 / 256
        assert abs(n.mean() - 32767.5) < 5 * 18918 / 256
    assert abs(np.corrcoef(of_m, of_v)[0, 1]) < 5 / 256 and abs(np.corrcoef(of_m[1:], of_m[:-1])[0, 1]) < 5 / 256
    assert abs(np.corrcoef(of_m, noise(0, 1 << 16, 4, 7)[0])[0, 1]) < 5 / 256
    assert int(mix(0)) == 0 and int(mix(1)) != int(mix(2))
