"""AdamW on the device: moments in 32 and in 8 bits against their definitions, many tensors, odd sizes and places,
recorded steps."""
import numpy as np
import pytest

import xshinnosuke_amd as xs
from xshinnosuke_amd import backend as be
from xshinnosuke_amd.layers import Dense, ReLU
from xshinnosuke_amd.nn.models import Sequential
from xshinnosuke_amd.optim import AdamW
from adamw_plain import Plain

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24                                     # half a step of float32


@pytest.fixture(autouse=True)
def _fresh_state(gpu):
    xs.GLOBAL.INPUTS, xs.GLOBAL.USE_CUDA = None, False
    yield
    xs.GLOBAL.INPUTS, xs.GLOBAL.USE_CUDA = None, False


def _params(values):
    """Device parameters that lie in one array, one element apart: odd places, and guards around them."""
    flat = np.full(sum(v.size + 1 for v in values) + 1, 7.0, np.float32)
    places, at = [], 1
    for v in values:
        flat[at:at + v.size] = v.ravel()
        places.append(at)
        at += v.size + 1
    memory = be.to_device(flat)
    params = [xs.Parameter(xs.Tensor(memory.leading(a, a + v.size).reshape(v.shape), requires_grad=True)) for a, v in zip(places, values)]
    guards = np.setdiff1d(np.arange(flat.size), np.concatenate([np.arange(a, a + v.size) for a, v in zip(places, values)]))
    return params, memory, guards


def _starts(sizes):
    return np.concatenate([[0], np.cumsum([-(-n // 256) * 256 for n in sizes])[:-1]]).astype(int)


def _gradient(rng, shape):
    """Elements of very different sizes, a few zeros."""
    g = rng.standard_normal(shape) * np.exp(2 * rng.standard_normal(shape) - 3)
    return np.where(rng.random(shape) < 0.05, 0, g).astype(np.float32)


def _check_parameters(params, plain, changes, steps):
    for p, q, change in zip(params, plain, changes):
        # a step rounds p three times and forms the change with ten roundings on moments that carry four a step
        tol = steps * EPS * (3 * np.abs(q.p).max() + (10 + 4 * steps) * change)
        assert np.abs(p.numpy().ravel().astype(np.float64) - q.p).max() <= tol


SIZES = [(1,), (3,), (2, 2), (255,), (256,), (257,), (1, 1000), (1023,), (64, 64), (4097,), (33, 129)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shapes", [[(5,)], SIZES, [(7, 3)] * 100, [(1000, 1033), (1 << 20,)]], ids=["one", "sizes", "hundred", "large"])
def test_steps_follow_the_definition(bits, shapes):
    rng = np.random.default_rng(len(shapes))
    values = [rng.standard_normal(s).astype(np.float32) for s in shapes]
    params, memory, guards = _params(values)
    kw = dict(lr=0.01, betas=(0.9, 0.99), epsilon=1e-8)
    opt = AdamW(params, weight_decay=0.1, state_bits=bits, seed=99, **kw)
    starts = _starts([v.size for v in values])
    plain = [Plain(v, decay=0.1, bits=bits, seed=99, start=int(s), **kw) for v, s in zip(values, starts)]
    changes, steps = [0.0] * len(params), 4
    most = [[0.0, 0.0] for _ in params]
    for _ in range(steps):
        for i, (p, q) in enumerate(zip(params, plain)):
            g = _gradient(rng, p.shape)
            p.grad = xs.Tensor(be.to_device(g))
            changes[i] = max(changes[i], np.abs(q.step(g)).max())
            most[i] = [max(most[i][0], np.abs(g).max()), max(most[i][1], np.abs(g).max() ** 2)]
        opt.step()
    _check_parameters(params, plain, changes, steps)
    assert np.all(memory.numpy()[guards] == 7.0)
    (got, m, v), = opt.moments()
    assert got == params and m.size == starts[-1] + -(-values[-1].size // 256) * 256
    for q, s, top in zip(plain, starts, most):
        mine = m.numpy()[s:s + q.p.size], v.numpy()[s:s + q.p.size]
        if bits == 8:
            assert np.array_equal(mine[0], q.m.values()) and np.array_equal(mine[1], q.v.values())
        else:
            for a, b, t in zip(mine, (q.m, q.v), top):
                assert np.abs(a - b).max() <= 5 * steps * EPS * t


@pytest.mark.parametrize("bits,size", [(32, 8_000_037), (8, 12_900_037)])
def test_steps_whose_operands_are_streamed(bits, size):
    test_steps_follow_the_definition(bits, [(777,), (size,)])


def test_moments_decoded_in_one_call_equal_those_in_parts():
    rng = np.random.default_rng(8)
    blocks = 101_000
    codes = [be.to_device(rng.integers(0, 256, blocks * 256, dtype=np.uint8)) for _ in range(2)]
    exponents = [be.to_device(rng.integers(least, 254, blocks, dtype=np.uint8)) for least in (48, 64)]
    whole = be.kernels.adamw_moments(*codes, *exponents)
    for a, b in ((0, 50_000), (50_000, blocks)):
        part = be.kernels.adamw_moments(*[c.leading(256 * a, 256 * b) for c in codes], *[e.leading(a, b) for e in exponents])
        for x, y in zip(whole, part):
            assert np.array_equal(x.leading(256 * a, 256 * b).numpy(), y.numpy())


def test_extreme_gradients_in_eight_bits():
    """Infinite, NaN, huge and vanishing gradients: a block that held one reads as NaN, the others are not touched."""
    rng = np.random.default_rng(3)
    n = 256 * 6 + 17
    value = rng.standard_normal(n).astype(np.float32)
    params, _, _ = _params([value])
    opt, plain = AdamW(params, state_bits=8, seed=5), Plain(value, bits=8, seed=5)
    g = _gradient(rng, (n,))
    g[10], g[256 + 3], g[512 + 255], g[768:1024], g[1024:1280], g[-1] = np.inf, np.nan, 3e38, 1e-30, 0, 1e18
    g[1280:1536] *= 1e-16
    for _ in range(3):
        params[0].grad = xs.Tensor(be.to_device(g))
        plain.step(g)
        opt.step()
        g = _gradient(rng, (n,))
    (_, m, v), = opt.moments()
    for mine, theirs in ((m, plain.m.values()), (v, plain.v.values())):
        mine = mine.numpy()[:n]
        assert np.array_equal(mine, theirs, equal_nan=True)
    assert np.isnan(m.numpy()[:512]).all() and np.isnan(v.numpy()[:768]).all() and np.isfinite(m.numpy()[768:]).all()
    p = params[0].numpy()
    with np.errstate(invalid='ignore'):
        assert np.array_equal(np.isnan(p), np.isnan(plain.p)) and np.isnan(p[:256]).all() and np.isfinite(p[768:]).all()


def test_second_moment_in_eight_bits_follows_falling_gradients():
    """A thousand steps after the gradients have become ten times smaller the second moment's mean has followed them: to the
    nearest code it would have stayed where it was."""
    rng = np.random.default_rng(4)
    n = 1 << 16
    params, _, _ = _params([rng.standard_normal(n).astype(np.float32)])
    opt = AdamW(params, state_bits=8, lr=1e-6, betas=(0.9, 0.99), seed=1)
    expected = np.zeros(n)
    signs = [np.sign(rng.standard_normal(n)).astype(np.float32) for _ in range(4)]
    for size, steps in ((1.0, 50), (0.1, 400)):
        grads = [xs.Tensor(be.to_device(s * np.float32(size))) for s in signs]
        for k in range(steps):
            params[0].grad = grads[k % 4]
            opt.step()
            expected = 0.99 * expected + 0.01 * size * size
    v = opt.moments()[0][2].numpy().astype(np.float64)
    # one element's spread: an eighth of a step's value sized move with odds of 0.01 * 8: below 60 % of the value; 256 of them each
    assert abs(v.mean() / expected.mean() - 1) < 5 * 0.6 / 256
    assert abs(expected.mean() - 0.01) < 0.01


@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_steps_equal_eager_steps(bits):
    def run(recorded):
        rng = np.random.default_rng(6)
        params, memory, _ = _params([rng.standard_normal(s).astype(np.float32) for s in ((40, 30), (30,), (513,))])
        grads = [be.to_device(_gradient(rng, p.shape)) for p in params]
        for p, g in zip(params, grads):
            p.grad = xs.Tensor(g)
        opt = AdamW(params, state_bits=bits)
        seen, graph = [], None
        for k in range(6):
            for g in grads:
                g.set(_gradient(rng, g.shape))
            if recorded and k >= 2:
                if graph is None:
                    graph = be.StepGraph()
                    with graph.capture():
                        opt.step()
                graph.replay()
            else:
                opt.step()
            seen.append(memory.numpy())
            be.zeros((1000 + k,)).numpy()                # eager work between the replays
            be.synchronize()
        (_, m, v), = opt.moments()
        return seen + [m.numpy(), v.numpy()]

    for a, b in zip(run(False), run(True)):
        assert np.array_equal(a, b)


def test_moments_are_not_made_while_recording():
    params, _, _ = _params([np.ones(5, np.float32)])
    params[0].grad = xs.Tensor(be.to_device(np.ones(5, np.float32)))
    opt = AdamW(params)
    graph = be.StepGraph()
    with pytest.raises(be.XsmiError, match="before a step is recorded"):
        with graph.capture():
            opt.step()


def test_moving_between_host_and_device_keeps_the_moments():
    rng = np.random.default_rng(7)
    value = rng.standard_normal(300).astype(np.float32)
    p = xs.Parameter(xs.Tensor(value.copy(), requires_grad=True))
    opt, plain, change = AdamW([p]), Plain(value), 0.0
    for place in ('cpu', 'cuda', 'cuda', 'cpu', 'cuda'):
        p.cuda_() if place == 'cuda' else p.cpu_()
        xs.GLOBAL.USE_CUDA = False
        g = _gradient(rng, (300,))
        p.grad = xs.Tensor(be.to_device(g) if place == 'cuda' else g)
        change = max(change, np.abs(plain.step(g)).max())
        opt.step()
        assert p.device == place
    _check_parameters([p], [plain], [change], 5)


def test_a_lot_of_host_and_new_parameters_moves_to_the_device():
    """Parameters with and without steps behind them, all on the device from now on: each keeps its own count."""
    rng = np.random.default_rng(17)
    values = [rng.standard_normal(n).astype(np.float32) for n in (7, 300, 11)]
    params = [xs.Parameter(xs.Tensor(v.copy(), requires_grad=True)) for v in values]
    plain = [Plain(v) for v in values]
    opt, changes = AdamW(params), [0.0] * 3
    for step in range(4):
        if step == 2:
            for p in params:
                p.cuda_()
            xs.GLOBAL.USE_CUDA = False
        for i, (p, q) in enumerate(zip(params, plain)):
            if i == 2 and step < 2:
                continue
            g = _gradient(rng, p.shape)
            p.grad = xs.Tensor(be.to_device(g) if step >= 2 else g)
            changes[i] = max(changes[i], np.abs(q.step(g)).max())
        opt.step()
    _check_parameters(params, plain, changes, 4)
    assert sorted(len(g[0]) for g in opt.moments()) == [1, 2]


def test_new_parameters_and_gradients_start_their_own_count():
    rng = np.random.default_rng(8)
    params, _, _ = _params([rng.standard_normal(n).astype(np.float32) for n in (10, 20)])
    late = params[1].numpy()
    params[0].grad = xs.Tensor(be.to_device(np.ones(10, np.float32)))
    opt = AdamW(params, lr=0.01, weight_decay=0)
    for _ in range(3):
        opt.step()
    assert np.array_equal(params[1].numpy(), late)
    params[1].grad = xs.Tensor(be.to_device(np.ones(20, np.float32)))
    opt.step()
    np.testing.assert_allclose(params[1].numpy(), late - 0.01, rtol=0, atol=1e-6)
    assert [len(g[0]) for g in opt.moments()] == [1, 1]
    params[0].requires_grad = False
    before = params[0].numpy()
    opt.step()
    assert np.array_equal(params[0].numpy(), before) and not np.array_equal(params[1].numpy(), late - 0.01)


@pytest.mark.parametrize("bits", [32, 8])
def test_fit_on_the_device_saves_and_goes_on(tmp_path, bits, monkeypatch):
    """fit() with and without a recorded step gives the same losses; a checkpoint goes on where it was."""
    np.random.seed(0)
    x, y = np.random.randn(40, 12).astype(np.float32), np.random.randint(0, 3, (40,))

    def net():
        np.random.seed(1)
        xs.GLOBAL.USE_CUDA = True
        n = Sequential(Dense(16, input_shape=(12,)), ReLU(), Dense(3))
        n.compile('adamw', 'cross_entropy', lr=0.01, state_bits=bits)
        return n

    a = net()
    first = a.fit(x, y, batch_size=8, epochs=2, verbose=0, shuffle=False)['train_loss']
    a.save(str(tmp_path / 'ck'))
    monkeypatch.setattr(xs.GLOBAL, 'STEP_GRAPH', True)
    assert net().fit(x, y, batch_size=8, epochs=2, verbose=0, shuffle=False)['train_loss'] == first
    monkeypatch.setattr(xs.GLOBAL, 'STEP_GRAPH', False)
    b = Sequential()
    b.load(str(tmp_path / 'ck.pkl'))
    more = [n.fit(x, y, batch_size=8, epochs=1, verbose=0, shuffle=False)['train_loss'] for n in (a, b)]
    assert more[0] == more[1] and more[0][0] < first[0]


def test_refusals():
    params, _, _ = _params([np.ones(5, np.float32)])
    params[0].grad = xs.Tensor(be.to_device(np.ones(4, np.float32)))
    with pytest.raises(ValueError, match="one size"):
        AdamW(params).step()
    params[0].grad = xs.Tensor(be.to_device(np.ones(5, np.int32)))
    with pytest.raises(ValueError, match="float32"):
        AdamW(params).step()
    with pytest.raises(ValueError):
        be.kernels.adamw_moments(*(be.zeros((n,), np.uint8) for n in (256, 256, 1, 2)))
    call = lambda *a: be.lib.call("xsmi_adamw_step", *a)  # noqa: E731
    m, s = be.zeros((512,)), be.zeros((3,), np.int64)
    import ctypes
    one = (ctypes.c_void_p * 1)(m.ptr)
    size = lambda v: (ctypes.c_size_t * 1)(v)  # noqa: E731
    rates = (0.1, 0.9, 0.999, 1e-8, 0.0, 0)
    for start, n, room, bits, rest in ((1, 5, 512, 32, rates), (512, 5, 512, 32, rates), (0, 513, 512, 32, rates), (0, 5, 500, 32, rates),
                                       (0, 5, 512, 16, rates), (0, 5, 512, 8, rates), (0, 5, 512, 32, (0.1, 1.0, 0.9, 0, 0, 0)),
                                       (0, 5, 512, 32, (-0.1, 0.9, 0.9, 0, 0, 0))):
        with pytest.raises(ValueError):
            call(1, one, one, size(start), size(n), m.ptr, m.ptr, None, None, room, bits, *rest, s.ptr)
    with pytest.raises(ValueError):
        call(1, one, one, size(0), size(5), m.ptr + 4, m.ptr, None, None, 256, 32, *rates, s.ptr)
