"""Dense layers with weights in 4 bits: packing, products of float32 and 8-bit rows against 64 bits, the layer, and the
path that serves a trained residual network with them."""
import numpy as np
import pytest

import xshinnosuke_amd as xs
from xshinnosuke_amd import backend as be
from xshinnosuke_amd.layers import Dense, Dense4Bit, ReLU, RMSNormalization
from xshinnosuke_amd.nn import Weight4Bit, functional as F
from xshinnosuke_amd.nn.models import Sequential
from dense4_plain import pack, quantize, up, values

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24                                     # half a step of float32


@pytest.fixture(autouse=True)
def _fresh_state(gpu):
    xs.GLOBAL.INPUTS, xs.GLOBAL.USE_CUDA = None, False
    yield
    xs.GLOBAL.INPUTS, xs.GLOBAL.USE_CUDA = None, False
    xs.GLOBAL.TRAINING = True


def _weight(rng, k, n, group):
    numbers = rng.integers(-8, 8, (k, n))
    scales = (np.exp(rng.standard_normal((up(k, 128) // group, n))) * 0.01).astype(np.float16)
    codes, padded = pack(numbers, scales, group)
    return Weight4Bit(be.to_device(codes), be.to_device(padded, np.float16), k, n, group), values(numbers, scales, group)


def _tolerance(x, w, group, whole=False):
    """Of sums over k: a group's multiplications add one after the other at worst, and so do the groups; float32 rows have been
    split, off by 2^-22 of a value and 2^-28 of the row's largest."""
    k = x.shape[1]
    groups = up(k, 128) // group
    size = np.abs(x) @ np.abs(w)
    if whole:
        return (2 * groups + 12) * EPS * size
    return ((group + groups + 12) * EPS + 2.0 ** -22) * size + 2.0 ** -28 * np.abs(x).max(1, keepdims=True) * np.abs(w).sum(0)


ROWS = [1, 2, 3, 4, 5, 8, 9, 13, 16, 17, 33, 48, 49, 64, 65, 130]
SHAPES = [(1, 1), (7, 3), (32, 16), (127, 17), (128, 15), (129, 100), (512, 1000), (1000, 33), (2177, 40), (9001, 19), (20000, 5)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("k,n", SHAPES)
def test_products(k, n, group):
    rng = np.random.default_rng(k + n)
    weight, w = _weight(rng, k, n, group)
    for m in ROWS:
        x = (rng.standard_normal((m, k)) * np.exp(rng.standard_normal(k))).astype(np.float32)
        bias = rng.standard_normal(n).astype(np.float32) if m % 2 else None
        more = np.zeros(n) if bias is None else bias
        with xs.no_grad():
            y = F.dense_4bit(xs.Tensor(be.to_device(x)), weight, None if bias is None else xs.Tensor(be.to_device(bias))).numpy()
        assert y.shape == (m, n)
        x = x.astype(np.float64)
        assert np.all(np.abs(y - (x @ w + more)) <= _tolerance(x, w, group) + EPS * np.abs(more)), m
        q = rng.integers(-127, 128, (m, k)).astype(np.int8)
        s = np.exp(rng.standard_normal(m)).astype(np.float32)
        with xs.no_grad():
            y = F.dense_4bit(xs.Tensor(be.to_device(q)), weight, None if bias is None else xs.Tensor(be.to_device(bias)),
                             scale=xs.Tensor(be.to_device(s))).numpy()
        x = q * s[:, None].astype(np.float64)
        assert np.all(np.abs(y - (x @ w + more)) <= _tolerance(x, w, group, True) + EPS * np.abs(more)), m


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("k,n", [(1500, 4100), (3000, 4130), (5000, 4150), (7500, 4110)])
def test_products_of_more_tiles_than_compute_units(k, n, group):
    test_products(k, n, group)


@pytest.mark.parametrize("m", [1, 3, 8, 40])
def test_rows_are_their_own(m):
    """Rows of very different sizes, zeros, the largest and smallest values, infinities and NaN: none changes another row."""
    rng = np.random.default_rng(m)
    k, n = 700, 50
    weight, w = _weight(rng, k, n, 64)
    x = rng.standard_normal((m, k)).astype(np.float32)
    bias = np.zeros(n, np.float32)
    run = lambda a: F.dense_4bit(xs.Tensor(be.to_device(a)), weight, xs.Tensor(be.to_device(bias))).numpy()  # noqa: E731
    with xs.no_grad():
        plain = run(x)
        for value in (np.inf, -np.inf, np.nan, 3e38, 0.0, 1e-42):
            y = x.copy()
            y[0] = 0 if value == 0 else y[0]
            y[0, 5] = value
            got = run(y)
            assert np.array_equal(got[1:], plain[1:])
            with np.errstate(invalid='ignore', over='ignore'):
                want = y[:1].astype(np.float64) @ w
                if abs(value) == np.inf or value != value:
                    assert np.array_equal(np.isnan(got[0]), np.isnan(want[0])) and np.array_equal(got[0][~np.isnan(got[0])], want[0][~np.isnan(want[0])])
                else:
                    # 2^-28 of the row's largest value where it leaves the others below float16
                    assert np.all(np.abs(got[0] - want[0]) <= _tolerance(y[:1].astype(np.float64), w, 64)[0])
        for size in (2.0 ** 100, 2.0 ** -100, 2.0 ** -120):
            y = x * np.float32(size)
            assert np.all(np.abs(run(y) - y.astype(np.float64) @ w) <= _tolerance(y.astype(np.float64), w, 64))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("k,n", [(1, 1), (33, 5), (128, 16), (300, 37), (1000, 64)])
def test_packing(k, n, group):
    rng = np.random.default_rng(k)
    w = (rng.standard_normal((k, n)) * np.exp(rng.standard_normal(n))).astype(np.float32)
    w[:, 0] = 0                                      # an output without weights
    w[k // 2:, n // 2] = 0
    weight = Weight4Bit.quantize(xs.Tensor(w), group)
    numbers, scales = quantize(w, group)
    codes, padded = pack(numbers, scales, group)
    assert np.array_equal(weight.scales.numpy(), padded) and np.array_equal(weight.codes.numpy(), codes)
    back = weight.dequantize().numpy()
    assert np.array_equal(back, values(numbers, scales, group).astype(np.float32))
    # half a step, the scale's own rounding over eight steps, and the end that has no number 8
    step = np.repeat(np.abs(scales.astype(np.float64)), group, 0)[:k]
    assert np.all(np.abs(back - w) <= step * (1 + 8 * 2.0 ** -10))


def test_no_memory_around_the_result_is_written():
    rng = np.random.default_rng(6)
    for m, k, n in ((1, 100, 5), (3, 300, 17), (20, 128, 33)):
        weight, w = _weight(rng, k, n, 32)
        x = rng.standard_normal((m, k)).astype(np.float32)
        around = be.to_device(np.full(m * n + 20, 9, np.float32))
        inside = around.leading(10, 10 + m * n).reshape(m, n)
        weight.product(be.to_device(x), out=inside)
        got = around.numpy()
        assert np.all(got[:10] == 9) and np.all(got[-10:] == 9)
        assert np.all(np.abs(got[10:-10].reshape(m, n) - x.astype(np.float64) @ w) <= _tolerance(x.astype(np.float64), w, 32))


def test_higher_dimensions_host_tensors_and_recorded_products():
    rng = np.random.default_rng(7)
    weight, w = _weight(rng, 200, 30, 64)
    x = rng.standard_normal((2, 3, 200)).astype(np.float32)
    with xs.no_grad():
        y = F.dense_4bit(xs.Tensor(be.to_device(x)), weight).numpy()
        host = F.dense_4bit(xs.Tensor(x.astype(np.float64)), weight)
    assert y.shape == (2, 3, 30) and host.eval.dtype == np.float64 and np.array_equal(host.eval, y)
    xs.GLOBAL.INPUTS = None
    for m in (1, 40):
        a = be.to_device(rng.standard_normal((m, 200)).astype(np.float32))
        with xs.no_grad():
            graph = xs.StepGraph()
            with graph.capture():
                out = F.dense_4bit(xs.Tensor(a), weight)
            for _ in range(4):
                a.set(rng.standard_normal((m, 200)).astype(np.float32))
                graph.replay()
                recorded = out.numpy()
                assert np.array_equal(recorded, F.dense_4bit(xs.Tensor(a), weight).numpy())
                be.zeros((999,)).numpy()


def test_two_recordings_and_eager_calls_share_a_workspace():
    rng = np.random.default_rng(11)
    weight, _ = _weight(rng, 700, 300, 32)
    inputs = [be.empty((m, 700)) for m in (100, 300, 500)]

    def fill():
        for a in inputs:
            a.set(rng.standard_normal(a.shape).astype(np.float32))

    with xs.no_grad():
        graphs, outs = [], []
        for a in inputs[:2]:                         # the second recording finds the first one's workspace too small
            a.set(np.zeros(a.shape, np.float32))
            graphs.append(xs.StepGraph())
            with graphs[-1].capture():
                outs.append(F.dense_4bit(xs.Tensor(a), weight))
        for turn in range(4):
            fill()
            for i in ((0, 1), (1, 0), (0, 1), (1,))[turn]:
                graphs[i].replay()
                if turn == 1:                        # a larger one between two replays
                    F.dense_4bit(xs.Tensor(inputs[2]), weight)
                recorded = outs[i].numpy()
                assert np.array_equal(recorded, F.dense_4bit(xs.Tensor(inputs[i]), weight).numpy())
            if turn == 2:
                graphs[0].close()


def test_a_trained_network_is_served_with_packed_weights(tmp_path):
    """Dense -> norm -> ReLU -> Dense, packed: the logits are those of the dequantised weights; a checkpoint keeps them."""
    np.random.seed(3)
    xs.GLOBAL.USE_CUDA = True
    x, y = np.random.randn(40, 20).astype(np.float32), np.random.randint(0, 4, (40,))
    net = Sequential(Dense(48, activation='tanh', input_shape=(20,)), RMSNormalization(), ReLU(), Dense(4))
    net.compile('adamw', 'cross_entropy', lr=0.01)
    net.fit(x, y, batch_size=16, epochs=3, verbose=0)
    packed = [Dense4Bit.from_dense(l, 32) if isinstance(l, Dense) else l for l in net._graph]
    small = Sequential(*packed)
    small.compile('sgd', 'cross_entropy')
    got = small.predict(x, batch_size=16).numpy()
    small.save(str(tmp_path / 'small'))
    again = Sequential()
    again.load(str(tmp_path / 'small.pkl'))
    assert np.array_equal(again.predict(x, batch_size=16).numpy(), got)
    w1, w2 = (packed[i].weight.dequantize().numpy().astype(np.float64) for i in (0, 3))
    b1, b2 = (packed[i].bias.numpy().reshape(-1).astype(np.float64) for i in (0, 3))
    h = np.tanh(x @ w1 + b1)
    h = h / np.sqrt((h * h).mean(1, keepdims=True) + 1e-6) * net._graph[1].parameters()[0].numpy()
    want = np.maximum(h, 0) @ w2 + b2
    # some 300 roundings of values of one, in sums of 48 terms
    assert np.linalg.norm(got - want) <= 300 * EPS * np.linalg.norm(np.abs(h) @ np.abs(w2))
    with pytest.raises(NotImplementedError):
        small.fit(x, y, batch_size=16, epochs=1, verbose=0)


def test_one_request_through_norm_and_packed_layers():
    """Stream + branch -> norm in 8 bits -> packed layer -> ReLU -> stream: the run of a residual network that serves."""
    rng = np.random.default_rng(8)
    for m in (1, 5, 20):
        d, layers = 256, []
        for _ in range(3):
            layers.append((_weight(rng, d, d, 64), rng.standard_normal(d).astype(np.float32)))
        branch, stream = rng.standard_normal((2, m, d)).astype(np.float32)
        b, s = xs.Tensor(be.to_device(branch)), xs.Tensor(be.to_device(stream))
        with xs.no_grad():
            for (weight, _), gamma in layers:
                q, scale, s = F.rms_norm_8bit(b, xs.Tensor(be.to_device(gamma)), s)
                b = F.relu(F.dense_4bit(q, weight, scale=scale))
                # each layer from what the last one gave: numbers exactly, products to their roundings
                stream = branch + stream
                assert np.array_equal(s.numpy(), stream)
                w = stream.astype(np.float64)
                y = w / np.sqrt((w * w).mean(1, keepdims=True) + 1e-6) * gamma
                step = np.abs(y).max(1, keepdims=True) / 127
                numbers = np.rint(y / step)
                assert np.array_equal(q.numpy(), numbers)
                want = np.maximum(numbers * step @ values_of(weight), 0)
                assert np.all(np.abs(b.numpy() - want) <= _tolerance(numbers * step, values_of(weight), 64, True))
                branch = b.numpy()
                xs.GLOBAL.INPUTS = None


def test_one_layer_twice_in_a_forward():
    rng = np.random.default_rng(10)
    weight, w = _weight(rng, 200, 200, 64)
    layer, x = Dense4Bit(weight), rng.standard_normal((70, 200)).astype(np.float32)
    with xs.no_grad():
        first = layer(xs.Tensor(be.to_device(x)))
        second = layer(first)
        again = F.dense_4bit(first, weight)
    assert first is not second and np.array_equal(second.numpy(), again.numpy())
    assert np.all(np.abs(first.numpy() - x.astype(np.float64) @ w) <= _tolerance(x.astype(np.float64), w, 64))


def values_of(weight):
    return weight.dequantize().numpy().astype(np.float64)


def test_refusals():
    rng = np.random.default_rng(9)
    weight, _ = _weight(rng, 64, 32, 32)
    x, q, s = be.to_device(np.ones((2, 64), np.float32)), be.to_device(np.ones((2, 64), np.int8)), be.to_device(np.ones(2, np.float32))
    square, over = _weight(rng, 64, 64, 32)[0], be.zeros((4, 64))
    t = xs.Tensor
    with xs.no_grad():
        for call in (lambda: F.dense_4bit(t(q), weight), lambda: F.dense_4bit(t(x), weight, scale=t(s)), lambda: F.dense_4bit(t(x.reshape(4, 32)), weight),
                     lambda: F.dense_4bit(t(q), weight, scale=t(s.leading(0, 1))), lambda: F.dense_4bit(t(x), weight, t(s)),
                     lambda: weight.product(x, out=be.empty((2, 31))), lambda: square.product(over.leading(0, 2), out=over.leading(1, 3)), lambda: Weight4Bit(weight.codes, weight.scales, 64, 32, 64),
                     lambda: Weight4Bit(weight.codes, weight.scales, 64, 33, 32), lambda: Weight4Bit.quantize(x, 48), lambda: Weight4Bit.quantize(s, 32),
                     lambda: Weight4Bit.quantize(be.empty((0, 4)), 32), lambda: Dense4Bit.from_dense(Dense(3)), lambda: Dense4Bit(x)):
            with pytest.raises(ValueError):
                call()
        assert F.dense_4bit(t(be.empty((0, 64))), weight).eval.shape == (0, 32)
    with pytest.raises(NotImplementedError):
        F.dense_4bit(t(x, requires_grad=True), weight)
    need = be.lib.raw("xsmi_dense_4bit_workspace_bytes")
    assert need(1, 64, 32, 32) == 0 and need(200, 64, 32, 32) > 0 and need(1 << 21, 64, 32, 32) == 0 and need(200, 64, 32, 16) == 0
    y = be.empty((200, 32))
    big = be.to_device(np.ones((200, 64), np.float32))
    for ws, size, codes in ((None, 0, weight.codes.ptr), (y.ptr, 16, weight.codes.ptr), (None, 0, None), (None, 0, weight.codes.ptr + 4)):
        with pytest.raises(ValueError):
            be.lib.call("xsmi_dense_4bit", big.ptr, None, codes, weight.scales.ptr, None, y.ptr, 200, 64, 32, 32, ws, size)
