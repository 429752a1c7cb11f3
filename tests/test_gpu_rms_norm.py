"""rms_norm on the device against the formula in 64 bits: forward, backward, 8-bit rows, sizes, extreme rows, wiring."""
import numpy as np
import pytest

import xshinnosuke_amd as xs
from xshinnosuke_amd import backend as be
from xshinnosuke_amd.layers import Dense, ReLU, RMSNormalization
from xshinnosuke_amd.nn import functional as F
from xshinnosuke_amd.nn.models import Module
from xshinnosuke_amd.optim import AdamW

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24                                     # half a step of float32


@pytest.fixture(autouse=True)
def _fresh_state(gpu):
    xs.GLOBAL.INPUTS, xs.GLOBAL.USE_CUDA = None, False
    yield
    xs.GLOBAL.INPUTS, xs.GLOBAL.USE_CUDA = None, False


def _roundings(rows, cols):
    """Roundings that a value can have gone through: a thread adds at most 16 squares, or cols / 1024, one after the other, a
    row's threads meet in at most 6 + 16 further additions, and a dozen products follow."""
    return 16 + cols / 1024 + 22 + 12


def _dev(a, **kw):
    return xs.Tensor(be.to_device(a), **kw)


SIZES = [(1, 1), (5, 1), (3, 2), (7, 3), (1, 4), (33, 5), (17, 63), (1, 64), (5, 65), (130, 127), (4, 256), (9, 257), (3, 1000), (1030, 1024),
         (2, 1025), (2051, 333), (5, 4095), (3, 4096), (2, 4097), (300, 5000), (2, 16383), (1, 16384), (3, 16385), (2, 40001)]


def _case(rng, rows, cols):
    size = np.exp(rng.standard_normal(cols))
    x, r, dy, ds = (rng.standard_normal((rows, cols)).astype(np.float32) for _ in range(4))
    return (x * size).astype(np.float32), (r * size).astype(np.float32), rng.standard_normal(cols).astype(np.float32), dy, ds


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_forward_and_backward(rows, cols, residual):
    rng = np.random.default_rng(rows * 31 + cols)
    x, r, gamma, dy, ds = _case(rng, rows, cols)
    tx, tr, tg = _dev(x, requires_grad=True), _dev(r, requires_grad=True), xs.Parameter(_dev(gamma, requires_grad=True))
    before = [rng.standard_normal(a.shape).astype(np.float32) if rows % 2 else None for a in (x, r, gamma)]
    for t, b in zip((tx, tr, tg), before):           # gradients are added to, or written where there is nothing yet
        if b is not None:
            t.grad = _dev(b)
    eps = 1e-3
    if residual:
        y, s = F.rms_norm(tx, tg, tr, epsilon=eps)
        assert np.array_equal(s.numpy(), x + r)
        s.grad = _dev(ds)
    else:
        y = F.rms_norm(tx, tg, epsilon=eps)
    got = y.numpy()
    y.backward(_dev(dy))
    n = _roundings(rows, cols)
    s64 = (x + r if residual else x).astype(np.float64)
    rstd = 1 / np.sqrt((s64 ** 2).mean(1, keepdims=True) + eps)
    xhat, a = s64 * rstd, gamma.astype(np.float64) * dy
    assert np.all(np.abs(got - xhat * gamma) <= n * EPS * np.abs(xhat * gamma) + 1e-37)
    want = rstd * (a - xhat * (a * xhat).mean(1, keepdims=True))
    most = rstd * (np.abs(a) + np.abs(xhat) * np.abs(a * xhat).mean(1, keepdims=True))
    if residual:
        want, most = want + ds, most + np.abs(ds)
    for t, b in zip((tx, tr) if residual else (tx,), before):
        w, m = (want, most) if b is None else (want + b, most + np.abs(b))
        assert np.all(np.abs(t.grad.numpy() - w) <= 2 * n * EPS * m)
    want, most = (dy * xhat).sum(0), np.abs(dy * xhat).sum(0)
    if before[2] is not None:
        want, most = want + before[2], most + np.abs(before[2])
    # terms added one after the other: a workgroup's rows, then sixteenths of up to 16384 lots, then sixteen
    assert np.all(np.abs(tg.grad.numpy() - want) <= (n + rows / 256 + min(rows, 16384) / 16 + 18) * EPS * most)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", [(40003, 13), (20001, 60), (9000, 200), (9001, 300), (6001, 700), (513, 1024), (600, 5000)])
def test_forward_and_backward_of_many_rows(rows, cols, residual):
    test_forward_and_backward(rows, cols, residual)


@pytest.mark.parametrize("rows,cols", [(70_000, 240), (17_000, 1000), (4_100, 4000), (2_100, 8000)])
def test_forward_and_backward_of_operands_that_are_streamed(rows, cols):
    test_forward_and_backward(rows, cols, True)


@pytest.mark.parametrize("rows,cols", SIZES)
def test_rows_in_eight_bits(rows, cols):
    rng = np.random.default_rng(rows * 37 + cols)
    x, r, gamma, _, _ = _case(rng, rows, cols)
    x[0], r[0] = 0, 0                                # a row without anything
    with xs.no_grad():
        q, scale, s = F.rms_norm_8bit(_dev(x), _dev(gamma), _dev(r), epsilon=1e-6)
        q1, scale1 = F.rms_norm_8bit(_dev(x), _dev(gamma), epsilon=1e-6)
    assert np.array_equal(s.numpy(), x + r) and q.eval.dtype == np.int8
    for base, numbers, steps in ((x + r, q, scale), (x, q1, scale1)):
        w = base.astype(np.float64)
        y = w / np.sqrt((w ** 2).mean(1, keepdims=True) + 1e-6) * gamma
        most = np.abs(y).max(1, keepdims=True)
        assert np.array_equal(numbers.numpy(), np.rint(y * (127 / np.where(most > 0, most, 1))))
        np.testing.assert_allclose(steps.numpy(), most[:, 0] / 127, rtol=1.01 * EPS)
        assert np.all(np.abs(numbers.numpy() * steps.numpy()[:, None].astype(np.float64) - y) <= most / 254 * (1 + 1e-5))


@pytest.mark.parametrize("cols", [3, 200, 1000, 5000, 20000])
def test_rows_that_are_not_finite_stay_by_themselves(cols):
    rng = np.random.default_rng(cols)
    x, _, gamma, dy, _ = _case(rng, 6, cols)
    gamma = np.abs(gamma) + 0.1
    clean = x.copy()
    x[1, 0], x[2, cols - 1], x[3], x[4] = np.nan, np.inf, 0, 1e-30
    tx, tg = _dev(x, requires_grad=True), xs.Parameter(_dev(gamma.astype(np.float32), requires_grad=True))
    y = F.rms_norm(tx, tg)
    got = y.numpy()
    y.backward(_dev(dy))
    assert np.isnan(got[1]).all() and np.isnan(got[2, cols - 1]) and not got[3].any()
    assert np.isfinite(got[[0, 3, 4, 5]]).all() and np.isfinite(tx.grad.numpy()[[0, 3, 4, 5]]).all()
    alone = F.rms_norm(_dev(clean[[0, 5]]), tg)
    assert np.array_equal(got[[0, 5]], alone.numpy())
    xs.GLOBAL.INPUTS = None
    with xs.no_grad():
        q, scale = F.rms_norm_8bit(_dev(x), _dev(gamma.astype(np.float32)))
    assert np.isnan(scale.numpy()[1:3]).all() and not q.numpy()[1:4].any() and scale.numpy()[3] == 0
    assert np.abs(q.numpy()[[0, 4, 5]]).max(1).tolist() == [127] * 3


def test_memory_around_the_rows_stays_as_it_was():
    """Rows of an odd length that start and end inside a buffer."""
    rng = np.random.default_rng(5)
    for cols in (3, 129, 1001):
        rows, pad = 5, 7
        x, _, gamma, dy, _ = _case(rng, rows, cols)
        buffers = [be.to_device(np.full(rows * cols + 2 * pad, 9, np.float32)) for _ in range(3)]
        inside = [b.leading(pad, pad + rows * cols).reshape(rows, cols) for b in buffers]
        inside[0].set(x)
        y, s, rstd = be.kernels.rms_norm_fwd(inside[0], be.to_device(gamma), 1e-6, y=inside[1])
        inside[2].set(np.zeros_like(x))
        be.kernels.rms_norm_bwd(be.to_device(dy), s, rstd, be.to_device(gamma), dx1=inside[2])
        for b in buffers:
            full = b.numpy()
            assert np.all(full[:pad] == 9) and np.all(full[-pad:] == 9) and not np.any(full[pad:-pad] == 9)


@pytest.mark.parametrize("both", [False, True])
def test_backward_in_one_pass_equals_that_in_steps(both):
    """The residual stream through two norms; a retained sum takes the steps apart."""
    rng = np.random.default_rng(9)
    x, r, gamma, dy, _ = _case(rng, 40, 96)

    def run(retain):
        tx, tr, g1, g2 = _dev(x, requires_grad=True), _dev(r, requires_grad=both), *(xs.Parameter(_dev(gamma, requires_grad=True)) for _ in range(2))
        y1, s1 = F.rms_norm(tx, g1, tr)
        s1.retain_grad(retain)
        y2, s2 = F.rms_norm(y1, g2, s1)
        s2.retain_grad(retain)
        y2.backward(_dev(dy))
        if retain:
            assert s1.grad is not None
        return [t.grad.numpy() for t in (tx, g1, g2) + ((tr,) if both else ())]

    for a, b in zip(run(False), run(True)):
        # the same terms in another order: four roundings of terms below the largest gradient
        assert np.abs(a - b).max() <= 4 * 2 * EPS * max(1, np.abs(b).max())


def test_a_gradient_of_the_sum_that_was_set_on_the_host():
    rng = np.random.default_rng(16)
    x, r, gamma, dy, ds = _case(rng, 5, 70)
    grads = []
    for place in (be.to_device, np.array):
        tx, tr, tg = _dev(x, requires_grad=True), _dev(r, requires_grad=True), xs.Parameter(_dev(gamma, requires_grad=True))
        y, s = F.rms_norm(tx, tg, tr)
        s.grad = xs.Tensor(place(ds))
        y.backward(_dev(dy))
        grads.append([t.grad.numpy() for t in (tx, tr, tg)])
        xs.GLOBAL.INPUTS = None
    assert all(np.array_equal(a, b) for a, b in zip(*grads))


def test_one_tensor_as_both_addends():
    rng = np.random.default_rng(10)
    x, _, gamma, dy, _ = _case(rng, 5, 70)
    tx, tg = _dev(x, requires_grad=True), xs.Parameter(_dev(gamma, requires_grad=True))
    y, _ = F.rms_norm(tx, tg, tx)
    y.backward(_dev(dy))
    ux, ug = xs.Tensor(x.astype(np.float64), requires_grad=True), xs.Parameter(xs.Tensor(gamma.astype(np.float64), requires_grad=True))
    xs.GLOBAL.INPUTS = None
    y, _ = F.rms_norm(ux, ug, ux)
    y.backward(xs.Tensor(dy.astype(np.float64)))
    for a, b in ((tx, ux), (tg, ug)):
        assert np.abs(a.grad.numpy() - b.grad.numpy()).max() <= 100 * EPS * np.abs(b.grad.numpy()).max()


def test_several_normalisations_of_one_sum():
    """The stream that one norm returns goes through another norm of its own, and on."""
    rng = np.random.default_rng(13)
    x, r, gamma, dy, _ = _case(rng, 6, 50)
    grads = []
    for device in (True, False):
        tensor = (lambda a, **k: _dev(a, **k)) if device else (lambda a, **k: xs.Tensor(a.astype(np.float64), **k))
        tx, tr = tensor(x, requires_grad=True), tensor(r, requires_grad=True)
        gammas = [xs.Parameter(tensor(gamma + k, requires_grad=True)) for k in range(3)]
        y, s = F.rms_norm(tx, gammas[0], tr)
        z = F.rms_norm(s, gammas[1]) + F.rms_norm(s, gammas[2])
        (z + y + s).backward(tensor(dy))
        grads.append([t.grad.numpy() for t in (tx, tr, *gammas)])
    for a, b in zip(*grads):
        assert np.abs(a - b).max() <= 4 * _roundings(6, 50) * EPS * np.abs(b).max()


def test_more_rows_than_one_launch_takes():
    rng = np.random.default_rng(14)
    rows = (1 << 21) + 5
    x, r, gamma, _, _ = _case(rng, rows, 2)
    with xs.no_grad():
        y, s = F.rms_norm(_dev(x), _dev(gamma), _dev(r))
        q, scale, _ = F.rms_norm_8bit(_dev(x), _dev(gamma), _dev(r))
    w = (x + r).astype(np.float64)
    want = w / np.sqrt((w * w).mean(1, keepdims=True) + 1e-6) * gamma
    assert np.array_equal(s.numpy(), x + r) and np.all(np.abs(y.numpy() - want) <= _roundings(1, 2) * EPS * np.abs(want))
    most = np.abs(want).max(1)
    assert np.all(np.abs(q.numpy() - want * (127 / most)[:, None]) <= 0.5 + 1e-9) and np.allclose(scale.numpy(), most / 127, rtol=2 * EPS)


def test_rows_in_eight_bits_past_the_threads_of_one_launch_and_offsets_of_32_bits():
    rng = np.random.default_rng(15)
    rows, cols = (1 << 24) + 3, 257
    gamma, row = (rng.standard_normal(cols).astype(np.float32) for _ in range(2))
    x = be.zeros((rows, cols))
    at = (0, 1 << 21, rows - 1)
    for i in at:
        x.leading(i, i + 1).set(row[None])
    with xs.no_grad():
        q, scale = F.rms_norm_8bit(xs.Tensor(x), _dev(gamma))
    w = row.astype(np.float64)
    want = w / np.sqrt((w * w).mean() + 1e-6) * gamma
    most = np.abs(want).max()
    scales = scale.numpy()
    assert np.array_equal(np.flatnonzero(scales), at) and np.allclose(scales[list(at)], most / 127, rtol=2 * EPS, atol=0)
    for i in at:
        assert np.all(np.abs(q.eval.leading(i, i + 1).numpy()[0] - want * (127 / most)) <= 0.5 + 1e-9)
    assert not q.eval.leading(rows - 3, rows - 1).numpy().any()
    del x, q, scale
    be.release_cached_memory()


def test_only_the_scales_or_only_the_rows_want_a_gradient():
    rng = np.random.default_rng(11)
    x, r, gamma, dy, _ = _case(rng, 5, 70)
    full = None
    for rows, scales in ((True, True), (True, False), (False, True)):
        tx, tr, tg = _dev(x, requires_grad=rows), _dev(r), xs.Parameter(_dev(gamma, requires_grad=scales))
        y, s = F.rms_norm(tx, tg, tr)
        y.backward(_dev(dy))
        got = [t.grad.numpy() if t.grad is not None else None for t in (tx, tg)]
        full = full or got
        assert (got[0] is not None) == rows and (got[1] is not None) == scales and tr.grad is None
        for a, b in zip(got, full):
            assert a is None or np.array_equal(a, b)


class _Block(Module):
    def __init__(self, width):
        super().__init__()
        self.norm, self.dense, self.act = RMSNormalization(), Dense(width, kernel_initializer='he_normal'), ReLU()

    def forward(self, x, residual=None):
        y, s = (self.norm(x), x) if residual is None else self.norm(x, residual)
        return self.act(self.dense(y)), s


class _Net(Module):
    """A residual network of dense layers: each block's output is added to the stream by the next norm."""

    def __init__(self, width, classes, depth):
        super().__init__()
        self.blocks = [_Block(width) for _ in range(depth)]
        self.norm, self.head = RMSNormalization(), Dense(classes, kernel_initializer='he_normal')

    def forward(self, x):
        x, s = self.blocks[0](x)
        for b in self.blocks[1:]:
            x, s = b(x, s)
        y, _ = self.norm(x, s)
        return self.head(y)


@pytest.mark.parametrize("bits", [32, 8])
def test_residual_network_trains_the_same_launch_by_launch_and_recorded(bits):
    """Gradients of a residual network equal the host's in 64 bits, and a recorded AdamW step equals the eager one."""
    rng = np.random.default_rng(12)
    x, labels = rng.standard_normal((24, 40)).astype(np.float32), rng.integers(0, 5, (24,))

    def build(device):
        np.random.seed(4)
        net = _Net(40, 5, 3)
        if device:
            net.to('cuda')
        tx = xs.Tensor(x).to('cuda') if device else xs.Tensor(x.astype(np.float64))
        ty = xs.Tensor(labels).to('cuda') if device else xs.Tensor(labels)
        with xs.no_grad():
            net(tx)
        xs.GLOBAL.INPUTS = None
        params = [p for b in net.blocks for l in (b.norm, b.dense) for p in l.parameters()] + net.norm.parameters() + net.head.parameters()
        return net, tx, ty, params

    def step(net, tx, ty, opt):
        opt.zero_grad()
        loss = xs.nn.CrossEntropyLoss()(net(tx), ty)
        loss.backward()
        opt.step()
        return loss

    grads = []
    for device in (False, True):
        xs.GLOBAL.USE_CUDA = False
        net, tx, ty, params = build(device)
        loss = xs.nn.CrossEntropyLoss()(net(tx), ty)
        loss.backward()
        grads.append([p.grad.numpy() for p in params])
    for a, b in zip(*grads):
        # a chain of four products of 40 terms and four norms, each of below 50 roundings
        assert np.linalg.norm(b - a) <= 8 * 50 * EPS * max(np.linalg.norm(a), 1e-3)
    ends = []
    for recorded in (False, True):
        net, tx, ty, params = build(True)
        opt, graph = AdamW(params, lr=0.01, state_bits=bits), None
        for k in range(6):
            if recorded and k >= 2:
                if graph is None:
                    graph = be.StepGraph()
                    with graph.capture():
                        loss = step(net, tx, ty, opt)
                graph.replay()
            else:
                loss = step(net, tx, ty, opt)
            loss.item()
            be.zeros((512,)).numpy()
        ends.append([p.numpy() for p in params])
    for a, b in zip(*ends):
        assert np.array_equal(a, b)


def test_refusals():
    x, g = be.to_device(np.ones((4, 8), np.float32)), be.to_device(np.ones(8, np.float32))
    K = be.kernels
    for call in (lambda: K.rms_norm_fwd(x, x.leading(0, 1).reshape(-1).leading(0, 4), 1e-6), lambda: K.rms_norm_fwd(x, g, 1e-6, residual=g),
                 lambda: K.rms_norm_fwd(x, g, -1.0), lambda: K.rms_norm_int8(x, g, float('nan')), lambda: K.rms_norm_fwd(be.empty((4, 8), np.int32), g, 1e-6),
                 lambda: K.rms_norm_bwd(g, x, g.leading(0, 4), g), lambda: K.rms_norm_bwd(x, x, g, g)):
        with pytest.raises(ValueError):
            call()
    raw = lambda *a: be.lib.call("xsmi_rms_norm_bwd", *a)  # noqa: E731
    p = x.ptr
    for bad in ((p, p, p, p, None, p, 0.5, None, 0.0, None, 0.0, 4, 8, None, 0), (p, p, p, p, None, None, 0.0, p, 0.0, None, 0.0, 4, 8, None, 0),
                (p, p, p, p, None, p, 0.0, p, 0.0, None, 0.0, 4, 8, None, 0), (p, p, p, p, None, p, 0.0, None, 0.0, p, 0.0, 4096, 256, p, 16),
                (p, p, p, p, None, p, 0.0, None, 0.0, None, 0.0, 4, 0, None, 0), (p, None, p, p, None, p, 0.0, None, 0.0, None, 0.0, 4, 8, None, 0)):
        with pytest.raises(ValueError):
            raw(*bad)
    with pytest.raises(ValueError):
        be.lib.call("xsmi_rms_norm_fwd", p, p, p, None, p, None, 4, 8, 1e-6)
    empty = F.rms_norm(xs.Tensor(be.empty((0, 8))), xs.Tensor(g))
    assert empty.eval.shape == (0, 8)
