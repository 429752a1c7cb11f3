"""The operators of wide residual networks of dense layers -- their normalisation, their optimizer step and the products
with their packed weights -- as cases that can be timed and compared.

A case is a dict of plain values; its ``"kind"`` names the operator:

``adamw``   one AdamW step over all parameters of a network, moments held in 32 or in 8 bits: ``optim.AdamW.step``
``norm``    root-mean-square normalisation of rows, with or without the addition of a residual before it, forward and
            backward: ``nn.functional.rms_norm`` and ``Tensor.backward``
``dense4``  rows times a weight held in 4 bits with a scale for each group of inputs: ``nn.functional.dense_4bit``
``serve``   residual addition, normalisation, rows rounded to 8 bits, their product with a 4-bit weight: one layer of a
            network that answers requests: ``nn.functional.rms_norm_8bit`` and ``nn.functional.dense_4bit``

``own = False`` computes them with elementary torch operations; ``own = True`` calls this repository's package, on arrays
of the package that hold the same values.

Formats that both sides read (the package's header describes them too):

*4-bit weights* of K inputs and N outputs: inputs are padded to a multiple of 128, outputs to one of 16.  ``codes`` is
(outputs / 16, inputs / 128, 64, 16) bytes: lane l of chunk c of tile t holds output 16 t + l % 16; its byte 4 j + b holds
inputs 128 c + 32 j + 8 (l // 16) + 2 b (low four bits) and the one after it (high four bits), each a two's complement
number in -8 .. 7.  ``scales`` is (inputs / group, outputs) float16; a weight is number times scale.

*8-bit moments*: blocks of 256 elements share an exponent byte E, that of the block's largest value (at least 48 for the
first moment, 64 for the second; 255: the block has a value of 2^127 or more, or none that is finite).  A code holds the
exponent and the three leading bits of the fraction: with D = 14 (first moment: a sign bit and seven bits) or 30 (second
moment: eight bits), code k > 0 is the float whose bits are (k - 1 + 8 (E - D)) << 20, and 0 is zero.  Rounding is
stochastic, by 16 bits for each element and moment of a hash of its position, the step and a seed.
"""
import math

import numpy as np
import torch

own = False


# --------------------------------------------------------------------------- the cases
def listed():
    return [
        # The README network's four parameters: 13,570 numbers, a step that is all latency.
        {"name": "adamw_small_net", "kind": "adamw", "net": "small", "width": 0, "layers": 0, "bits": 32, "decay": 0.01},
        # ResNet-18 of the benchmark, its filters, norms and classifier: 82 tensors from 64 to 2.4 million elements.
        {"name": "adamw_resnet18", "kind": "adamw", "net": "resnet18", "width": 1000, "layers": 0, "bits": 32, "decay": 0.01},
        # The same parameters with both moments in 8 bits.
        {"name": "adamw8_resnet18", "kind": "adamw", "net": "resnet18", "width": 1000, "layers": 0, "bits": 8, "decay": 0.01},
        # Eight square dense layers of 4096 with biases and norms: 134 million elements, all bandwidth.
        {"name": "adamw8_dense_4096", "kind": "adamw", "net": "dense", "width": 4096, "layers": 8, "bits": 8, "decay": 0.1},
        # A training batch of 32 feature vectors of 512, what ResNet-18 hands its classifier: latency.
        {"name": "norm_32x512", "kind": "norm", "rows": 32, "cols": 512, "residual": False},
        # The middle of a wide residual network in training: 16384 rows of 4096 and their residual stream.
        {"name": "norm_16384x4096", "kind": "norm", "rows": 16384, "cols": 4096, "residual": True},
        # No size is a round one.
        {"name": "norm_ragged_1021x2731", "kind": "norm", "rows": 1021, "cols": 2731, "residual": True},
        # The classifier of ResNet-18 for one image at a time.
        {"name": "dense4_1x512_1000", "kind": "dense4", "rows": 1, "inputs": 512, "outputs": 1000, "group": 64, "bias": True},
        # One row through a square layer: every weight is read for one product.
        {"name": "dense4_1x8192_8192", "kind": "dense4", "rows": 1, "inputs": 8192, "outputs": 8192, "group": 128, "bias": False},
        # predict() over a batch: each weight serves 200 rows.
        {"name": "dense4_200x4096_8192", "kind": "dense4", "rows": 200, "inputs": 4096, "outputs": 8192, "group": 128, "bias": True},
        # One request through the norm and the layer behind it.
        {"name": "serve_1x4096_16384", "kind": "serve", "rows": 1, "inputs": 4096, "outputs": 16384, "group": 128},
        # Requests that wait are answered together; no size is a round one.
        {"name": "serve_ragged_43x5000_7001", "kind": "serve", "rows": 43, "inputs": 5000, "outputs": 7001, "group": 32},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("adamw", "norm", "dense4", "serve"))
    if kind == "adamw":
        net = rng.choice(("small", "resnet18", "dense", "dense", "dense"))
        while True:
            case = {"kind": "adamw", "net": net, "width": {"small": _log_int(rng, 4, 64), "resnet18": _log_int(rng, 10, 1000)}.get(
                net, rng.choice((_log_int(rng, 16, 4096), 64 * _log_int(rng, 1, 64)))), "layers": _log_int(rng, 1, 48) if net == "dense" else 0,
                "bits": rng.choice((32, 8)), "decay": rng.choice((0.0, 0.01, 0.1))}
            if sum(math.prod(s) for s in _shapes(case)) <= 100_000_000:
                return case
    if kind == "norm":
        while True:
            case = {"kind": "norm", "rows": _log_int(rng, 1, 65536), "cols": rng.choice((_log_int(rng, 16, 16384), 64 * _log_int(rng, 1, 256))),
                    "residual": rng.random() < 0.6}
            if case["rows"] * case["cols"] <= 16384 * 4096:
                return case
    rows = rng.choice((1, _log_int(rng, 1, 16), _log_int(rng, 1, 256)))
    while True:
        case = {"kind": kind, "rows": rows, "inputs": rng.choice((_log_int(rng, 1, 16384), 128 * _log_int(rng, 1, 128))),
                "outputs": rng.choice((_log_int(rng, 1, 16384), 16 * _log_int(rng, 4, 1024))), "group": rng.choice((32, 64, 128))}
        if kind == "dense4":
            case["bias"] = rng.random() < 0.5
        if case["inputs"] * case["outputs"] <= 1 << 27:
            return case


def _shapes(case):
    """Of the parameters of the networks that the adamw cases train, in the order of their forward."""
    width = case["width"]
    if case["net"] == "small":                    # 2 x 2 filters on 28 x 28 images, 2 x 2 pooling, ten classes
        filters = width or 8
        return [(filters, 1, 2, 2), (1, filters), (169 * filters, 10), (1, 10)]
    if case["net"] == "dense":                    # width x width layers, each with its bias and its norm's scale
        return [s for _ in range(case["layers"]) for s in ((width, width), (1, width), (width,))]
    shapes = [(64, 3, 7, 7), (1, 64), (64,), (64,)]
    for c_in, c_out in ((64, 64), (64, 64), (64, 128), (128, 128), (128, 256), (256, 256), (256, 512), (512, 512)):
        shapes += [(c_out, c_in, 3, 3), (1, c_out), (c_out,), (c_out,), (c_out, c_out, 3, 3), (1, c_out), (c_out,), (c_out,)]
        if c_in != c_out:
            shapes += [(c_out, c_in, 1, 1), (1, c_out), (c_out,), (c_out,)]
    return shapes + [(512, width), (1, width)]


def _up(n, to):
    return -(-n // to) * to


# --------------------------------------------------------------------------- prepare
LR, BETAS, EPS, NOISE_SEED = 1e-3, (0.9, 0.999), 1e-8, 1234
NORM_EPS = 1e-6


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    state = {"case": dict(case)}
    if case["kind"] == "adamw":
        # The parameters lie in one buffer, each from a multiple of 256 elements on, and so do their gradients.
        shapes = _shapes(case)
        starts = np.cumsum([0] + [_up(math.prod(s), 256) for s in shapes])
        inside = torch.ones(int(starts[-1]), device="cuda")
        for s, a, b in zip(shapes, starts, starts[1:]):
            inside[int(a) + math.prod(s):int(b)] = 0
        # gradients as training has them: each parameter's of another size, a few elements far above the others
        size = torch.exp(1.5 * normal(len(shapes)) - 6).repeat_interleave(torch.from_numpy(np.diff(starts)).cuda())
        grad = normal(int(starts[-1])) * torch.exp(normal(int(starts[-1]))) * size * inside
        state.update(p=normal(int(starts[-1])) * 0.05 * inside, g=grad, shapes=shapes, starts=[int(v) for v in starts], t=0)
        if case["bits"] == 8:
            n = int(starts[-1])
            code = lambda k: torch.zeros(k, dtype=torch.uint8, device="cuda")  # noqa: E731
            state.update(m8=code(n), v8=code(n), me=code(n // 256), ve=code(n // 256))
        else:
            state.update(m=torch.zeros_like(grad), v=torch.zeros_like(grad))
    elif case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        channel = torch.exp(0.5 * normal(cols))           # some channels are larger than others, in every row
        state.update(x=normal(rows, cols) * channel, gamma=1 + 0.2 * normal(cols), dy=normal(rows, cols) * 0.1)
        if case["residual"]:
            state.update(r=normal(rows, cols) * channel * 2, ds=normal(rows, cols) * 0.1)
    else:
        rows, k, n = case["rows"], case["inputs"], case["outputs"]
        channel = torch.exp(0.5 * normal(k))
        state["x"] = normal(rows, k) * channel
        state["codes"], state["scales"] = _pack(normal(n, k) * 0.02, case["group"])
        if case["kind"] == "serve":
            state.update(r=normal(rows, k) * channel * 2, gamma=1 + 0.2 * normal(k))
        elif case["bias"]:
            state["bias"] = normal(n) * 0.1
    if own:
        _handles(state)
    return state


def _pack(w, group):
    """(N, K) weights in 4 bits: a group's value of largest magnitude becomes -8, whatever its sign."""
    n, k = w.shape
    rows, cols = _up(n, 16), _up(k, 128)
    full = torch.zeros(rows, cols, device=w.device)
    full[:n, :k] = w
    groups = full.view(rows, cols // group, group)
    extreme = torch.gather(groups, 2, groups.abs().argmax(2, keepdim=True)).squeeze(2)
    scales = (extreme / -8).half()
    s = scales.float().unsqueeze(2)
    number = torch.where(s == 0, torch.zeros_like(groups), torch.round(groups / torch.where(s == 0, torch.ones_like(s), s)).clamp(-8, 7))
    number = number.to(torch.int32).view(rows // 16, 16, cols // 128, 4, 4, 4, 2) & 15      # tile, output, chunk, j, lane // 16, b, half
    byte = number[..., 0] | number[..., 1] << 4
    codes = byte.permute(0, 2, 4, 1, 3, 5).reshape(rows // 16, cols // 128, 64, 16).to(torch.uint8)
    return codes, scales.t().contiguous()


# --------------------------------------------------------------------------- this repository's package
class _Memory:
    """A device array's memory as torch takes it; torch keeps this object, and so the array, alive with its view."""

    def __init__(self, array):
        self.array = array
        self.__cuda_array_interface__ = {"shape": array.shape, "typestr": array.dtype.str, "data": (array.ptr, False),
                                         "version": 2}


def _view(array):
    return torch.as_tensor(_Memory(array), device="cuda")


def _array(values):
    """A package array with a torch tensor's values."""
    from xshinnosuke_amd import backend as be
    kinds = {torch.float32: np.float32, torch.float16: np.float16, torch.uint8: np.uint8}
    array = be.empty(tuple(values.shape), kinds[values.dtype])
    be.synchronize()                              # whatever used this memory before has ended
    _view(array).copy_(values)
    torch.cuda.synchronize()
    return array


def _handles(state):
    """The state's tensors as the package's tensors, parameters, weights and optimizer."""
    import xshinnosuke_amd as xs
    case = state["case"]
    xs.GLOBAL.USE_CUDA = True
    if case["kind"] == "adamw":
        flat, grads = _array(state.pop("p")), _array(state.pop("g"))
        params = []
        for shape, start in zip(state["shapes"], state["starts"]):
            stop = start + math.prod(shape)
            params.append(xs.Parameter(xs.Tensor(flat.leading(start, stop).reshape(shape), requires_grad=True)))
            params[-1].grad = xs.Tensor(grads.leading(start, stop).reshape(shape))
        for name in ("m", "v", "m8", "v8", "me", "ve"):      # the optimizer makes its own
            state.pop(name, None)
        opt = xs.optim.AdamW(params, lr=LR, betas=BETAS, epsilon=EPS, weight_decay=case["decay"], state_bits=case["bits"], seed=NOISE_SEED)
        state.update(opt=opt, flat=flat, flat_view=_view(flat), views={})
    elif case["kind"] == "norm":
        for name in ("x", "r"):
            if name in state:
                state[name] = xs.Tensor(_array(state[name]), requires_grad=True)
        state["gamma"] = xs.Parameter(xs.Tensor(_array(state["gamma"]), requires_grad=True))
        for name in ("dy", "ds"):
            if name in state:
                state[name] = xs.Tensor(_array(state[name]))
    else:
        state["w"] = xs.nn.Weight4Bit(_array(state.pop("codes")), _array(state.pop("scales")), case["inputs"], case["outputs"], case["group"])
        for name in ("x", "r", "gamma", "bias"):
            if name in state:
                state[name] = xs.Tensor(_array(state[name]))


def _outputs(state, arrays):
    """Torch views of ``arrays``; the views of those that keep their memory from pass to pass are kept."""
    kept = state.setdefault("views", {})
    out = []
    for i, a in enumerate(arrays):
        if i not in kept or kept[i][0] != a.address():
            kept[i] = (a.address(), _view(a))
        out.append(kept[i][1])
    return out


def _run_own(state):
    import xshinnosuke_amd as xs
    F = xs.nn.functional
    case = state["case"]
    if case["kind"] == "adamw":
        state["opt"].step()
        (_, m, v), = state["opt"].moments()
        return [state["flat_view"]] + _outputs(state, [m, v])
    if case["kind"] == "norm":
        x, gamma = state["x"], state["gamma"]
        x.zero_grad()
        gamma.zero_grad()
        if not case["residual"]:
            y = F.rms_norm(x, gamma, epsilon=NORM_EPS)
            out = [y.eval]
            y.backward(state["dy"])
            return _outputs(state, out + [x.grad.eval, gamma.grad.eval])
        r = state["r"]
        r.zero_grad()
        y, s = F.rms_norm(x, gamma, r, epsilon=NORM_EPS)
        out = [y.eval, s.eval]
        s.grad = state["ds"]                      # what the later layers' backward has left on the residual stream
        y.backward(state["dy"])
        return _outputs(state, out + [x.grad.eval, r.grad.eval, gamma.grad.eval])
    with xs.no_grad():
        if case["kind"] == "dense4":
            y = F.dense_4bit(state["x"], state["w"], state.get("bias"))
            out = [y.eval]
        else:
            q, scale, s = F.rms_norm_8bit(state["x"], state["gamma"], state["r"], epsilon=NORM_EPS)
            y = F.dense_4bit(q, state["w"], scale=scale)
            out = [y.eval, s.eval]
    xs.GLOBAL.INPUTS = None
    return _outputs(state, out)


# --------------------------------------------------------------------------- the plain forms
def run(state):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "adamw":
        return _plain_adamw(state)
    if kind == "norm":
        return _plain_norm(state)
    w = _plain_weight(state)
    if kind == "dense4":
        y = state["x"] @ w.t()
        return [y + state["bias"] if "bias" in state else y]
    s = state["x"] + state["r"]
    wide = s.double()                             # a row's 8-bit numbers lie next to a border now and then
    normed = wide * torch.rsqrt((wide * wide).mean(1, keepdim=True) + NORM_EPS) * state["gamma"].double()
    most = normed.abs().amax(1, keepdim=True)
    q = torch.round(normed * (127 / torch.where(most == 0, torch.ones_like(most), most)))
    y = (q.float() @ w.t()) * (most / 127).float()
    return [y, s]


def _plain_weight(state):
    """(N, K) float32 weights from their 4-bit form."""
    case, codes = state["case"], state["codes"].to(torch.int32)
    tiles, chunks = codes.shape[:2]
    number = torch.stack((codes & 15, codes >> 4), 4).view(tiles, chunks, 4, 16, 4, 4, 2)      # tile, chunk, lane // 16, output, j, b, half
    number = number.permute(0, 3, 1, 4, 2, 5, 6).reshape(tiles * 16, chunks * 128)
    number = (number ^ 8) - 8
    scale = state["scales"].float().t().unsqueeze(2)
    w = number.float().view(tiles * 16, -1, case["group"]) * scale
    return w.reshape(tiles * 16, -1)[:case["outputs"], :case["inputs"]]


def _plain_norm(state):
    s = state["x"] + state["r"] if "r" in state else state["x"]
    gamma, dy = state["gamma"], state["dy"]
    rstd = torch.rsqrt((s * s).mean(1, keepdim=True) + NORM_EPS)
    xhat = s * rstd
    y = xhat * gamma
    up = dy * gamma
    dx = rstd * (up - xhat * (up * xhat).mean(1, keepdim=True))
    dgamma = (dy * xhat).sum(0)
    if "r" not in state:
        return [y, dx, dgamma]
    dx = dx + state["ds"]
    return [y, s, dx, dx, dgamma]


def _plain_adamw(state):
    case, p, g = state["case"], state["p"], state["g"]
    state["t"] += 1
    t, (b1, b2) = state["t"], BETAS
    if case["bits"] == 8:
        m, v = _decode(state["m8"], state["me"], 14, True), _decode(state["v8"], state["ve"], 30, False)
    else:
        m, v = state["m"], state["v"]
    # every product and sum is rounded to 32 bits by itself: the 8-bit codes are defined by these values
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * (1 - b2) * g
    p.mul_(1 - LR * case["decay"])
    p.sub_(m * (LR / (1 - b1 ** t)) / (v.sqrt() * (1 / math.sqrt(1 - b2 ** t)) + EPS))
    if case["bits"] == 8:
        noise = _noise(m.numel(), t)
        _encode(m, noise & 0xFFFF, state["m8"], state["me"], 14, 48, True)
        _encode(v, noise >> 16, state["v8"], state["ve"], 30, 64, False)
        return [p, _decode(state["m8"], state["me"], 14, True), _decode(state["v8"], state["ve"], 30, False)]
    state["m"].copy_(m)
    state["v"].copy_(v)
    return [p, state["m"], state["v"]]


_ALL = 0xFFFFFFFF


def _mix(h):
    """A hash of 32-bit numbers, which a 64-bit type holds; the multipliers are fractional bits of the roots of 2 and 3."""
    h = h ^ (h >> 16)
    h = (h * 0x6A09E667) & _ALL
    h = h ^ (h >> 15)
    h = (h * 0xBB67AE85) & _ALL
    return h ^ (h >> 16)


def _noise(n, t):
    key = _mix((NOISE_SEED + t * 0x9E3779B1) & _ALL)
    return _mix((torch.arange(n, device="cuda") * 0x9E3779B1 + key) & _ALL).to(torch.int64)


def _decode(code, exponent, depth, signed):
    k = code.view(-1, 256).to(torch.int32)
    e = exponent.to(torch.int32).unsqueeze(1)
    sign = (k >> 7) << 31 if signed else torch.zeros_like(k)
    k = k & 127 if signed else k
    bits = torch.where(k == 0, torch.zeros_like(k), (k - 1 + 8 * (e - depth)) << 20)
    return torch.where(e == 255, torch.full_like(bits, 0x7FC00000), bits | sign).view(-1).view(torch.float32)


def _encode(x, noise, code, exponent, depth, least, signed):
    bits = x.abs().view(torch.int32).view(-1, 256)
    noise = noise.to(torch.int32).view(-1, 256)
    e = (bits.amax(1, keepdim=True) >> 23).clamp(min=least)
    bad = e >= 254
    floor = ((e - depth) << 23).view(torch.float32)
    k = ((bits + (noise << 4) + 8) >> 20) + 1 - 8 * (e - depth)
    low = (bits.view(torch.float32) > (noise.float() + 0.5) * (2.0 ** -16) * floor).to(torch.int32)
    k = torch.where(bits < ((e - depth) << 23), low, k)
    if signed:
        k = k | ((x.view(-1, 256) < 0).to(torch.int32) << 7)
    code.copy_(torch.where(bad, torch.zeros_like(k), k).view(-1))
    exponent.copy_(torch.where(bad, torch.full_like(e, 255), e).view(-1))


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        # parameters and moments read and written, gradients read; 8-bit moments come back as the numbers they stand for
        return {"bytes": n * (4 * 3 + 8 * 2 if case["bits"] == 32 else 4 * 3 + 2 * 2 + 8), "flops": 15 * n}
    if case["kind"] == "norm":
        n = case["rows"] * case["cols"]
        forward, backward = (16, 20) if case["residual"] else (8, 12)      # x [r] -> y [s]; dy, s [ds] -> dx [dr]
        return {"bytes": n * (forward + backward) + 8 * case["cols"] + 4 * case["rows"], "flops": 16 * n}
    rows, k, n = case["rows"], case["inputs"], case["outputs"]
    weights = k * n // 2 + 2 * n * -(-k // case["group"])
    if case["kind"] == "dense4":
        return {"bytes": weights + 4 * (rows * (k + n) + (n if case["bias"] else 0)), "flops": 2 * rows * k * n}
    return {"bytes": weights + 4 * (rows * (3 * k + n) + k), "flops": 2 * rows * k * n + 12 * rows * k}


# --------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    """What ``run`` returns for these inputs, from the operators' definitions in 64 bits."""
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    f = {k: v.double() for k, v in state.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["kind"] == "adamw":
        return _exact_adamw(case, f["p"], f["g"])
    if case["kind"] == "norm":
        s = f["x"] + f["r"] if "r" in f else f["x"]
        n = s.shape[1]
        root = torch.sqrt(torch.linalg.vector_norm(s, dim=1, keepdim=True) ** 2 / n + NORM_EPS)
        y = s / root * f["gamma"]
        # derivative of s_j / root: the identity over the root, less s s^T over n root^3
        a = f["gamma"] * f["dy"]
        dx = a / root - s * (a * s).sum(1, keepdim=True) / (n * root ** 3)
        dgamma = (f["dy"] * s / root).sum(0)
        return [y, dx, dgamma] if "r" not in f else [y, s, dx + f["ds"], dx + f["ds"], dgamma]
    w = _exact_weight(case, state["codes"], f["scales"])
    if case["kind"] == "dense4":
        y = torch.matmul(f["x"], w)
        return [y if "bias" not in f else y + f["bias"]]
    total = (state["x"] + state["r"]).double()    # the residual stream is held in 32 bits
    root = torch.sqrt(torch.linalg.vector_norm(total, dim=1, keepdim=True) ** 2 / total.shape[1] + NORM_EPS)
    normed = total / root * f["gamma"]
    step = normed.abs().max(1, keepdim=True).values / 127
    number = torch.where(step > 0, torch.round(normed / step), 0.0)
    return [torch.matmul(number * step, w), total]


def _exact_weight(case, codes, scales):
    """(K, N) weights, each looked up at its place in the packed form."""
    k = torch.arange(case["inputs"], device="cuda").unsqueeze(1)
    n = torch.arange(case["outputs"], device="cuda").unsqueeze(0)
    within = k % 128
    lane = 16 * (within % 32 // 8) + n % 16
    byte = codes[n // 16, k // 128, lane, 4 * (within // 32) + within % 8 // 2].to(torch.int16)
    number = torch.where(k % 2 == 1, byte // 16, byte % 16)
    number = torch.where(number > 7, number - 16, number)
    return number.double() * scales[k // case["group"], n]


def _single(x):
    """Rounded to 32 bits, where the definition says so."""
    return x.float().double()


def _exact_adamw(case, p, g):
    """The first step, from moments of zero."""
    b1, b2 = BETAS
    c1, c2 = (float(np.float32(1 - b)) for b in BETAS)
    m, v = (1 - b1) * g, (1 - b2) * g * g
    new = p * (1 - LR * case["decay"]) - LR * (m / (1 - b1)) / (torch.sqrt(v / (1 - b2)) + EPS)
    if case["bits"] == 32:
        return [new, m, v]
    # The 8-bit form of the 32-bit moments: a position on the scale of the code, its whole part and what the noise makes
    # of the rest.
    n = g.numel()
    key = int(_mix(np.int64((NOISE_SEED + 0x9E3779B1) & _ALL)))
    h = _mix((torch.arange(n, device="cuda", dtype=torch.int64) * 0x9E3779B1 + key) & _ALL)
    moments = ((_single(c1 * g), h % 65536, 14, 48), (_single(_single(c2 * g) * g), torch.div(h, 65536, rounding_mode="floor"), 30, 64))
    return [new] + [_exact_code(x, (noise.double() + 0.5) / 65536, depth, least) for x, noise, depth, least in moments]


def _power(e):
    """2 ** e, of whole numbers."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_code(x, noise, depth, least):
    blocks, noise = x.abs().view(-1, 256), noise.view(-1, 256)
    lowest = torch.frexp(blocks.max(1, keepdim=True).values).exponent.clamp(min=least - 126) - 1 - depth
    _, e = torch.frexp(torch.where(blocks == 0, torch.ones_like(blocks), blocks))
    step = _power(torch.maximum(e - 1, lowest) - 3)          # an eighth of the power of two below
    fine = torch.floor(blocks / step + noise) * step
    floor = _power(lowest).expand_as(blocks)
    value = torch.where(blocks < floor, torch.where(blocks / floor > noise, floor, torch.zeros_like(floor)), fine)
    return (torch.sign(x).view(-1, 256) * value).view(-1).float()
