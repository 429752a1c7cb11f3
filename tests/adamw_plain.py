"""AdamW written out in NumPy: the parameters in 64 bits, the 8-bit moments from their definition in include/xsmi355.h."""
import numpy as np

STRIDE = 0x9E3779B1
F = np.float32


def mix(h):
    h = np.asarray(h, np.uint32)
    with np.errstate(over='ignore'):
        h = h ^ (h >> np.uint32(16))
        h = h * np.uint32(0x6A09E667)
        h = h ^ (h >> np.uint32(15))
        h = h * np.uint32(0xBB67AE85)
        return h ^ (h >> np.uint32(16))


def noise(start, n, t, seed):
    """(first moment's, second moment's) 16 bits of noise for the elements at places start .. start + n - 1."""
    place = np.arange(start, start + n, dtype=np.uint64)
    key = mix((seed + t * STRIDE) & 0xFFFFFFFF)
    with np.errstate(over='ignore'):
        h = mix((place & np.uint64(0xFFFFFFFF)).astype(np.uint32) * np.uint32(STRIDE) + key
                + (place >> np.uint64(32)).astype(np.uint32) * np.uint32(0x510E527F))
    return (h & np.uint32(0xFFFF)).astype(np.int64), (h >> np.uint32(16)).astype(np.int64)


class Code:
    """One moment in 8 bits: code (signed: with a sign bit) and exponent of each block of 256."""

    def __init__(self, n, signed):
        self.n, self.signed = n, signed
        self.depth, self.least = (14, 48) if signed else (30, 64)
        self.code = np.zeros(-(-n // 256) * 256, np.int64)
        self.exponent = np.zeros(self.code.size // 256, np.int64)

    def values(self):
        e = np.repeat(self.exponent, 256)
        k = self.code & 127 if self.signed else self.code
        place = k - 1 + 8 * (e - self.depth)                      # exponent * 8 + the three leading bits of the fraction
        value = np.where(k == 0, 0.0, (1 + place % 8 / 8) * np.exp2((place // 8 - 127).astype(np.float64)))
        if self.signed:
            value = np.where(self.code >= 128, -value, value)
        return np.where(e == 255, np.nan, value)[:self.n].astype(F)

    def store(self, x, noise):
        full, extra = np.zeros(self.code.size, F), np.zeros(self.code.size, np.int64)
        full[:self.n], extra[:self.n] = x, noise
        size = np.abs(full).astype(np.float64).reshape(-1, 256)
        extra = extra.reshape(-1, 256)
        most = size.max(1)
        bad = ~(most < 2.0 ** 127)
        with np.errstate(divide='ignore', invalid='ignore'):
            e = np.maximum(np.where(bad | (most == 0), 0, np.floor(np.log2(np.where(most > 0, most, 1)))) + 127, self.least)
        e = np.where(np.exp2(e - 126) <= most, e + 1, e)          # log2 rounds
        e = np.where((np.exp2(e - 127) > most) & (e > self.least), e - 1, e).astype(np.int64)
        floor = np.exp2((e - self.depth - 127).astype(np.float64))[:, None]
        with np.errstate(invalid='ignore', divide='ignore', over='ignore'):
            own = np.floor(np.log2(np.where(size > 0, size, 1)))
            own = np.where(np.exp2(own + 1) <= size, own + 1, np.where(np.exp2(own) > size, own - 1, own))
            # sixteenth-of-a-million steps above the power of two below it: an exact whole number for a 32-bit value
            steps = np.floor((size / np.exp2(own) - 1) * 2 ** 23 + (extra * 16 + 8)) // 2 ** 20
            k = 1 + 8 * (own + 127 - (e - self.depth)[:, None]) + steps
            k = np.where(size < floor, size > (extra + 0.5) / 65536 * floor, k)
        k = np.where(bad[:, None], 0, np.nan_to_num(k)).astype(np.int64)
        if self.signed:
            k = np.where(~bad[:, None] & (full.reshape(-1, 256) < 0), k | 128, k)
        self.code, self.exponent = k.reshape(-1), np.where(bad, 255, e)


class Plain:
    """One parameter.  bits 8: ``start`` is its place among the optimizer's moments."""

    def __init__(self, p, lr=1e-3, betas=(0.9, 0.999), epsilon=1e-8, decay=0.01, bits=32, seed=0, start=0):
        self.p = np.asarray(p, np.float64).reshape(-1).copy()
        self.lr, self.betas, self.epsilon, self.decay, self.bits, self.seed, self.start = lr, betas, epsilon, decay, bits, seed, start
        n, self.t = self.p.size, 0
        self.m, self.v = (np.zeros(n), np.zeros(n)) if bits == 32 else (Code(n, True), Code(n, False))

    def step(self, g):
        (b1, b2), g = self.betas, np.asarray(g, F).reshape(-1)
        self.t += 1
        with np.errstate(all='ignore'):
            if self.bits == 32:
                g = g.astype(np.float64)
                m = self.m = b1 * self.m + (1 - b1) * g
                v = self.v = b2 * self.v + (1 - b2) * g * g
            else:                    # each product and sum rounded to 32 bits
                m = self.m.values() * F(b1) + g * F(1 - b1)
                v = self.v.values() * F(b2) + g * F(1 - b2) * g
                of_m, of_v = noise(self.start, g.size, self.t, self.seed)
                self.m.store(m, of_m)
                self.v.store(v, of_v)
                m, v = m.astype(np.float64), v.astype(np.float64)
            change = self.lr / (1 - b1 ** self.t) * m / (np.sqrt(v / (1 - b2 ** self.t)) + self.epsilon)
            self.p = self.p * (1 - self.lr * self.decay) - change
        return change
