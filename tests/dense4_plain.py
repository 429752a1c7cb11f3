"""4-bit dense weights in NumPy, by the layout that include/xsmi355.h gives."""
import numpy as np


def up(v, to):
    return -(-v // to) * to


def pack(numbers, scales, group):
    """(K, N) whole numbers and (groups, N) scales -> codes and scales with the padding."""
    k, n = numbers.shape
    kp, np_ = up(k, 128), up(n, 16)
    full = np.zeros((kp, np_), np.int64)
    full[:k, :n] = numbers
    codes = np.zeros((np_ // 16, kp // 128, 64, 16), np.uint8)
    for i in range(kp):
        c, r = divmod(i, 128)
        j, r = divmod(r, 32)
        quarter, r = divmod(r, 8)
        for o in range(16):
            codes[:, c, quarter * 16 + o, 4 * j + r // 2] |= ((full[i, o::16] & 15) << (4 * (r % 2))).astype(np.uint8)
    s = np.zeros((kp // group, np_), np.float16)
    s[:scales.shape[0], :n] = scales
    return codes, s


def quantize(w, group):
    """(K, N) float32 weights -> whole numbers and float16 scales."""
    k, n = w.shape
    groups = up(k, 128) // group
    numbers, scales = np.zeros((k, n), np.int64), np.zeros((groups, n), np.float16)
    for g in range(-(-k // group)):
        part = w[g * group:(g + 1) * group]
        extreme = part[np.abs(part).argmax(0), np.arange(n)]
        scales[g] = (extreme / np.float32(-8)).astype(np.float16)
        s = scales[g].astype(np.float32)
        with np.errstate(divide='ignore', invalid='ignore'):
            numbers[g * group:(g + 1) * group] = np.where((s == 0) | (part == 0), 0, np.clip(np.rint(part / s), -8, 7))
    return numbers, scales


def values(numbers, scales, group):
    return numbers * np.repeat(scales.astype(np.float64), group, 0)[:numbers.shape[0]]
