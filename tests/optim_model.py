"""Plain implementations of the optimiser's operators in numpy, written from their definitions: the AdamW step in 64 bits, codes and
scales of 8-bit moments bit by bit, the random bits that round them."""
import numpy as np

BLOCK = 128
U = 2.0 ** -24  # half a step of float32, relative
MASK64 = (1 << 64) - 1


def mix64(z):
    z = (z + 0x9E3779B97F4A7C15) & MASK64
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & MASK64
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & MASK64
    return z ^ (z >> 31)


def random_bits(seed, step, first_number, n):
    """20 bits for the first moment, 20 for the second, 16 for the parameter, of elements first_number ... first_number + n - 1."""
    key = np.uint64(mix64((mix64(seed) + step) & MASK64) & 0xFFFFFFFF)
    number = np.arange(first_number, first_number + n, dtype=np.uint64)
    low = np.uint64(0xFFFFFFFF)
    x = ((number >> np.uint64(1)) & low) * np.uint64(0x9E3779B1) & low
    x ^= x >> np.uint64(15)
    x ^= key
    x = x * np.uint64(0xBB67AE85) & low
    x ^= x >> np.uint64(15)
    x = x * np.uint64(0xA54FF53B) & low
    x ^= x >> np.uint64(15)
    x = x.astype(np.int64)
    rm = np.where(number % 2 == 0, x & 0xFFFFF, x >> 12)
    return rm, (rm * 0x5D3) & 0xFFFFF, (rm * 0xE2B >> 4) & 0xFFFF


def bits_of(x):
    return np.ascontiguousarray(x, dtype=np.float32).view(np.int32).astype(np.int64)


def floats_of(bits):
    return np.ascontiguousarray(bits).astype(np.uint32).view(np.float32)


def padded(x, n=None):
    n = -(-x.size // BLOCK) * BLOCK if n is None else n
    return np.concatenate([x, np.zeros(n - x.size, x.dtype)])


def encode(m, v, rm, rv):
    """Codes (whole blocks) and scales [blocks, 2] of float32 moments."""
    out, scales = [], []
    for x, r, binades in ((m, rm, 15), (v, rv, 31)):
        x, r = padded(np.abs(x).astype(np.float32)).reshape(-1, BLOCK), padded(np.asarray(r, np.int64)).reshape(-1, BLOCK)
        sign = padded(np.signbit(m if binades == 15 else np.abs(v))).reshape(-1, BLOCK)
        bits = bits_of(x) & 0x7FFFFFFF
        top = bits.max(1, keepdims=True)
        d = np.maximum(((top + 0x100100) >> 23) - binades, 1)
        with np.errstate(over="ignore", invalid="ignore"):
            code = (bits_of(x + floats_of(d << 23)) + r - (d << 23)) >> 20
        if binades == 31:
            code = np.maximum(code, np.minimum(bits, 1))
        else:
            code = code | sign.astype(np.int64) << 7
        lost = top + 0x100100 >= 0x7F800000  # not finite, or rounding up might make it so
        out.append(np.where(lost, 0, code).astype(np.uint8).reshape(-1))
        scales.append(np.where(lost, 255, d).astype(np.uint8))
    return out[0], out[1], np.concatenate(scales, 1)


def decode(mc, vc, scale):
    """What codes stand for, in 64 bits (exact: a difference of two floats of a few bits)."""
    out = []
    for k, codes in enumerate((mc, vc)):
        c = codes.reshape(-1, BLOCK).astype(np.int64)
        d = scale[:, k:k + 1].astype(np.int64)
        size = c & 127 if k == 0 else c
        unit = np.exp2(d - 127.0)
        x = unit * ((1 + (size % 8) / 8.0) * np.exp2(size // 8) - 1)
        x = np.where(d == 0, 0.0, x)
        x = np.where(d == 255, np.nan, x)
        out.append((np.where(c > 127, -x, x) if k == 0 else x).reshape(-1))
    return out


def moments_in_float(m, v, g, beta1, beta2, scale=1.0):
    """Both moments after a step, every operation rounded to float32 on its own in the documented order."""
    f = np.float32
    with np.errstate(over="ignore", invalid="ignore", under="ignore"):
        x = g.astype(f) * f(scale)
        m = m.astype(f) * f(beta1) + x * f(1.0 - beta1)
        v = v.astype(f) * f(beta2) + (x * f(1.0 - beta2)) * x
    return m, v


def step64(p, g, m, v, step, lr, weight_decay=0.0, beta1=0.9, beta2=0.999, eps=1e-8, scale=1.0):
    """One AdamW step in 64 bits: parameter, both moments, and how far a step in float32 may be off each.

    With u half a step of float32: a moment is a sum of two products of two or three factors, each product and the constants in it
    rounded (3 and 4 roundings for the first, 3 and 6 for the second, 1 for the sum). The divisor takes 8 (half of the second
    moment's, root, constant, product, eps, sum), the quotient one more, the parameter 3 and its sum 1. Below 2^-126 roundings are
    absolute, 2^-150 each."""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    x = g * scale
    size_m, size_v = np.abs(beta1 * m) + np.abs((1 - beta1) * x), beta2 * v + (1 - beta2) * x * x
    m, v = beta1 * m + (1 - beta1) * x, beta2 * v + (1 - beta2) * x * x
    mh, vh = m / (1 - beta1 ** step), v / (1 - beta2 ** step)
    d = np.sqrt(vh) + eps
    new = p - lr * weight_decay * p - lr * mh / d
    tol_p = 5 * U * np.abs(p) + 22 * U * lr / (1 - beta1 ** step) * size_m / d + 1e-44
    return new, m, v, tol_p, 5 * U * size_m + 1e-44, 7 * U * size_v + 1e-44
