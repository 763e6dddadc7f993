"""What the operators that leave entries out compute, by their definitions in 64 bits with numpy."""
import numpy as np

M32 = 0xFFFFFFFF
HALF_STEP = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # of a rounding, relative to the value


def philox4x32(counter, key, rounds=7):
    """counter: four arrays of uint64 below 2^32, key: two integers. Salmon et al., 2011."""
    low, shift = np.uint64(M32), np.uint64(32)
    x = [np.asarray(c, np.uint64) for c in counter]
    k0, k1 = key
    for _ in range(rounds):
        p, q = np.uint64(0xD2511F53) * x[0], np.uint64(0xCD9E8D57) * x[2]
        x = [(q >> shift) ^ x[1] ^ np.uint64(k0), q & low, (p >> shift) ^ x[3] ^ np.uint64(k1), p & low]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return x


def dropout_bits(n, seed, step, first=0):
    """The 16 bits of elements first .. first + n - 1."""
    at = np.arange(first, first + n, dtype=np.uint64)
    block = at >> np.uint64(3)
    step &= (1 << 64) - 1
    words = philox4x32([block & np.uint64(M32), block >> np.uint64(32), np.full_like(block, step & M32), np.full_like(block, step >> 32)],
                       (seed & M32, seed >> 32))
    w = np.stack(words, 1)[np.arange(n), (at.astype(np.int64) >> 1) & 3]
    return np.where(at & np.uint64(1), w >> np.uint64(16), w & np.uint64(0xFFFF)).astype(np.int64)


def threshold(p):
    return int(np.floor(p * 65536 + 0.5))


def dropout(x, p, seed, step, residual=None):
    """Flat arrays in 64 bits, and which elements are left out."""
    t = threshold(p)
    out = dropout_bits(x.size, seed, step) < t
    y = np.where(out, 0.0, x.astype(np.float64) * (65536.0 / (65536 - t) if t < 65536 else 0.0))
    return (y if residual is None else y + residual.astype(np.float64)), out


def select_kept(score, budget, recent=0, length=None):
    """score: [rows, n]. Indices [rows, budget] and counts [rows]."""
    rows, n = score.shape
    index, count = np.full((rows, budget), -1, np.int64), np.zeros(rows, np.int64)
    for row in range(rows):
        m = n if length is None else min(max(int(length[row]), 0), n)
        s = score[row, :m].astype(np.float64)
        if m <= budget:
            kept = np.arange(m)
        else:
            free = m - recent
            order = np.lexsort((np.arange(free), -np.where(np.isnan(s[:free]), -np.inf, s[:free]), np.isnan(s[:free])))
            kept = np.sort(np.r_[order[:budget - recent], np.arange(free, m)])
        index[row, :len(kept)], count[row] = kept, len(kept)
    return index, count


def keep_rows(a, index, dim):
    """a: an array, index: [K] or [rows, K]; rows of zeros where an index is none."""
    if index.ndim == 2:
        return np.stack([keep_rows(x, i, dim - 1) for x, i in zip(a, index)]) if len(index) else a[:, :0]
    there = (index >= 0) & (index < a.shape[dim])
    if a.shape[dim] == 0:
        return np.zeros(a.shape[:dim] + (len(index),) + a.shape[dim + 1:], a.dtype)
    out = np.take(a, np.where(there, index, 0), axis=dim)
    out[(slice(None),) * dim + (~there,)] = 0
    return out
