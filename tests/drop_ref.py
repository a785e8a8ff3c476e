"""Dropout on the host: the kept elements from Philox4x32-10 in numpy, and the ops' formulas in single precision."""
import numpy as np

LOW = np.uint64(0xFFFFFFFF)


def philox(c, k0, k1):
    """Ten rounds over four arrays of 32-bit words (held in 64)."""
    for r in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        w0, w1 = np.uint64(k0 + r * 0x9E3779B9 & 0xFFFFFFFF), np.uint64(k1 + r * 0xBB67AE85 & 0xFFFFFFFF)
        c = [b >> np.uint64(32) ^ c[1] ^ w0, b & LOW, a >> np.uint64(32) ^ c[3] ^ w1, a & LOW]
    return c


def keep(n, p, seed, step, site, first=0):
    """Which of the elements first .. first + n - 1 stay (first a multiple of 4)."""
    blocks = np.arange((n + 3) // 4, dtype=np.uint64) + np.uint64(first // 4)
    full = lambda v: np.full(blocks.shape, v & 0xFFFFFFFF, np.uint64)  # noqa: E731
    w = philox([blocks & LOW, blocks >> np.uint64(32), full(step), full(1 + site)], seed & 0xFFFFFFFF, seed >> 32)
    return np.stack(w, 1).reshape(-1)[:n] >= np.uint64(int(np.rint(float(np.float32(p)) * 2.0 ** 32)))


def drop(x, kept, p):
    scale = np.float32(1.0 / (1.0 - float(np.float32(p))))
    with np.errstate(all="ignore"):
        return np.where(kept, x * scale, np.float32(0.0)).astype(np.float32)
