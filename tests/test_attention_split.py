"""CPU: the error of a float held as two halves, and of the product of two such, as the matrix kernels take them."""
import numpy as np


def split(x):
    h = x.astype(np.float16)
    return h.astype(np.float64), (x - h.astype(np.float32)).astype(np.float16).astype(np.float64)


def test_two_halves_and_their_product():
    """Bounds of two roundings to 11 bits: 2^-11 for the first, 2^-23 after the second (what the first leaves is a multiple
    of the float's last bit, and below half a unit of 2^-10), 2^-22 for the product of the two lower parts."""
    rng = np.random.default_rng(1)
    x, y = (np.ldexp(1.0 + rng.random(1 << 21), 14).astype(np.float32) for _ in range(2))
    x[:4] = np.ldexp(np.float32([1 + 2.0 ** -11, 1 + 2.0 ** -11 + 2.0 ** -23, 1 + 2.0 ** -11 - 2.0 ** -23, 1.0]), 14)
    (xh, xl), (yh, yl) = split(x), split(y)
    x, y = x.astype(np.float64), y.astype(np.float64)
    assert (np.abs(x - xh) <= 2.0 ** -11 * x).all() and (np.abs(x - xh) > 2.0 ** -12 * x).any()
    assert (np.abs(x - xh - xl) <= 2.0 ** -23 * x).all() and (np.abs(x - xh - xl) > 2.0 ** -24 * x).any()
    assert (np.abs(xl * yl) <= 2.0 ** -22 * x * y).all() and (np.abs(xl * yl) > 2.0 ** -24 * x * y).any()
    off = np.abs(x * y - (xh * yh + xl * yh + xh * yl)) / (x * y)
    assert off.max() <= 2.0 ** -21 * (1 + 2.0 ** -10) and off.mean() <= 2.0 ** -23


def test_small_elements_beside_the_largest():
    """Below 2^-2, where the lower part is no normal half, the error stays under 2^-25."""
    rng = np.random.default_rng(2)
    x = np.ldexp(1.0 + rng.random(1 << 20), rng.integers(-40, -2, 1 << 20)).astype(np.float32)
    h, l = split(x)
    assert np.abs(x.astype(np.float64) - h - l).max() <= 2.0 ** -25
