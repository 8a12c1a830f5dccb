"""Values in four bits written out in 64 bits with numpy, for the tests."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def scales(x):
    """bytes [.., dim / 32] of the blocks of x [.., dim] (float64)"""
    b = np.abs(np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], -1, 32))
    top = np.where(np.isnan(b).any(-1), np.inf, np.nan_to_num(b, nan=0.0, posinf=np.inf).max(-1))
    borders = 7.0 * 2.0 ** np.arange(-126, 128)                      # the first that is not below it
    return np.where(top < 2.0 ** 127, np.searchsorted(borders, top) + 1, 255).astype(np.uint8)


def codes(x, e):
    """codes [.., dim] of x for scales e: the nearest, of two the even one"""
    b = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], -1, 32)
    y = np.abs(b) / 2.0 ** (e.astype(np.float64)[..., None] - 127)
    far = np.abs(y[..., None] - GRID)
    near = far.min(-1, keepdims=True)
    even = np.where((far == near) & (np.arange(8) % 2 == 0), 0, np.where(far == near, 1, 2))
    return (even.argmin(-1) + 8 * np.signbit(b)).astype(np.uint8).reshape(x.shape)


def unpack(packed):
    """codes [.., dim] of bytes [.., dim / 2]"""
    return np.stack([packed & 15, packed >> 4], axis=-1).reshape(*packed.shape[:-1], -1)


def pack(c):
    return (c[..., 0::2] | (c[..., 1::2] << 4)).astype(np.uint8)


def values(c, e):
    """float64 of codes [.., dim] and scales [.., dim / 32]"""
    v = np.where(c >= 8, -1.0, 1.0) * GRID[c & 7]
    by = np.where(e == 255, np.nan, 2.0 ** (e.astype(np.float64) - 127))
    return (v.reshape(*c.shape[:-1], -1, 32) * by[..., None]).reshape(c.shape)


def rounded(x):
    """the values that four bits hold of x"""
    e = scales(x)
    with np.errstate(invalid="ignore"):
        return values(codes(x, np.where(e == 255, 127, e).astype(np.uint8)), e)


def holds(packed, e, x, delta):
    """Whether codes and scales are those of x or of something up to delta [.., 1] from each of its values (a sum rounded otherwise may lie
    on the other side of a border)."""
    b = np.abs(x.reshape(*x.shape[:-1], -1, 32)).max(-1)
    low, high = 7.0 * 2.0 ** (e.astype(np.float64) - 128), 7.0 * 2.0 ** (e.astype(np.float64) - 127)
    good = (b <= high + delta) & ((b > low - delta) | (e == 1))
    c = unpack(packed)
    by = np.repeat(2.0 ** (e.astype(np.float64) - 127), 32, axis=-1)
    middle = np.concatenate([[0.0], (GRID[1:] + GRID[:-1]) / 2, [np.inf]])
    n, y = c & 7, np.where(c >= 8, -x, x) / by                       # (of the code's sign)
    slack = np.repeat(np.broadcast_to(delta, b.shape), 32, axis=-1) / by
    inside = (y >= np.where(n == 0, -slack, middle[n] - slack)) & (y <= middle[n + 1] + slack)
    return bool(good.all() and inside.all())
