"""MXFP4 rows and their products restated in numpy, in 64 bits: blocks of 32 values, a byte e and 16 bytes of codes, E2M1(code) 2^(e - 127); activations as whole numbers of -255 .. 255 times 2^s."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def values(packed):
    """packed blocks, uint8 [..., K / 32 * 17] -> float64 [..., K]"""
    b = packed.reshape(*packed.shape[:-1], -1, 17)
    code = np.concatenate([b[..., 1:] & 15, b[..., 1:] >> 4], -1)
    e = b[..., :1].astype(np.int64)
    v = np.where(code & 8, -1.0, 1.0) * GRID[code & 7] * np.ldexp(1.0, e - 127)
    return np.where(e == 255, np.nan, v).reshape(*packed.shape[:-1], -1)


def quantise(x):
    """float32 [..., K] -> packed blocks, uint8 [..., K / 32 * 17]"""
    b = np.asarray(x, np.float32).astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    top = np.abs(b).max(-1)
    good = np.isfinite(top)
    e = np.where(good & (top > 0), np.frexp(np.where(good, top, 1.0))[1] - 1 - 2 + 127, 0)
    e = np.where(good, np.maximum(e, 0), 255)
    with np.errstate(invalid="ignore", over="ignore"):
        m = np.abs(b) * np.ldexp(1.0, 127 - e)[..., None]
        code = np.searchsorted((GRID[1:] + GRID[:-1]) / 2, np.where(good[..., None], m, 0.0), side="left")  # (a tie belongs to the value below)
    code = np.where(good[..., None], code, 0).astype(np.uint8)
    code |= np.where((b < 0) & (code > 0), 8, 0).astype(np.uint8)
    return np.concatenate([e[..., None].astype(np.uint8), code[..., :16] | (code[..., 16:] << 4)], -1).reshape(*x.shape[:-1], -1)


def activations(x):
    """float32 [..., K] -> what a product takes for them, float64"""
    b = np.asarray(x, np.float32).astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    top = np.abs(b).max(-1, keepdims=True)
    good = np.isfinite(top)
    with np.errstate(invalid="ignore"):
        s = np.frexp(np.where(good, top, 1.0))[1] - 8
        s = np.where(np.rint(np.ldexp(np.where(good, top, 1.0), -s)) > 255, s + 1, s)
        s = np.clip(s, -120, 120)
        q = np.clip(np.rint(np.ldexp(b, -s)), -255, 255)
        return np.where(good, np.ldexp(q, s), np.nan).reshape(x.shape)


def product(x, w):
    """float32 [..., K], packed [N, K / 32 * 17] -> (float64 [..., N], the sum of the magnitudes)"""
    a, v = activations(x), values(w)
    return a @ v.T, np.abs(a) @ np.abs(v).T


def check(name, got, want, mags, K, extra=0.0):
    """f32 sums of 2 K exact products (two digits of every activation) in whatever order: off by at most 2 K roundings of 2^-24 of the sum of magnitudes each; and, roundings being as often up as
    down, by 2^-24 sqrt(2 K) of the whole in the 2-norm (the mean of n growing partial sums' roundings is sqrt(n / 6) of it).  extra: magnitude of what is added behind the sum, one more rounding."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, (name, got.shape, want.shape)
    nan = np.isnan(want)
    assert np.array_equal(nan, np.isnan(got)), name
    d, m = np.abs(got - want)[~nan], (mags + 0 * want)[~nan]
    ex = (extra + 0 * want)[~nan]
    over = d > 2.0**-24 * (2 * K * m + m + ex)
    assert not over.any(), (name, float(d.max()), int(over.sum()))
    norm = float(np.linalg.norm(want[~nan]))
    rel = float(np.linalg.norm(d)) / norm if norm else 0.0
    assert rel <= 2.0**-24 * (np.sqrt(2 * K) + 1), (name, rel)
    return rel


def experts(x, w, ids, bias=None):
    """x [T, 1 or U, K], w [E, N, packed], ids [T, U] -> (float64 [T, U, N], magnitudes); NaN rows of zeros magnitude where the id names no expert"""
    T, U = ids.shape
    y, m = np.zeros((T, U, w.shape[1])), np.zeros((T, U, w.shape[1]))
    for e in range(w.shape[0]):
        t, u = np.nonzero(ids == e)
        if len(t):
            y[t, u], m[t, u] = product(x[t, u % x.shape[1]], w[e])
            if bias is not None:
                y[t, u] += bias[e].astype(np.float64)
    return y, m
