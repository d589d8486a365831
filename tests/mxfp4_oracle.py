"""Plain 64-bit forms of the MXFP4 operators, for the tests: the format's values,
the quantizer by the distance to each value, products of exact values, and how
far f32 sums may be from them."""
import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def values(qs, s):
    """codes uint8 [.., n / 2], scales uint8 [.., n / 32] -> f64 [.., n]"""
    c = np.stack((qs & 15, qs >> 4), -1).reshape(*qs.shape[:-1], -1)
    v = np.where(c >= 8, -1.0, 1.0) * GRID[c & 7]
    with np.errstate(invalid="ignore"):
        d = np.where(s == 255, np.nan, np.ldexp(1.0, s.astype(np.int64) - 127))
        return (v.reshape(*s.shape, 32) * d[..., None]).reshape(v.shape)


def quantize(x):
    """x f64 [.., n] (values of a storage type) -> (codes, scales)"""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(b).max(-1)  # (NaN where a block holds one)
    ok = np.isfinite(amax)
    e = np.frexp(np.where(ok & (amax > 0), amax, 1.0))[1] - 1  # floor(log2)
    s = np.where(amax == 0, 0, np.clip(e - 2 + 127, 0, 254))
    s = np.where(ok, s, 255)
    y = np.where(ok[..., None], b, 0.0) / np.ldexp(1.0, np.where(ok, s, 127) - 127)[..., None]
    d = np.abs(np.abs(y)[..., None] - GRID)
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])  # the even code wins a tie
    code = order[np.argmin(d[..., order], -1)]
    code = np.where(np.abs(y) > 6, 7, code) + 8 * np.signbit(b)
    code = code.reshape(*x.shape[:-1], -1).astype(np.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, s.astype(np.uint8)


def product(w, x):
    """y = x w^T in 64 bits and its bound: every product is exact; a term passes one addition a matrix instruction
    of its accumulator's (of 64 elements or more each, or of 32 with two accumulators taking turns: in / 64 of them) and
    those of accumulators', waves' and parts' joins, at most 24, each addition off by at most a step (2^-23) of the sum
    of magnitudes."""
    y, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    return y, (w.shape[1] / 64 + 25) * 2.0**-23 * mag
