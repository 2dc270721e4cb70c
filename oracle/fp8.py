"""CPU definition of the 8-bit head (TEST INFRASTRUCTURE ONLY: see oracle/__init__.py), in 64 bits.

A block of 128 consecutive values of a row (the last may be shorter) is q * 2^e: e the least whole number >= -127 with
max|x| <= 448 * 2^e, q = x / 2^e rounded to the nearest e4m3 value (sign, 4 exponent bits of bias 7, 3 fraction bits,
subnormals of 2^-9; ties to the even fraction).  The value is then held in bf16, which takes something from it only below
2^-133, bf16's least value (e < -124: nearest, ties to even).  A value that is not finite becomes NaN."""
import numpy as np

BLOCK = 128


def e4m3_values():
    """The 127 finite non-negative values, ascending: code c stands for entry c."""
    c = np.arange(127)
    e, f = c >> 3, c & 7
    return np.where(e == 0, f * 2.0 ** -9, (8 + f) * 2.0 ** (e - 10.0))


def round_e4m3(v):
    """|v| <= 448 to the nearest e4m3 value: by search in the table, ties to the even code."""
    t = e4m3_values()
    a = np.abs(v)
    hi = np.clip(np.searchsorted(t, a), 1, 126)
    lo = hi - 1
    up, down = t[hi] - a, a - t[lo]
    c = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return np.copysign(t[c], v)


def block_exponents(x):
    """[rows, K] -> [rows, ceil(K / 128)] exponents of the finite blocks."""
    rows, k = x.shape
    a = np.abs(np.pad(np.asarray(x, np.float64), ((0, 0), (0, -k % BLOCK)))).reshape(rows, -1, BLOCK).max(2)
    m, p = np.frexp(a)  # a = m * 2^p, m in [0.5, 1); 448 = 0.875 * 2^9
    return np.where(a > 0, np.maximum(p - 9 + (m > 0.875), -127), -127).astype(np.int64)


def values(x):
    """What x [rows, K] stands for in 8 bits, float64."""
    x = np.asarray(x, np.float64)
    bad = ~np.isfinite(x)
    x = np.where(bad, 0.0, x)
    e = np.repeat(block_exponents(x), BLOCK, 1)[:, :x.shape[1]]
    v = np.ldexp(round_e4m3(np.ldexp(x, -e)), e)
    return np.where(bad, np.nan, np.ldexp(np.rint(np.ldexp(v, 133)), -133))
