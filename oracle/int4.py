"""CPU definition of the 4-bit head (TEST INFRASTRUCTURE ONLY: see oracle/__init__.py), in 64 bits.

A group of consecutive values of a row (the last may be shorter) is s (q - z): lo = min(0, least), hi = max(0, largest),
s = (hi - lo) times the fp32 number nearest 1/15, both steps in fp32, rounded to bf16 (ties to even); z = -lo / s and q = value / s + z,
quotients rounded to the nearest whole number (ties to even), both held in 0 .. 15.  A group with s = 0 is 0; one with a value
that is not finite, or whose range hi - lo is not, is NaN."""
import numpy as np


def round_bf16(x):
    """fp32 >= 0 -> the nearest bf16 value (ties to even), as fp32."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return (((u + 0x7FFF + ((u >> 16) & 1)) >> 16) << 16).astype(np.uint32).view(np.float32)


def quantise(w, group):
    """w [N, K] fp32 -> (codes [N, K], scales [N, groups] fp32, zeros [N, groups])."""
    w = np.asarray(w, np.float32)
    n, k = w.shape
    b = np.pad(w, ((0, 0), (0, -k % group))).reshape(n, -1, group)
    bad = ~np.isfinite(b).all(2)
    b = np.where(bad[:, :, None], np.float32(0), b)
    lo, hi = np.minimum(b.min(2), 0), np.maximum(b.max(2), 0)
    with np.errstate(over="ignore"):
        s = ((hi - lo) * np.float32(1 / 15)).astype(np.float32)
    bad |= ~np.isfinite(s)
    s = round_bf16(np.where(bad, np.float32(0), s))
    bad |= ~np.isfinite(s)
    d = np.where((s > 0) & ~bad, s, np.float32(1))
    z = np.clip(np.rint(-lo / d), 0, 15)
    q = np.clip(np.rint(b / d[:, :, None]) + z[:, :, None], 0, 15)
    s = np.where(bad, np.float32(np.nan), s)
    return q.reshape(n, -1)[:, :k].astype(np.uint8), s, z.astype(np.uint8)


def values(codes, scales, zeros, group):
    """The weights that codes stand for, float64."""
    k = codes.shape[1]
    z = np.full(scales.shape, 8) if zeros is None else zeros & 15
    spread = lambda t: np.repeat(np.asarray(t, np.float64), group, 1)[:, :k]  # noqa: E731
    return spread(scales) * ((codes & 15).astype(np.float64) - spread(z))
