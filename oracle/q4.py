"""The 4-bit form of K and V in 64 bits, and attention over what it holds (test infrastructure).

Of 32 consecutive values of a head vector, m is the one of the largest magnitude (the first of
equals); the step is m / -8 rounded to binary16, at most 65504 in magnitude; x is kept as
step * n, n = x / step rounded to the nearest whole number (ties to even), within -8 .. 7. A
group that holds an infinity or NaN becomes NaN, one with step 0 zeros.
"""

from __future__ import annotations

import numpy as np

GROUP = 32


def quantise(x):
    """(n + 8 as uint8 `[..., d]`, steps as float16 `[..., d / 32]`) of f32 values."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(all="ignore"):
        at = np.abs(g).argmax(-1)[..., None]
        m = np.take_along_axis(g, at, -1).astype(np.float64)
        finite = np.isfinite(g).all(-1, keepdims=True)
        step = np.clip(np.where(finite, m, 0.0) / -8.0, -65504.0, 65504.0).astype(np.float16)
        s = step.astype(np.float64)
        n = np.clip(np.rint(np.where(finite, g, 0.0).astype(np.float64) / np.where(s == 0, 1.0, s)), -8, 7)
        n = np.where(finite & (s != 0), n, 0)
    step = np.where(finite, step, np.float16(np.nan))
    return (n + 8).astype(np.uint8).reshape(x.shape), step[..., 0]


def values(codes, steps):
    """What they stand for, f64."""
    n = codes.astype(np.float64).reshape(*codes.shape[:-1], -1, GROUP) - 8
    return (n * steps.astype(np.float64)[..., None]).reshape(codes.shape)


def rows(codes, steps):
    """The bytes of head vectors as pages are read and written: `[..., 72]`."""
    b = codes[..., ::2] | (codes[..., 1::2] << 4)
    return np.concatenate([b, np.ascontiguousarray(steps).view(np.uint8)], -1)


def from_rows(b):
    c = np.stack([b[..., :64] & 15, b[..., :64] >> 4], -1).reshape(*b.shape[:-1], 128)
    return c, np.ascontiguousarray(b[..., 64:]).view(np.float16)


def attend(q, k, v, first, last, scale):
    """Attention of q `[rows][hq][d]` over k, v `[keys][hkv][d]`, row r over the keys first[r] ..
    last[r]; all in 64 bits. Returns (out `[rows][hq][d]`, a bound on the error of f32 sums).

    The bound: a score's 128 products are exact or cut 2^-21, its sum rounds 128 times at
    most and its scaling twice, dS <= (128 + 8 + 2) 2^-24 sum |q k| scale. A weight e^S is then
    off by at most its share e^dS - 1 <= 1.01 dS, and 2^-21 by the exponential and its argument
    (arguments up to 2^7 with 2^-24 each); in sum and quotient twice. Sums over keys round once
    a key at most, a weight times step is cut 2^-21: (keys + 16) 2^-24 of sum w |v|. That cut is
    also absolute, half of binary16's smallest number: with weights scaled to 2^11 (2^-4 where a
    step of V reaches 8) against a largest weight of 1 and codes to 8, 2^-25 8 / 2^11 = 2^-33
    (2^-18, of values that reach 64) a key. (The kernels scale to 2^13 whatever V: 2^-38 |v| a key.)
    """
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    group = q.shape[1] // k.shape[1]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    u = 2.0 ** -24
    for r in range(q.shape[0]):
        ks, vs = k[first[r]:last[r] + 1], v[first[r]:last[r] + 1]
        for h in range(q.shape[1]):
            s = ks[:, h // group] @ q[r, h] * scale
            size = np.abs(ks[:, h // group]) @ np.abs(q[r, h]) * abs(scale)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[r, h] = w @ vs[:, h // group]
            ds = 138 * u * size.max() + 8 * u + 2 * u * (np.abs(s).max() + (s.max() - s.min()))
            bound[r, h] = (w @ np.abs(vs[:, h // group])) * (2.1 * ds + (2 * len(s) + 32) * u)
            bound[r, h] += len(s) * (2.0 ** -33 if np.abs(vs[:, h // group]).max() < 56 else 2.0 ** -18)
    return out, bound + 1e-30
