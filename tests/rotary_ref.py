"""Plain 64-bit rotary positions, and the error that the kernels' arithmetic
allows, from the arithmetic alone.

With u = 2^-24 (fp32): the angle in turns is off by 2 2^-53 of itself (two
roundings in 64 bits); brought within half a turn and doubled, it is rounded to
fp32, off by 2^-25, which is d = pi 2^-25 < 1.6 u radians; put back to first order
with one rounding, d^2 is left, nothing here, and that rounding, u. Sine and cosine
are right to 2 ulp (2 u), their product with the magnitude to u, the products with
x and y and their sum to u each: with (|x| + |y|) m in front,
    (1 + 2 + 1 + 1 + 1) u + the 64-bit angle's own error.
The result is rounded to its type (half a step)."""

from __future__ import annotations

import math

import numpy as np

HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def rotate(x, position, frequencies, *, interleaved=False, magnitude=1.0, transpose=False, dtype="f32"):
    """x [.., T, D] (float64) at `position` (broadcast against x's axes but the
    last): the turned rows and their error bounds."""
    part = 2 * len(frequencies)
    a = slice(0, part, 2) if interleaved else slice(0, part // 2)
    b = slice(1, part, 2) if interleaved else slice(part // 2, part)
    angle = np.asarray(position, np.float64)[..., None] * np.asarray(frequencies, np.float64)
    # (numpy reduces 64-bit angles of this size to well below their own rounding)
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle) * (-1.0 if transpose else 1.0)
    out, bound = x.copy(), np.zeros(x.shape)
    p, q = x[..., a], x[..., b]
    out[..., a], out[..., b] = p * c - q * s, q * c + p * s
    e = (6.0 * 2.0 ** -24 + 4.0 * 2.0 ** -53 * np.abs(angle)) * abs(magnitude) * (np.abs(p) + np.abs(q))
    half = 2.0 ** -25 if dtype == "f16" else 2.0 ** -134 if dtype == "bf16" else 2.0 ** -150  # subnormals
    bound[..., a] = e + HALF[dtype] * (np.abs(out[..., a]) + e) + half
    bound[..., b] = e + HALF[dtype] * (np.abs(out[..., b]) + e) + half
    return out, bound


def frequencies(part, base=10000.0):
    return [base ** (-2.0 * i / part) for i in range(part // 2)]


def parts(part, factor, original, low=1.0, high=32.0, base=10000.0):
    out = []
    for f in frequencies(part, base):
        turns = original * f / (2 * math.pi)
        if turns >= high:
            out.append(f)
        elif turns <= low:
            out.append(f / factor)
        else:
            g = (turns - low) / (high - low)
            out.append(g * f + (1 - g) * f / factor)
    return out
