"""Plain 64-bit implementation of the windowed and paged attention, and the
error that the kernels' arithmetic allows, from the arithmetic alone.

With u = 2^-24 (fp32) and d = half a step of the type that probabilities are
rounded to (0 for fp32), the kernels form, per score x in log2 units,
  products exactly summed in fp32 over D terms     D u sum|q k| scale log2e
  scale, bias and cap, a few fp32 operations       6 u (|x| + |bias|) (+ 8 u cap)
  x - max and exp2 (1 ulp, and the argument)       2 u (|x| + |max|) + 2 u
so a probability is off by e = ln2 (sum of those) relative, plus d. Numerator
and denominator use the same rounded p (w: exact weights, o: exact row):
  |err| <= (e + d) / (1 - e - d) sum w |v - o| + n u (sum w |v| + |o|) + out |o|
with n fp32 additions over the row (keys, and the joins) and the output's
half step `out`."""

from __future__ import annotations

import math

import numpy as np

HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
LOG2E = math.log2(math.e)


def seen_keys(position: int, length: int, window: int, sinks: int) -> np.ndarray:
    j = np.arange(max(0, min(length, position + 1)))
    if window:
        j = j[(position - j < window) | (j < sinks)]
    return j


def attend_row(q, k, v, position, length, *, window=0, sinks=0, scale=None, slope=0.0, softcap=0.0,
               dtype="f32", out_dtype="f32", hidden=()):
    """q [D], k [N, D], v [N, Dv] (float64): the row and its error bound. `hidden`:
    keys that are not seen for another reason."""
    j = seen_keys(position, length, window, sinks)
    if len(hidden):
        j = j[~np.isin(j, hidden)]
    if j.size == 0:
        return np.zeros(v.shape[1]), np.zeros(v.shape[1])
    scale = 1.0 / math.sqrt(q.size) if scale is None else scale
    k, v = k[j], v[j]
    bias = slope * (j - position)
    x = (k @ q) * scale + bias
    mag = (np.abs(k) @ np.abs(q)) * abs(scale)
    u = 2.0 ** -24
    err = q.size * u * mag + 6 * u * (np.abs(x) + np.abs(bias))
    if softcap:
        x = softcap * np.tanh(x / softcap)
        err += 8 * u * softcap
    top = x.max()
    err += 2 * u * (np.abs(x) + abs(top) + 8)
    w = np.exp(x - top)
    w /= w.sum()
    o = w @ v
    # e is per key: the weighted sum of what each is off by
    e = err + 2 * u + (0.0 if dtype == "f32" else HALF[dtype])
    spread = (w * e) @ np.abs(v - o) / (1 - e.max())
    bound = spread + (j.size + 8) * u * (w @ np.abs(v) + np.abs(o)) + HALF[out_dtype] * np.abs(o) + 1e-30
    if out_dtype == "f16":
        bound = bound + 2.0 ** -25  # half a step of the subnormals
    return o, bound
