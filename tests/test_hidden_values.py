"""The check of hidden values finds what it is for: a leak planted in rows that a plain
implementation forms, on the CPU."""

from __future__ import annotations

import numpy as np
import pytest

from hidden_values import check_rows
from serving_ref import attend_row

NAN, INF = float("nan"), float("inf")


def plain(bad_value, window=0, sinks=0):
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((2, 2, 3, 8)), rng.standard_normal((2, 40, 8)), rng.standard_normal((2, 40, 8))
    lengths, bad = [20, 39], [[18], [18]]
    k[:, 18, 1] = v[:, 18, 1] = bad_value
    out = np.empty((2, 2, 3, 8))
    with np.errstate(invalid="ignore"):
        for b in range(2):
            for h in range(2):
                for t in range(3):
                    out[b, h, t] = attend_row(q[b, h, t], k[b], v[b], lengths[b] - 3 + t, lengths[b], window=window,
                                              sinks=sinks)[0]
    return lambda out: check_rows("plain", out, q, lambda b, h: (k[b], v[b]), lambda b, t: lengths[b] - 3 + t,
                                  lambda b: lengths[b], bad, 1, dtype="f32", window=window, sinks=sinks), out


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("options,rows", [(dict(), (10, 2)), (dict(window=5, sinks=2), (4, 8))])
def test_leaks_are_found(bad, options, rows):
    check, out = plain(bad, **options)
    assert check(out) == rows
    hidden = [(0, 0, 0), (0, 1, 0)]  # before the key
    if options:
        hidden += [(1, 0, 2), (1, 1, 0)]  # behind the window
    for at in hidden:
        for value in (NAN, INF, 1e3):
            leak = out.copy()
            leak[at][1] = value
            with pytest.raises(AssertionError):
                check(leak)
    for at in ((0, 0, 1), (0, 1, 2)):  # rows that see the key
        lost = out.copy()
        lost[at] = 0.0
        with pytest.raises(AssertionError, match="did not take"):
            check(lost)
