"""What a row does not see does not reach it: rows of an attention some of whose
keys hold a NaN or an infinity, in V's column `column` and maybe in K, against
the 64-bit rows of serving_ref.py, within the bound that it derives."""

from __future__ import annotations

import numpy as np

from serving_ref import attend_row, seen_keys


def check_rows(label, out, q, rows, position, length, bad, column, *, dtype, heads=None, hidden=(), **options):
    """out, q [B,H,T,.] (float64); rows(b, h) -> K and V [N,.] of head h's sequence;
    position(b, t), length(b); bad: a list of keys per sequence. A row that sees one has
    no number in the column; any other is finite and right. Returns how many of
    either there were."""
    B, H, T, _ = q.shape
    window, sinks = options.get("window", 0), options.get("sinks", 0)
    touched = clean = 0
    for b in range(B):
        for t in range(T):
            p, n = position(b, t), length(b)
            sees = np.isin(bad[b], seen_keys(p, n, window, sinks)).any() if len(bad[b]) else False
            for h in range(H) if heads is None else heads:
                row = out[b, h, t]
                if sees:
                    assert not np.isfinite(row[column]), f"{label}: row {b, h, t} sees what it did not take"
                    touched += 1
                    continue
                k, v = rows(b, h)
                ref, bound = attend_row(q[b, h, t], k, v, p, n, dtype=dtype, out_dtype=dtype, hidden=hidden, **options)
                assert np.isfinite(row).all(), f"{label}: row {b, h, t} is not finite"
                off = np.abs(row - ref)
                assert (off <= bound).all(), f"{label}: row {b, h, t} off by {off.max():.3e}"
                clean += 1
    return touched, clean
