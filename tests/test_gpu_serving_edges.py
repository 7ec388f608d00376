"""GPU tests of the serving operators where an argument stands at the edge of what
the interface allows, against plain 64-bit rows within a bound from the arithmetic."""

from __future__ import annotations

import math

import numpy as np
import pytest

from serving_ref import attend_row
from test_gpu_serving import NAN, TYPES, compare, f64, randn

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


# --- padding rows against values that they do not see ------------------------

@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (16, 1, 128), (32, 2, 64), (40, 1, 256)])
@pytest.mark.parametrize("bad", [NAN, math.inf])
def test_padding_rows_of_single_queries(ofh, dt, H, Hkv, D, bad):
    """One query row per sequence, past the end of most: it is 0 whatever K and V of
    the sequence's own keys hold, split over the keys or not; a row that is there
    sees its window and nothing else."""
    lengths, N, at, window = [0, 5, 40, 60, 61, 100], 100, 60, 20
    B = len(lengths)
    q, k, v = (randn(i, (B, h, n, D), dt) for i, h, n in ((1, H, 1), (2, Hkv, N), (3, Hkv, N)))
    for b, n in enumerate(lengths):
        seen = range(at + 1 - window, at + 1) if n > at else ()
        hidden = [j for j in range(N) if j not in seen]
        k[b, :, hidden] = bad
        v[b, :, hidden] = bad
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    rows = {}
    for b, length in enumerate(lengths):
        for h in range(H):
            rows[b, h, 0] = (np.zeros(D), np.zeros(D)) if length <= at else attend_row(
                f64(q[b, h, 0]), f64(k[b, h * Hkv // H]), f64(v[b, h * Hkv // H]), at, length, window=window, dtype=dt,
                out_dtype=dt)
    for splits in (0, 1):
        out = ofh.window_attention(q.cuda(), k.cuda(), v.cuda(), lengths=n, query_offset=at, window=window,
                                   max_key_splits=splits)
        compare(out, rows, dt, f"single rows {dt} H{H}/{Hkv} D{D} splits {splits}")
    # without a window, every sequence shorter than the position
    n = torch.tensor([min(x, at) for x in lengths], dtype=torch.int32).cuda()
    for splits in (0, 1):
        out = ofh.window_attention(q.cuda(), k.cuda(), v.cuda(), lengths=n, query_offset=at, max_key_splits=splits)
        assert int(out.ne(0).sum()) == 0


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,Hkv", [(2, 2), (16, 1), (32, 1), (32, 2)])
@pytest.mark.parametrize("options", [dict(), dict(window=16, sink_tokens=2)])
@pytest.mark.parametrize("bad", [NAN, math.inf])
def test_padding_rows_of_prompts(ofh, dt, H, Hkv, options, bad):
    """A padded batch whose last real key of each sequence has a bad V: the row at
    that position sees it, the rows before it are as without it, the padding rows
    are 0. (Groups of 16 and 32 heads fill a tile with one token.)"""
    lengths, N, D = [0, 1, 17, 33, 46, 47], 47, 64
    B = len(lengths)
    q, k, v = (randn(i, (B, h, N, D), dt) for i, h in ((1, H), (2, Hkv), (3, Hkv)))
    for b, n in enumerate(lengths):
        if n:
            v[b, :, n - 1] = bad
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    out = ofh.window_attention(q.cuda(), k.cuda(), v.cuda(), lengths=n, **options)
    clean = torch.nan_to_num(v, nan=0.0, posinf=0.0)
    rows = {}
    for b, length in enumerate(lengths):
        if length:
            assert not np.isfinite(f64(out[b, :, length - 1])).any()
        for h in (0, H // 2, H - 1):
            for t in range(N):
                if t >= length:
                    rows[b, h, t] = (np.zeros(D), np.zeros(D))
                elif t < length - 1:
                    rows[b, h, t] = attend_row(f64(q[b, h, t]), f64(k[b, h * Hkv // H]), f64(clean[b, h * Hkv // H]), t,
                                               length, window=options.get("window", 0),
                                               sinks=options.get("sink_tokens", 0), dtype=dt, out_dtype=dt)
    compare(out, rows, dt, f"padded prompts {dt} H{H}/{Hkv} {options}")
