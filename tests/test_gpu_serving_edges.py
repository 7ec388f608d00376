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


# --- soft-caps far from the scores --------------------------------------------

def capped_row(q, k, v, position, scale, slope, cap, dt):
    """The row of attend_row with a soft-cap, and its bound where the cap's error goes
    by the score's size instead of the cap's: 16 u |y| (of z = y / cap, its square,
    the fraction's two polynomials and their quotient, each a rounding or two, and past
    |z| = 1 a few u cap < 1.4 u |y|)."""
    u = 2.0 ** -24
    j = np.arange(position + 1)
    k, v = k[j], v[j]
    bias = slope * (j - position)
    y = (k @ q) * scale + bias
    err = q.size * u * (np.abs(k) @ np.abs(q)) * scale + 6 * u * (np.abs(y) + np.abs(bias)) + 16 * u * np.abs(y)
    cap = float(np.float32(cap))
    x = cap * np.tanh(y / cap)
    err += 2 * u * (np.abs(x) + abs(x.max()) + 8)
    w = np.exp(x - x.max())
    w /= w.sum()
    o = w @ v
    half = {"f32": 0.0, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[dt]
    e = err + 2 * u + half
    bound = (w * e) @ np.abs(v - o) / (1 - e.max()) + (j.size + 8) * u * (w @ np.abs(v) + np.abs(o))
    return o, bound + 1e-30


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("scale,cap", [(0.125, 257.0), (8.0, 300.0), (0.125, 3e4), (0.125, 1e9), (0.125, 3e38), (8.0, 1e6)])
def test_large_soft_caps(ofh, dt, slopes, scale, cap):
    """Caps far past the scores leave them as they are, in every kernel."""
    H, N, D = 4, 150, 64
    q, k, v = (randn(i, (1, h, N, D), dt) for i, h in ((1, H), (2, 1), (3, 1)))
    alibi = 2.0 ** -torch.arange(1.0, H + 1)
    given = alibi.cuda() if slopes else None
    options = dict(scale=scale, softcap=cap, alibi_slopes=given, out_dtype=torch.float32)
    table = torch.arange(10, dtype=torch.int32)[None].cuda()
    pools = [torch.nn.functional.pad(t, (0, 0, 0, 160 - N)).view(10, 1, 16, D).cuda() for t in (k[0, 0], v[0, 0])]
    n = torch.tensor([N], dtype=torch.int32).cuda()
    for M, out in [(N, ofh.window_attention(q.cuda(), k.cuda(), v.cuda(), **options)),
                   (1, ofh.window_attention(q[:, :, N - 1:].cuda(), k.cuda(), v.cuda(), query_offset=N - 1, **options)),
                   (3, ofh.paged_attention(q[:, :, N - 3:].cuda(), *pools, table, n, **options))]:
        rows = {(0, h, t): capped_row(f64(q[0, h, N - M + t]), f64(k[0, 0]), f64(v[0, 0]), N - M + t, scale,
                                      float(alibi[h]) if slopes else 0.0, cap, dt)
                for h in range(H) for t in sorted({0, M // 3, M // 2, M - 1})}
        compare(out, rows, dt, f"cap {cap} {dt} scale {scale} M{M}")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [48, 128, 256])
@pytest.mark.parametrize("B,H,N", [(1, 2, 150), (8, 16, 300)])
def test_large_soft_caps_by_head_dim(ofh, dt, D, B, H, N):
    """Every head dim's kernels, with 64 and with 128 rows per workgroup."""
    q, k, v = (randn(i, (B, h, N, D), dt) for i, h in ((1, H), (2, 1), (3, 1)))
    scale, cap = 1.0 / math.sqrt(D), 1e5
    out = ofh.window_attention(q.cuda(), k.cuda(), v.cuda(), softcap=cap, out_dtype=torch.float32)
    rows = {(b, h, t): capped_row(f64(q[b, h, t]), f64(k[b, 0]), f64(v[b, 0]), t, scale, 0.0, cap, dt)
            for b in {0, B - 1} for h in {0, H - 1} for t in (0, 63, N - 1)}
    compare(out, rows, dt, f"cap {cap} {dt} B{B} H{H} N{N} D{D}")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cap", [1e-45, 1e-39, 1e-30, 1e-13])
def test_tiny_soft_caps(ofh, dt, cap):
    """Caps next to zero leave every score next to zero: the mean of the values that
    are seen, also where a score is exactly 0 and the cap is subnormal."""
    H, N, D = 4, 150, 64
    q, k, v = (randn(i, (1, h, N, D), dt) for i, h in ((1, H), (2, 1), (3, 1)))
    k[0, 0, ::5] = 0.0
    for M in (N, 1):
        out = ofh.window_attention(q[:, :, N - M:].cuda(), k.cuda(), v.cuda(), query_offset=N - M, softcap=cap,
                                   out_dtype=torch.float32)
        rows = {(0, h, t): capped_row(f64(q[0, h, N - M + t]), f64(k[0, 0]), f64(v[0, 0]), N - M + t, 0.125, 0.0,
                                      max(cap, 1e-30), dt) for h in range(H) for t in sorted({0, M // 2, M - 1})}
        compare(out, rows, dt, f"cap {cap} {dt} M{M}")


# --- page numbers ------------------------------------------------------------

@pytest.mark.parametrize("numbers", [[1.5], [1.0, 2.0], [True], [False, 1], ["1"], [None], np.array([1.0]), torch.tensor([1.5]),
                                     torch.tensor([True])])
def test_page_numbers_are_integers(ofh, numbers):
    """What is no integer is refused, not rounded to a page; nothing is copied."""
    pool = torch.arange(8.0 * 16, device="cuda").view(8, 16)
    before = pool.clone()
    other = [5, 6][:len(numbers)]
    for src, dst in ((numbers, other), (other, numbers)):
        with pytest.raises(ValueError, match="integers"):
            ofh.copy_pages([pool], src, dst)
    assert torch.equal(pool, before)


@pytest.mark.parametrize("numbers", [[1, 2], (1, 2), range(1, 3), np.array([1, 2]), [np.int32(1), np.int64(2)],
                                     torch.tensor([1, 2]), torch.tensor([1, 2], dtype=torch.int32),
                                     [torch.tensor(1), torch.tensor(2)]])
def test_page_numbers_of_every_integer_kind(ofh, numbers):
    pool = torch.arange(8.0 * 16, device="cuda").view(8, 16)
    want = pool.clone()
    want[5:7] = want[1:3]
    ofh.copy_pages([pool], numbers, [5, 6])
    assert torch.equal(pool, want)
    with pytest.raises(ValueError, match="within the pool"):
        ofh.copy_pages([pool], [1 << 70], [1])


# --- a batch with uneven numbers of new tokens ----------------------------------

@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_uneven_batches_by_their_last_tokens(ofh, dt):
    """write takes the rows of each sequence from the front; attend the last tokens
    that every sequence has, and no more."""
    import onednn_flash_cache as C
    H, D, counts = 4, 64, [5, 2, 3]
    cache = C.PagedCache(layers=1, num_pages=12, page_size=16, kv_heads=1, head_dim=D, dtype=TYPES[dt])
    seqs = [cache.add() for _ in counts]
    first = cache.extend(seqs, [17, 17, 17])
    old = [randn(i, (3, 1, 17, D), dt) for i in (1, 2)]
    first.write(0, *(t.cuda() for t in old))
    batch = cache.extend(seqs, counts)
    new = [randn(i, (3, 1, 5, D), dt) for i in (3, 4)]
    batch.write(0, *(t.cuda() for t in new))
    q = randn(5, (3, H, 2, D), dt)
    rows = {}
    for b, n in enumerate(counts):
        k, v = (f64(torch.cat([o[b, 0], t[b, 0, :n]])) for o, t in zip(old, new))
        for h in range(H):
            for t in range(2):
                rows[b, h, t] = attend_row(f64(q[b, h, t]), k, v, 17 + n - 2 + t, 17 + n, dtype=dt, out_dtype=dt)
    compare(batch.attend(0, q.cuda()), rows, dt, f"uneven batch {dt}")
    with pytest.raises(ValueError, match="q has 5 tokens"):
        batch.attend(0, randn(5, (3, H, 5, D), dt).cuda())


# --- streams -------------------------------------------------------------------

def test_a_torch_stream_given(ofh):
    """A torch stream in place of its handle, also for calls that take scratch on it."""
    side = torch.cuda.Stream()
    q = randn(1, (1, 8, 1, 128), "bf16").cuda()
    k = randn(2, (1, 2, 6000, 128), "bf16").cuda()
    pools = k.view(2, 375, 16, 128).transpose(0, 1).contiguous()
    table = torch.arange(375, dtype=torch.int32)[None].cuda()
    n = torch.tensor([6000], dtype=torch.int32).cuda()
    attend = ofh.PagedAttention(pools, pools, table, n, heads=8)
    assert attend.workspace_bytes > 0
    want = ofh.window_attention(q, k, k, query_offset=5999), attend(q)
    row, pool = randn(3, (1, 2, 1, 128), "bf16").cuda(), pools.clone()
    torch.cuda.synchronize()
    got = ofh.window_attention(q, k, k, query_offset=5999, stream=side), attend(q, stream=side)
    ofh.cache_write(row, row, pool, pool, table, n, stream=side)
    ofh.copy_pages([pool], [374], [0], stream=side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(pool[374, :, 15], row[0, :, 0]) and torch.equal(pool[0], pool[374])


# --- workspaces ------------------------------------------------------------------

def test_an_empty_workspace_is_none_of_the_librarys(ofh):
    """A given workspace is the one that a call uses: an empty one is refused where
    scratch is needed, and does where it is not."""
    q = randn(1, (1, 8, 1, 128), "bf16").cuda()
    k = randn(2, (1, 2, 6000, 128), "bf16").cuda()
    pools = k.view(2, 375, 16, 128).transpose(0, 1).contiguous()
    table = torch.arange(375, dtype=torch.int32)[None].cuda()
    n = torch.tensor([6000], dtype=torch.int32).cuda()
    empty = torch.empty(0, dtype=torch.uint8, device="cuda")
    for call in (lambda **o: ofh.window_attention(q, k, k, query_offset=5999, **o),
                 lambda **o: ofh.paged_attention(q, pools, pools, table, n, **o)):
        with pytest.raises(ofh.OfhError) as e:
            call(workspace=empty)
        assert e.value.code == ofh.OFH_ERROR_WORKSPACE_TOO_SMALL
        assert torch.equal(call(workspace=empty, max_key_splits=1), call(max_key_splits=1))
        assert torch.equal(call(workspace=torch.empty(1 << 24, dtype=torch.uint8, device="cuda")), call())


# --- many tokens in one write ------------------------------------------------------

def test_writes_of_half_a_million_tokens(ofh):
    """32 prompts of 16384 tokens and 32 heads: as many work items as 16-byte chunks
    need, which a launch holds. (One sequence's rows stand for all of them, and only
    the last pages of two sequences have a place.)"""
    B, H, T, D, page = 32, 32, 16384, 128, 16
    k = randn(1, (1, H, T, D), "bf16").cuda()
    v = randn(2, (1, H, T, D), "bf16").cuda()
    pools = [torch.full((3, H, page, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    table = torch.full((B, T // page), -1, dtype=torch.int32)
    table[0, -1], table[B - 1, -1] = 2, 0
    n = torch.full((B,), T, dtype=torch.int32).cuda()
    ofh.cache_write(k.expand(B, H, T, D), v.expand(B, H, T, D), *pools, table.cuda(), n)
    for rows, pool in ((k, pools[0]), (v, pools[1])):
        last = rows[0, :, T - page:]
        assert torch.equal(pool[2], last) and torch.equal(pool[0], last) and bool((pool[1] == 7.0).all())
