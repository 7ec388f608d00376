"""GPU parity of the serving operators against the plain 64-bit implementation
of serving_ref.py, within the bound that it derives from the arithmetic."""

from __future__ import annotations

import math
import threading

import numpy as np
import pytest

from serving_ref import attend_row

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NAN = float("nan")


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def randn(seed, shape, dt):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=gen).to(TYPES[dt])


def f64(t):
    return t.detach().cpu().double().numpy()


def compare(out, rows, dt, label):
    """rows: (b, h, t) -> (value, bound)."""
    out = f64(out)
    worst = 0.0
    for at, (ref, bound) in rows.items():
        got = out[at]
        assert np.isfinite(got).all(), f"{label}: row {at} is not finite"
        off = np.abs(got - ref)
        worst = max(worst, float((off / (bound + 1e-300)).max()))
        assert (off <= bound).all(), f"{label}: row {at} off by {off.max():.3e}, bound {bound[off.argmax()]:.3e}"
    print(f"{label}: at most {worst:.2f} of the bound", flush=True)


def pick(n, most, seed):
    """All of range(n), or `most` of them with both ends."""
    if n <= most:
        return list(range(n))
    mid = np.random.default_rng(seed).choice(n - 2, most - 2, replace=False) + 1
    return [0, *sorted(int(i) for i in mid), n - 1]


# --- windowed attention -----------------------------------------------------

def check_window(F, dt, B, H, Hkv, M, N, D, Dv=None, *, lengths=None, slopes=False, seed=0, out_f32=False, rows=24,
                 q=None, k=None, v=None, splits=0, **options):
    Dv = Dv or D
    q = randn(seed, (B, H, M, D), dt) if q is None else q
    k = randn(seed + 1, (B, Hkv, N, D), dt) if k is None else k
    v = randn(seed + 2, (B, Hkv, N, Dv), dt) if v is None else v
    alibi = 2.0 ** -torch.arange(1.0, H + 1) if slopes else None
    out = F.window_attention(
        q.cuda(), k.cuda(), v.cuda(), lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32).cuda(),
        alibi_slopes=None if alibi is None else alibi.cuda(), out_dtype=torch.float32 if out_f32 else None,
        max_key_splits=splits, **options)
    offset = options.get("query_offset", 0)
    ref = {}
    for b in range(B):
        n = N if lengths is None else max(0, min(lengths[b], N))
        for h in pick(H, 5, seed):
            for t in pick(M, rows, seed + h):
                if lengths is not None and offset + t >= n:
                    ref[b, h, t] = (np.zeros(Dv), np.zeros(Dv))
                    continue
                ref[b, h, t] = attend_row(
                    f64(q[b, h, t]), f64(k[b, h * Hkv // H]), f64(v[b, h * Hkv // H]), offset + t, n,
                    window=options.get("window", 0), sinks=options.get("sink_tokens", 0),
                    scale=options.get("scale"), slope=float(alibi[h]) if slopes else 0.0,
                    softcap=options.get("softcap", 0.0), dtype=dt, out_dtype="f32" if out_f32 else dt)
    compare(out, ref, dt, f"window {dt} B{B} H{H}/{Hkv} M{M} N{N} D{D}/{Dv} {options} lengths {lengths}")
    return out


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 33, 63, 64, 65, 200, 300])
def test_window_lengths(ofh, dt, tokens):
    for i, (window, sinks) in enumerate([(0, 0), (1, 0), (1, 1), (17, 3), (64, 64), (100, 5), (4096, 4)]):
        check_window(ofh, dt, 1, 4, 2, tokens, tokens, 64, window=window, sink_tokens=sinks, seed=7 * i)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D,Dv", [(8, 8), (32, 40), (64, 64), (80, 80), (96, 128), (128, 64), (136, 136), (192, 128), (256, 256)])
def test_window_head_dims(ofh, dt, D, Dv):
    check_window(ofh, dt, 2, 3, 1, 70, 70, D, Dv, window=33, sink_tokens=2, seed=D)
    check_window(ofh, dt, 1, 2, 2, 150, 150, D, Dv, seed=D + 1, out_f32=True)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_window_many_tiles(ofh, dt, D):
    """More tiles than the GPU runs at once: 128 rows per workgroup in 16 bits, a
    tile per wavefront in fp32; with each rule of the scores, and a NaN that half of
    the rows do not see."""
    B, H, Hkv, N = 3, 64, 16, 257
    lengths = [257, 100, 190]
    check_window(ofh, dt, B, H, Hkv, N, N, D, lengths=lengths, window=90, sink_tokens=70, seed=D)
    check_window(ofh, dt, B, H, Hkv, N, N, D, window=33, sink_tokens=1, seed=D, slopes=True, softcap=9.0)
    check_window(ofh, dt, B, H, Hkv, N, N, D, lengths=lengths, seed=D, scale=-0.1)
    q, k, v = (randn(i, (B, h, N, D), dt) for i, h in ((1, H), (2, Hkv), (3, Hkv)))
    v2 = v.clone()
    v2[:, :, 130, 5] = NAN
    clean, out = (f64(ofh.window_attention(q.cuda(), k.cuda(), t.cuda(), window=60)) for t in (v, v2))
    sees = np.array([130 <= t < 190 for t in range(N)])
    assert not np.isfinite(out[:, :, sees, 5]).any()
    tol = 1e-5 if dt == "f32" else 2.0 ** -6
    assert np.abs(out[:, :, ~sees] - clean[:, :, ~sees]).max() <= tol * np.abs(clean).max()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (8, 8), (6, 2), (5, 1), (40, 1)])
def test_window_head_groups(ofh, dt, H, Hkv):
    check_window(ofh, dt, 2, H, Hkv, 45, 45, 64, window=20, sink_tokens=4, seed=H)
    check_window(ofh, dt, 1, H, Hkv, 3, 500, 128, query_offset=497, window=300, sink_tokens=20, seed=H)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_window_scores(ofh, dt):
    for i, options in enumerate([dict(softcap=3.0), dict(slopes=True), dict(slopes=True, softcap=20.0),
                                 dict(scale=0.7), dict(scale=-0.2), dict(scale=0.0)]):
        check_window(ofh, dt, 1, 4, 2, 130, 130, 64, window=50, sink_tokens=3, seed=i, **options)
        check_window(ofh, dt, 1, 4, 4, 40, 40, 128, seed=i + 50, **options)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_window_padded_batch(ofh, dt):
    """Sequences from none to all of the rows: padding rows are zero, and what
    stands in padding (NaN) reaches nothing."""
    B, H, Hkv, N, D = 6, 4, 2, 140, 64
    lengths = [0, 1, 64, 139, 140, 500]
    q, k, v = (randn(i, (B, h, N, D), dt) for i, h in ((1, H), (2, Hkv), (3, Hkv)))
    for b, n in enumerate(lengths):
        for t in (q, k, v):
            t[b, :, n:] = NAN
    for options in (dict(), dict(window=30, sink_tokens=4), dict(window=30, sink_tokens=4, query_offset=0, softcap=5.0)):
        check_window(ofh, dt, B, H, Hkv, N, N, D, lengths=lengths, q=q, k=k, v=v, **options)
    # a chunk of a prompt against the keys so far
    q2 = randn(9, (B, H, 50, D), dt)
    check_window(ofh, dt, B, H, Hkv, 50, N, D, lengths=[0, 0, 64, 139, 140, 99], q=q2, k=torch.nan_to_num(k),
                 v=torch.nan_to_num(v), query_offset=70, window=25, sink_tokens=1)
    check_window(ofh, dt, B, H, Hkv, 50, N, D, lengths=[-7, 0, 64, 139, 140, 99], q=q2, k=torch.nan_to_num(k),
                 v=torch.nan_to_num(v), query_offset=130)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_window_more_queries_than_keys(ofh, dt):
    """Rows past the last key see the keys of their window, and rows whose window
    has left them all behind see the first tokens or nothing (0)."""
    check_window(ofh, dt, 1, 2, 1, 200, 60, 64, window=40)
    check_window(ofh, dt, 1, 2, 1, 200, 60, 64, window=40, sink_tokens=3)
    check_window(ofh, dt, 1, 2, 1, 90, 20, 128)
    check_window(ofh, dt, 1, 2, 1, 5, 20, 128, query_offset=1 << 29, window=9)
    check_window(ofh, dt, 1, 2, 1, 5, 20, 128, query_offset=1 << 29, window=9, sink_tokens=2)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N", [1, 31, 700, 5000])
def test_window_few_rows_against_many_keys(ofh, dt, N):
    """The form for single tokens, split over the keys and joined, or not."""
    for splits in (0, 1, 3):
        check_window(ofh, dt, 2, 4, 2, 1, N, 128, query_offset=N - 1, splits=splits, seed=N)
        check_window(ofh, dt, 1, 4, 4, min(N, 9), N, 64, query_offset=max(0, N - 9), splits=splits, window=N // 2 + 1,
                     sink_tokens=8, seed=N)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [NAN, math.inf])
def test_window_hidden_values_do_not_reach_a_row(ofh, dt, D, bad):
    """A NaN or an infinity in the K or V row of key j reaches the rows that see
    j and no other, also where they share every tile with it."""
    H, M, window, sinks = 2, 150, 40, 5
    q, k, v = (randn(i, (1, h, M, D), dt) for i, h in ((1, H), (2, 1), (3, 1)))
    for j in (2, 20, 77, 149):
        for which in ("k", "v"):
            k2, v2 = k.clone(), v.clone()
            (k2 if which == "k" else v2)[0, 0, j, 3] = bad
            out = f64(ofh.window_attention(q.cuda(), k2.cuda(), v2.cuda(), window=window, sink_tokens=sinks))
            clean = f64(ofh.window_attention(q.cuda(), k.cuda(), v.cuda(), window=window, sink_tokens=sinks))
            sees = np.array([j <= t and (t - j < window or j < sinks) for t in range(M)])
            assert (~np.isfinite(out[0, :, sees])).any((1, 2)).all() or which == "k"
            tol = 1e-5 if dt == "f32" else 2.0 ** -6  # the redone products may sum in another order
            assert np.isfinite(out[0, :, ~sees]).all()
            assert np.abs(out[0, :, ~sees] - clean[0, :, ~sees]).max() <= tol * np.abs(clean).max()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [24, 40, 80, 136])
def test_infinite_keys_of_a_padded_head_dim(ofh, dt, D):
    """A score of -inf through an infinity in the last columns of K is a weight of
    0, also where the kernel's columns past the head dim repeat them."""
    H, N = 2, 200
    q, k, v = (randn(i, (1, h, N, D), dt) for i, h in ((1, H), (2, 1), (3, 1)))
    q[..., D - 1] = 1.0
    k[0, 0, 3::7, D - 1] = -math.inf
    k[0, 0, :2, D - 1] = 0.5
    for M in (N, 1):  # staged through LDS, and streamed
        out = f64(ofh.window_attention(q[:, :, N - M:].cuda(), k.cuda(), v.cuda(), query_offset=N - M, window=60, sink_tokens=2))
        keep = torch.ones(N, dtype=torch.bool)
        keep[3::7] = False
        ref = {(0, h, t): attend_row(f64(q[0, h, N - M + t]), f64(torch.nan_to_num(k[0, 0], neginf=0.0)), f64(v[0, 0]),
                                     N - M + t, N, window=60, sinks=2, dtype=dt, out_dtype=dt,
                                     hidden=np.flatnonzero(~keep.numpy())) for h in range(H) for t in pick(M, 20, D)}
        compare(out if isinstance(out, torch.Tensor) else torch.from_numpy(out), ref, dt, f"infinite keys {dt} D{D} M{M}")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_window_strides(ofh, dt):
    """[B,T,H,D] storage, heads of a wider tensor, broadcast keys, an output in
    another order with what lies around it untouched."""
    B, H, Hkv, N, D = 2, 6, 3, 77, 64
    q, k, v = (randn(i, (B, h, N, D), dt).cuda() for i, h in ((1, H), (2, Hkv), (3, Hkv)))
    ref = ofh.window_attention(q, k, v, window=30, sink_tokens=2)
    qt, kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v))
    assert torch.equal(ofh.window_attention(qt, kt, vt, window=30, sink_tokens=2), ref)
    wide = torch.full((B, N + 3, H + 2, D + 16), 7.0, dtype=TYPES[dt], device="cuda")
    out = wide[:, 1:N + 1, 1:H + 1, 8:D + 8].transpose(1, 2)
    ofh.window_attention(qt, k, vt, window=30, sink_tokens=2, out=out)
    assert torch.equal(out, ref)
    assert int((wide != 7.0).sum()) <= ref.numel()
    inner = torch.zeros_like(wide, dtype=torch.bool)
    inner[:, 1:N + 1, 1:H + 1, 8:D + 8] = True
    assert bool((wide[~inner] == 7.0).all())
    one = k[:1, :1]
    shared = ofh.window_attention(q, one.expand(B, Hkv, N, D), v, window=30)
    assert torch.equal(shared, ofh.window_attention(q, one.expand(B, Hkv, N, D).contiguous(), v, window=30))
    row = k[:1, :1, :1].expand(1, 1, N, D)  # axes of one element have a stride of no meaning
    alone = ofh.window_attention(q[:1], row, v[:1, :1], window=30)
    assert torch.equal(alone, ofh.window_attention(q[:1], row.contiguous(), v[:1, :1], window=30))
    low = ofh.window_attention(q, k, v, window=30, sink_tokens=2, out_dtype=torch.float32)
    assert torch.equal(low.to(ref.dtype), ref)


# --- paged attention --------------------------------------------------------

def make_cache(dt, lengths, Hkv, D, Dv, page, seed, *, order="phsd", spare=3, width=0):
    """Pools whose places outside the sequences hold NaN, scattered pages, a table
    with nonsense past each sequence's pages; and the sequences themselves."""
    rng = np.random.default_rng(seed)
    need = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(need) + spare
    place = rng.permutation(pages)[:sum(need)]
    width = max(width, max(need), 1)
    table = rng.choice([-1, -(1 << 31), (1 << 31) - 1, pages], size=(len(lengths), width)).astype(np.int32)
    k = [randn(seed + 100 + b, (Hkv, max(n, 0), D), dt) for b, n in enumerate(lengths)]
    v = [randn(seed + 200 + b, (Hkv, max(n, 0), Dv), dt) for b, n in enumerate(lengths)]
    pools = []
    for rows, dim in ((k, D), (v, Dv)):
        pool = torch.full((pages, Hkv, page, dim), NAN, dtype=TYPES[dt])
        at = 0
        for b, n in enumerate(lengths):
            for i in range(need[b]):
                part = rows[b][:, i * page:(i + 1) * page]
                pool[int(place[at]), :, :part.shape[1]] = part
                table[b, i] = place[at]
                at += 1
        if order == "pshd":
            pool = pool.transpose(1, 2).contiguous().cuda().transpose(1, 2)
        pools.append(pool.cuda())
    return pools[0], pools[1], torch.from_numpy(table).cuda(), k, v


def check_paged(F, dt, lengths, H, Hkv, T, D, Dv=None, *, page=16, slopes=False, seed=0, out_f32=False, order="phsd",
                splits=0, says=None, **options):
    """says: the lengths that the call is given (those of the sequences)."""
    Dv = Dv or D
    B = len(lengths)
    kp, vp, table, k, v = make_cache(dt, lengths, Hkv, D, Dv, page, seed, order=order)
    q = randn(seed, (B, H, T, D), dt)
    alibi = 2.0 ** -torch.arange(1.0, H + 1) if slopes else None
    given = torch.tensor(lengths if says is None else says, dtype=torch.int32).cuda()
    out = F.paged_attention(q.cuda(), kp, vp, table, given, alibi_slopes=None if alibi is None else alibi.cuda(),
                            out_dtype=torch.float32 if out_f32 else None, max_key_splits=splits, **options)
    ref = {}
    for b, n in enumerate(lengths):
        n = max(n, 0)
        for h in pick(H, 6, seed + b):
            for t in pick(T, 6, seed + h):
                ref[b, h, t] = attend_row(
                    f64(q[b, h, t]), f64(k[b][h * Hkv // H]), f64(v[b][h * Hkv // H]), n - T + t, n,
                    window=options.get("window", 0), sinks=options.get("sink_tokens", 0), scale=options.get("scale"),
                    slope=float(alibi[h]) if slopes else 0.0, softcap=options.get("softcap", 0.0), dtype=dt,
                    out_dtype="f32" if out_f32 else dt)
    compare(out, ref, dt, f"paged {dt} {lengths} H{H}/{Hkv} T{T} D{D}/{Dv} page {page} splits {splits} {options}")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_paged_lengths(ofh, dt, page):
    lengths = [0, 1, 2, 15, 16, 17, 31, 33, 127, 128, 129, 300]
    for T in (1, 3):
        check_paged(ofh, dt, lengths, 8, 2, T, 64, page=page, seed=T)
        check_paged(ofh, dt, lengths, 4, 4, T, 128, page=page, seed=T, window=20, sink_tokens=5)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D,Dv", [(8, 8), (40, 32), (64, 64), (80, 80), (128, 128), (96, 136), (192, 128), (256, 256)])
def test_paged_head_dims(ofh, dt, D, Dv):
    check_paged(ofh, dt, [70, 9], 6, 2, 1, D, Dv, seed=D)
    check_paged(ofh, dt, [70, 200], 6, 2, 2, D, Dv, seed=D, out_f32=True, window=50, sink_tokens=1)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,Hkv,T", [(1, 1, 1), (16, 1, 1), (17, 1, 1), (64, 2, 1), (8, 8, 5), (8, 1, 8), (12, 4, 16), (3, 3, 40)])
def test_paged_rows(ofh, dt, H, Hkv, T):
    """One to several tiles of rows, rows of one token and of many in a tile."""
    for D in (64, 128, 256):
        check_paged(ofh, dt, [90, T, 33], H, Hkv, T, D, seed=H + T)
        check_paged(ofh, dt, [190, T + 1, 33], H, Hkv, T, D, seed=H + T, window=24, sink_tokens=3)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("splits", [0, 1, 2, 7, 64])
def test_paged_splits(ofh, dt, splits):
    """Sequences of very different lengths: each is split by its own."""
    check_paged(ofh, dt, [4000, 3, 700, 0, 257], 8, 2, 1, 128, splits=splits, seed=splits)
    check_paged(ofh, dt, [2500, 100], 4, 1, 3, 64, splits=splits, page=64, seed=splits, window=2000, sink_tokens=70)
    check_paged(ofh, dt, [1500], 2, 1, 1, 256, splits=splits, page=32, seed=splits, out_f32=True)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_paged_scores(ofh, dt):
    for i, options in enumerate([dict(softcap=3.0), dict(slopes=True), dict(slopes=True, softcap=20.0), dict(scale=0.7),
                                 dict(scale=-0.2)]):
        check_paged(ofh, dt, [130, 1000], 4, 2, 2, 64, seed=i, **options)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_paged_layouts(ofh, dt):
    check_paged(ofh, dt, [130, 50], 4, 2, 1, 64, order="pshd", page=32)
    check_paged(ofh, dt, [130, 50], 4, 2, 3, 128, order="pshd", window=17)
    # lengths that the table cannot hold are taken as what it holds; negative ones as none
    check_paged(ofh, dt, [64, -5], 4, 2, 1, 64, says=[1 << 30, -5])
    B, H, T, D = 2, 4, 3, 64
    kp, vp, table, _, _ = make_cache(dt, [100, 70], 2, D, D, 16, 5)
    q = randn(1, (B, H, T, D), dt).cuda()
    n = torch.tensor([100, 70], dtype=torch.int32).cuda()
    ref = ofh.paged_attention(q, kp, vp, table, n)
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ofh.paged_attention(qt, kp, vp, table, n), ref)
    wide = torch.full((B, T, H + 1, D), 7.0, dtype=TYPES[dt], device="cuda")
    ofh.paged_attention(qt, kp, vp, table, n, out=wide[:, :, :H].transpose(1, 2))
    assert torch.equal(wide[:, :, :H].transpose(1, 2), ref) and bool((wide[:, :, H] == 7.0).all())
    # a table in a wider one, pools inside larger tensors
    big = torch.full((4, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    big[1:3, :table.shape[1]] = table
    assert torch.equal(ofh.paged_attention(q, kp, vp, big[1:3, :table.shape[1]], n), ref)
    both = torch.stack([kp, vp], 1)
    assert torch.equal(ofh.paged_attention(q, both[:, 0], both[:, 1], table, n), ref)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_paged_bad_entries_are_not_seen(ofh, dt):
    """The keys of a table entry outside the pool count for nothing."""
    for D, T in ((64, 1), (128, 2), (256, 1)):
        lengths = [200, 40]
        kp, vp, table, k, v = make_cache(dt, lengths, 1, D, D, 16, D)
        table[0, 3], table[0, 7], table[0, 8], table[1] = -1, kp.shape[0], (1 << 31) - 1, -9
        q = randn(3, (2, 2, T, D), dt)
        out = ofh.paged_attention(q.cuda(), kp, vp, table, torch.tensor(lengths, dtype=torch.int32).cuda())
        hidden = np.concatenate([np.arange(48, 64), np.arange(112, 144)])
        ref = {(0, h, t): attend_row(f64(q[0, h, t]), f64(k[0][0]), f64(v[0][0]), 200 - T + t, 200, dtype=dt,
                                     out_dtype=dt, hidden=hidden) for h in range(2) for t in range(T)}
        ref |= {(1, h, t): (np.zeros(D), np.zeros(D)) for h in range(2) for t in range(T)}
        compare(out, ref, dt, f"bad entries {dt} D{D}")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [NAN, math.inf])
def test_paged_hidden_values_do_not_reach_a_row(ofh, dt, bad):
    """With several new tokens: a draft token's key reaches it and those after it only."""
    for D, H in ((64, 2), (128, 1), (256, 3)):
        T, n, window = 6, 150, 40
        kp, vp, table, _, _ = make_cache(dt, [n], 1, D, D, 16, D)
        q = randn(3, (1, H, T, D), dt).cuda()
        length = torch.tensor([n], dtype=torch.int32).cuda()
        clean = f64(ofh.paged_attention(q, kp, vp, table, length, window=window))
        for j in (n - 1, n - 4, n - T - window + 3):
            page, row = int(table[0, j // 16]), j % 16
            v2 = vp.clone()
            v2[page, 0, row, 5] = bad
            out = f64(ofh.paged_attention(q, kp, v2, table, length, window=window))
            for t in range(T):
                p = n - T + t
                if j <= p and p - j < window:
                    assert not np.isfinite(out[0, :, t, 5]).any()
                    out[0, :, t, 5] = clean[0, :, t, 5]
            tol = 1e-5 if dt == "f32" else 2.0 ** -6
            assert np.abs(out - clean).max() <= tol * np.abs(clean).max()


def test_paged_offsets_past_32_bits(ofh):
    """A pool of more than 2^32 elements, the sequence in its last pages."""
    Hkv, S, D = 8, 16, 128
    pages = (1 << 32) // (Hkv * S * D) + 64
    pools = [torch.empty((pages, Hkv, S, D), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    n = 100
    k, v = randn(1, (Hkv, 112, D), "bf16"), randn(2, (Hkv, 112, D), "bf16")
    table = torch.arange(pages - 1, pages - 8, -1, dtype=torch.int32)
    lengths = torch.tensor([n], dtype=torch.int32).cuda()
    ofh.cache_write(k[None, :, :n].cuda(), v[None, :, :n].cuda(), *pools, table[None].cuda(), lengths)
    for i, p in enumerate(table.tolist()):
        m = min(16, n - 16 * i)
        assert torch.equal(pools[0][p, :, :m].cpu(), k[:, 16 * i:16 * i + m])
        assert torch.equal(pools[1][p, :, :m].cpu(), v[:, 16 * i:16 * i + m])
    ofh.copy_pages(pools, table.tolist(), list(range(7)))
    q = randn(3, (1, Hkv, 1, D), "bf16")
    far = ofh.paged_attention(q.cuda(), *pools, table[None].cuda(), lengths)
    near = ofh.paged_attention(q.cuda(), *pools, torch.arange(7, dtype=torch.int32)[None].cuda(), lengths)
    assert torch.equal(far, near)
    ref = {(0, h, 0): attend_row(f64(q[0, h, 0]), f64(k[h]), f64(v[h]), n - 1, n, dtype="bf16", out_dtype="bf16")
           for h in range(Hkv)}
    compare(far, ref, "bf16", "far pages")


def test_results_repeat(ofh):
    """The joined parts are added in one order: the same call gives the same bits."""
    kp, vp, table, _, _ = make_cache("bf16", [5000, 900], 2, 128, 128, 16, 1)
    q = randn(1, (2, 8, 1, 128), "bf16").cuda()
    n = torch.tensor([5000, 900], dtype=torch.int32).cuda()
    first = ofh.paged_attention(q, kp, vp, table, n)
    for _ in range(20):
        assert torch.equal(ofh.paged_attention(q, kp, vp, table, n), first)


# --- cache writes and page copies --------------------------------------------

@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D,Dv", [(64, 64), (128, 128), (1, 3), (6, 10), (96, 32)])
@pytest.mark.parametrize("page", [16, 64])
def test_cache_write(ofh, dt, D, Dv, page):
    """Rows land where the table says and nothing else changes: counts of none to
    all, rows before the first position, past the table and outside the pool
    left out."""
    B, Hkv, T, width = 7, 3, 21, 6
    pages = B * width + 2
    rng = np.random.default_rng(D + page)
    table = rng.permutation(pages)[:B * width].reshape(B, width).astype(np.int32)
    counts = np.array([21, 0, 5, 21, 1, 30, 8], np.int32)
    lengths = np.array([21, 40, 33, 9, 16, 6 * page, 6 * page + 4], np.int32)
    table[2, 1 if page == 16 else 0] = -1
    table[4, 0] = pages
    k, v = randn(1, (B, Hkv, T, D), dt), randn(2, (B, Hkv, T, Dv), dt)
    for source in ("bhtd", "bthd"):
        pools = [randn(5, (pages, Hkv, page, D), dt), randn(6, (pages, Hkv, page, Dv), dt)]
        want = [t.clone() for t in pools]
        for b in range(B):
            count = min(int(counts[b]), T)
            for t in range(count):
                pos = int(lengths[b]) - count + t
                if pos < 0 or pos >= width * page or not 0 <= table[b, pos // page] < pages:
                    continue
                want[0][table[b, pos // page], :, pos % page] = k[b, :, t]
                want[1][table[b, pos // page], :, pos % page] = v[b, :, t]
        kd, vd = k.cuda(), v.cuda()
        got = [t.cuda() for t in pools]
        if source == "bthd":
            kd, vd = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kd, vd))
            got = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in got]
        ofh.cache_write(kd, vd, *got, torch.from_numpy(table).cuda(), torch.from_numpy(lengths).cuda(),
                        counts=torch.from_numpy(counts).cuda())
        for g, w in zip(got, want):
            assert torch.equal(g.cpu(), w)


def test_cache_write_without_counts(ofh):
    """Every row is a token; one token per sequence."""
    k, v = randn(1, (3, 2, 1, 64), "bf16"), randn(2, (3, 2, 1, 64), "bf16")
    pools = [torch.zeros(9, 2, 16, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    table = torch.tensor([[4, 2], [8, 0], [1, 3]], dtype=torch.int32)
    lengths = [16, 17, 1]
    ofh.cache_write(k.cuda(), v.cuda(), *pools, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())
    for pool, rows in zip(pools, (k, v)):
        for b, n in enumerate(lengths):
            assert torch.equal(pool[table[b, (n - 1) // 16], :, (n - 1) % 16].cpu(), rows[b, :, 0])
        assert int((pool != 0).any(-1).sum()) == 6


@pytest.mark.parametrize("dt,shape", [("bf16", (2, 16, 128)), ("f16", (1, 16, 24)), ("f32", (3, 5)), ("bf16", (1, 7, 3)), ("bf16", (40, 64, 130))])
@pytest.mark.parametrize("moved", [1, 7, 400])
def test_copy_pages(ofh, dt, shape, moved):
    """More pairs and pools than a launch holds; pages that are no multiple of a chunk."""
    pages = 2 * moved + 5 if len(shape) < 3 or shape[0] < 40 else 20
    moved = min(moved, pages // 2 - 1)
    count = 130 if moved == 7 and len(shape) == 2 else 3
    pools = [randn(i, (pages, *shape), dt).cuda() for i in range(count)]
    want = [t.clone() for t in pools]
    order = np.random.default_rng(moved).permutation(pages)
    src, dst = order[:moved].astype(np.int32), order[moved:2 * moved].astype(np.int32)
    for t in want:
        t[torch.from_numpy(dst).long().cuda()] = t[torch.from_numpy(src).long().cuda()]
    ofh.copy_pages(pools, torch.from_numpy(src), dst.tolist())
    for g, w in zip(pools, want):
        assert torch.equal(g, w)


def test_copy_pages_of_a_wider_tensor(ofh):
    """Pages with something between them, which stays."""
    wide = torch.arange(20 * 40, dtype=torch.float32, device="cuda").reshape(20, 40)
    want = wide.clone()
    want[3, :30] = want[11, :30]
    ofh.copy_pages([wide[:, :30]], [11], [3])
    assert torch.equal(wide, want)
    # one page read for several
    ofh.copy_pages([wide], [7, 7, 7], [0, 1, 2])
    assert torch.equal(wide[:3], wide[7].expand(3, 40))


# --- how calls are made ----------------------------------------------------------

def _calls(F, seed=0):
    """One call of each operator on tensors of its own: (call, outputs)."""
    kp, vp, table, _, _ = make_cache("bf16", [3000, 500], 2, 128, 128, 16, seed)
    kp, vp = torch.nan_to_num(kp), torch.nan_to_num(vp)
    n = torch.tensor([3000, 500], dtype=torch.int32).cuda()
    q = randn(seed, (2, 8, 1, 128), "bf16").cuda()
    rows = randn(seed + 1, (2, 2, 1, 128), "bf16").cuda()
    p = randn(seed + 2, (2, 8, 300, 128), "bf16").cuda()
    pk = randn(seed + 3, (2, 2, 300, 128), "bf16").cuda()
    lengths = torch.tensor([300, 120], dtype=torch.int32).cuda()
    free = [i for i in range(kp.shape[0]) if i not in set(table.flatten().tolist())]

    def call():
        F.cache_write(rows, rows, kp, vp, table, n)
        F.copy_pages([kp, vp], [int(table[0, 0])], [free[0]])
        return [F.paged_attention(q, kp, vp, table, n), F.window_attention(p, pk, pk, window=64, sink_tokens=4,
                                                                           lengths=lengths), kp, vp]
    return call


def test_other_streams_and_threads(ofh):
    calls = [_calls(ofh, seed) for seed in range(4)]
    want = [[t.clone() for t in call()] for call in calls]
    torch.cuda.synchronize()
    got, streams = [None] * 4, [torch.cuda.Stream() for _ in range(4)]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(10):
                got[i] = calls[i]()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_a_stream_handle_given(ofh):
    """Calls on a stream that is not the current one, whose scratch is freed as they
    return while the stream still has them to run."""
    F = ofh
    side = torch.cuda.Stream()
    kp, vp, table, _, _ = make_cache("bf16", [6000], 2, 128, 128, 16, 4)
    n = torch.tensor([6000], dtype=torch.int32).cuda()
    q = randn(4, (1, 8, 1, 128), "bf16").cuda()
    attend = F.PagedAttention(kp, vp, table, n, heads=8)
    assert attend.workspace_bytes > 0
    want = attend(q)
    k = randn(5, (1, 2, 6000, 128), "bf16").cuda()
    alone = F.window_attention(q, k, k, query_offset=5999)
    torch.cuda.synchronize()
    outs = []
    torch.cuda._sleep(20_000_000)  # the side stream waits, the host goes on
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        outs.append((attend(q, stream=side.cuda_stream), F.window_attention(q, k, k, query_offset=5999, stream=side.cuda_stream)))
        for _ in range(8):  # what the current stream allocates now must not be that scratch
            torch.empty(attend.workspace_bytes, dtype=torch.uint8, device="cuda").fill_(255)
    torch.cuda.synchronize()
    for a, b in outs:
        assert torch.equal(a, want) and torch.equal(b, alone)


def test_captured_and_replayed(ofh):
    """Two graphs captured on one stream, replayed in turn with eager calls
    between them and at the same time: each replay is the eager result of the
    inputs as they are then."""
    def program(seed):
        kp, vp, table, _, _ = make_cache("bf16", [3000], 2, 128, 128, 16, seed)
        kp, vp = torch.nan_to_num(kp), torch.nan_to_num(vp)
        n = torch.tensor([2990], dtype=torch.int32).cuda()
        q, rows = randn(seed, (1, 8, 1, 128), "bf16").cuda(), randn(seed + 1, (1, 2, 1, 128), "bf16").cuda()
        attend = ofh.PagedAttention(kp, vp, table, n, heads=8)
        writer = ofh.CacheWriter(kp, vp, table, n)

        def step():
            writer(rows, rows)
            return attend(q)
        return step, (q, rows, n)

    programs = [program(0), program(10)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for step, _ in programs:
            step()
        for step, _ in programs:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(step())
            graphs.append(g)
    torch.cuda.synchronize()
    for it in range(4):
        for i, (step, (q, rows, n)) in enumerate(programs):
            q.copy_(randn(100 + it, q.shape, "bf16"))
            rows.copy_(randn(200 + it, rows.shape, "bf16"))
            n.fill_(2990 + it)
            graphs[i].replay()
            torch.cuda.synchronize()
            got = outs[i].clone()
            assert torch.equal(step(), got)
    want = [o.clone() for o in outs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_scratch_of_the_library(ofh):
    """C callers without a workspace: the stream's scratch, and under capture, where
    it cannot grow, the call unsplit."""
    import ctypes
    F = ofh
    kp, vp, table, _, _ = make_cache("bf16", [3000], 2, 128, 128, 16, 3)
    n = torch.tensor([3000], dtype=torch.int32).cuda()
    q = randn(3, (1, 8, 1, 128), "bf16").cuda()
    want = F.paged_attention(q, kp, vp, table, n)
    alone = F.paged_attention(q, kp, vp, table, n, max_key_splits=1)
    attend = F.PagedAttention(kp, vp, table, n, heads=8)
    assert attend.workspace_bytes > 0
    out = torch.empty_like(want)
    p = F.PagedParams.from_buffer_copy(attend._params)
    args = [ctypes.addressof(p), q.data_ptr(), kp.data_ptr(), vp.data_ptr(), out.data_ptr(), None, 0]
    side = torch.cuda.Stream()
    F.check(F.lib().ofh_paged_attention_fwd(*args, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    out.zero_()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        F.check(F.lib().ofh_paged_attention_fwd(*args, side.cuda_stream))
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) or torch.equal(out, alone)


def test_python_refusals(ofh):
    F = ofh
    q = torch.zeros(1, 4, 3, 64, device="cuda")
    k = torch.zeros(1, 2, 5, 64, device="cuda")
    pool = torch.zeros(8, 2, 16, 64, device="cuda")
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    n = torch.ones(1, dtype=torch.int32, device="cuda")
    for call, text in [
            (lambda: F.window_attention(q, k[:, :, :, :32], k), "k must be"),
            (lambda: F.window_attention(q, k.half(), k), "k must be torch.float32"),
            (lambda: F.window_attention(q, k, k, window=-1), "window must be"),
            (lambda: F.window_attention(q, k, k, window=2.0), "window must be"),
            (lambda: F.window_attention(q, k, k, lengths=n.long()), "lengths must be an int32"),
            (lambda: F.window_attention(q, k, k, lengths=n.cpu()), "lengths must be on"),
            (lambda: F.window_attention(q, k, k, alibi_slopes=torch.ones(3, device="cuda")), "alibi_slopes"),
            (lambda: F.window_attention(q, k, k, out=torch.zeros(1, 4, 3, 32, device="cuda")), "out must have shape"),
            (lambda: F.window_attention(q, k, k, out=torch.zeros(1, 4, 1, 64, device="cuda").expand(1, 4, 3, 64)), "broadcast"),
            (lambda: F.window_attention(q, k, k, out_dtype=torch.float16), "out_dtype"),
            (lambda: F.window_attention(q.repeat(2, 1, 1, 1), k[:1, :1, :1].expand(2, 2, 5, 64), k.repeat(2, 1, 1, 1)),
             "broadcast over every axis"),
            (lambda: F.window_attention(q[:, :3], k, k), "multiple of Hkv"),
            (lambda: F.paged_attention(q, pool, pool, table.long(), n), "page_table must be an int32"),
            (lambda: F.paged_attention(q, pool, pool, table, n.repeat(2)), "lengths must be an int32"),
            (lambda: F.paged_attention(q.repeat(2, 1, 1, 1), pool, pool, table.expand(2, 2), n.repeat(2)), "broadcast"),
            (lambda: F.cache_write(k.repeat(2, 1, 1, 1), k.repeat(2, 1, 1, 1), pool, pool, table.expand(2, 2), n.repeat(2)),
             "broadcast"),
            (lambda: F.paged_attention(q[:, :3], pool, pool, table, n), "multiple of the cache's heads"),
            (lambda: F.paged_attention(q.half(), pool, pool, table, n), "q must be a torch.float32"),
            (lambda: F.paged_attention(q, pool, pool[:4], table, n), "k_pages must be"),
            (lambda: F.PagedAttention(pool, pool, table, n, heads=4)(q), "q must be"),
            (lambda: F.cache_write(k, k, pool, pool, table, n, counts=n.cpu()), "counts must be on"),
            (lambda: F.cache_write(k[:, :1], k, pool, pool, table, n), "k must be"),
            (lambda: F.cache_write(k, k, pool[:1].expand(8, 2, 16, 64), pool, table, n), "broadcast"),
            (lambda: F.copy_pages([pool, pool[:4]], [0], [1]), "share shape"),
            (lambda: F.copy_pages([pool.transpose(1, 2)], [0], [1]), "contiguous"),
            (lambda: F.copy_pages([pool], [0, 1], [1]), "same length"),
            (lambda: F.copy_pages([pool], [1 << 40], [1]), "within the pool"),
            (lambda: F.copy_pages([pool], torch.tensor([0]).cuda(), [1]), "on the host")]:
        with pytest.raises(ValueError, match=text):
            call()
    for call, text in [(lambda: F.window_attention(q, k, k, sink_tokens=1), "sink_tokens need a window"),
                       (lambda: F.window_attention(q[..., :62], k[..., :62], k), "multiples of 4"),
                       (lambda: F.window_attention(q[..., 1:61], k[..., :60], k), "16-byte aligned"),
                       (lambda: F.paged_attention(q, pool[:, :, :8], pool[:, :, :8], table, n), "power of two"),
                       (lambda: F.paged_attention(q, pool, pool, table, n, softcap=-1.0), "softcap"),
                       (lambda: F.copy_pages([pool], [0, 1], [1, 2]), "both copied from and copied to")]:
        with pytest.raises(F.OfhError, match=text):
            call()


# --- together, as a program that serves sequences ---------------------------------

@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_serving_a_few_sequences(ofh, dt):
    """Prompts, decode steps, a fork that goes its own way, drafts of which some
    are dropped, an ended sequence and a compaction: every step's attention is the
    plain one over the tokens that the sequence then has."""
    import onednn_flash_cache as C
    F = ofh
    H, Hkv, D, layers, window, sinks = 4, 2, 64, 2, 40, 4
    options = dict(window=window, sink_tokens=sinks)
    cache = C.PagedCache(layers=layers, num_pages=40, page_size=16, kv_heads=Hkv, head_dim=D, dtype=TYPES[dt])
    texts = {}  # sequence -> per layer (k, v) [Hkv, n, D]
    seed = iter(range(10 ** 6))

    def ref(rows, q, seqs, layer, new):
        for b, s in enumerate(seqs):
            k, v = texts[s][layer]
            for h in range(H):
                for t in range(new):
                    n = k.shape[1]
                    rows[b, h, t] = attend_row(f64(q[b, h, t]), f64(k[h // 2]), f64(v[h // 2]), n - new + t, n,
                                               window=window, sinks=sinks, dtype=dt, out_dtype=dt)

    def step(seqs, new):
        batch = cache.extend(seqs, [new] * len(seqs))
        for layer in range(layers):
            q = randn(next(seed), (len(seqs), H, new, D), dt)
            k, v = (randn(next(seed), (len(seqs), Hkv, new, D), dt) for _ in range(2))
            for b, s in enumerate(seqs):
                old = texts[s][layer]
                texts[s][layer] = (torch.cat([old[0], k[b]], 1), torch.cat([old[1], v[b]], 1))
            batch.write(layer, k.cuda(), v.cuda())
            rows = {}
            ref(rows, q, seqs, layer, new)
            compare(batch.attend(layer, q.cuda(), **options), rows, dt, f"step of {new} layer {layer}")

    # a padded batch of prompts
    lengths = [70, 33, 5]
    seqs = [cache.add() for _ in lengths]
    batch = cache.extend(seqs, lengths)
    T = max(lengths)
    for s in seqs:
        texts[s] = [None] * layers
    for layer in range(layers):
        q = randn(next(seed), (3, H, T, D), dt)
        k, v = (randn(next(seed), (3, Hkv, T, D), dt) for _ in range(2))
        batch.write(layer, k.cuda(), v.cuda())
        out = F.window_attention(q.cuda(), k.cuda(), v.cuda(), lengths=batch.lengths, **options)
        rows = {}
        for b, n in enumerate(lengths):
            texts[seqs[b]][layer] = (k[b, :, :n], v[b, :, :n])
            for t in pick(n, 8, b):
                rows[b, 1, t] = attend_row(f64(q[b, 1, t]), f64(k[b, 0]), f64(v[b, 0]), t, n, window=window, sinks=sinks,
                                           dtype=dt, out_dtype=dt)
        compare(out, rows, dt, f"prompt layer {layer}")
    for _ in range(3):
        step(seqs, 1)
    child = cache.fork(seqs[0])
    texts[child] = list(texts[seqs[0]])
    step([child, seqs[0], seqs[2]], 1)
    step([child, seqs[1]], 4)          # drafts ...
    for s, keep in ((child, 2), (seqs[1], 1)):
        n = cache.pool.length(s) - 4 + keep
        cache.truncate(s, n)           # ... of which some stay
        texts[s] = [(k[:, :n], v[:, :n]) for k, v in texts[s]]
    cache.free(seqs[0])
    step([child, seqs[1], seqs[2]], 1)
    used = cache.pool.pages_in_use
    assert cache.compact() > 0
    rows, _ = cache.pool.table([child, seqs[1], seqs[2]], 40)
    assert max(max(r) for r in rows) < used
    for _ in range(2):
        step([seqs[2], child, seqs[1]], 1)
