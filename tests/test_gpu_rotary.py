"""GPU parity of rotary positions and of appending to a paged cache against the
plain 64-bit implementation of rotary_ref.py, within the bound that it derives
from the arithmetic."""

from __future__ import annotations

import threading

import numpy as np
import pytest

import rotary_ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def randn(seed, shape, dt):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=gen).to(TYPES[dt])


def f64(t):
    return t.detach().cpu().double().numpy()


def within(got, ref, bound, label):
    assert np.isfinite(got).all(), f"{label}: not finite"
    off = np.abs(got - ref)
    worst = float((off / (bound + 1e-300)).max()) if (bound > 0).any() else 0.0
    assert (off <= bound).all(), f"{label}: off by {off.max():.3e}, {worst:.2f} of the bound"
    return worst


def check(F, x, rotary, position, label, *, dt, got, transpose=False):
    """position: broadcast to [B, 1, T]."""
    ref, bound = rotary_ref.rotate(f64(x), position, rotary.frequencies.cpu().numpy(), interleaved=rotary.interleaved,
                                   magnitude=float(np.float32(rotary.magnitude)), transpose=transpose, dtype=dt)
    worst = within(f64(got), ref, bound, label)
    part = rotary.rotary_dim
    assert torch.equal(got[..., part:].cpu(), x[..., part:].cpu()), f"{label}: columns past rotary_dim"
    print(f"{label}: at most {worst:.2f} of the bound", flush=True)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,part", [(64, 64), (128, 128), (96, 64), (80, 20), (64, 2), (50, 34), (2, 2), (10, 6), (256, 256),
                                    (1024, 1024), (1023, 512)])
def test_rotary_rows(ofh, dt, interleaved, D, part):
    rotary = ofh.Rotary(D, rotary_dim=part, interleaved=interleaved)
    for i, (B, H, T) in enumerate([(1, 1, 1), (2, 3, 17), (3, 5, 64)]):
        x = randn(D + i, (B, H, T, D), dt).cuda()
        check(ofh, x, rotary, np.arange(T)[None, None] + 11, f"rotary {dt} {interleaved} {D}/{part} {B, H, T}", dt=dt,
              got=rotary(x, offset=11))
        check(ofh, x, rotary, np.arange(T)[None, None], f"rotary back {dt} {interleaved} {D}/{part} {B, H, T}", dt=dt,
              got=rotary(x, transpose=True), transpose=True)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_many_tokens(ofh, dt, interleaved):
    """Four tokens per workgroup, the last with fewer; more items than a pass of them."""
    for D, part, H, T in ((64, 32, 3, 1366), (128, 128, 40, 1367), (62, 30, 2, 1365)):
        rotary = ofh.Rotary(D, rotary_dim=part, interleaved=interleaved, magnitude=1.2)
        x = randn(D, (3, H, T, D), dt).cuda()
        check(ofh, x, rotary, np.arange(T)[None, None], f"rotary {dt} {interleaved} T{T}", dt=dt, got=rotary(x))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_positions(ofh, dt, interleaved):
    rotary = ofh.Rotary(64, interleaved=interleaved, scaling={"type": "parts", "factor": 8, "original_tokens": 4096},
                        magnitude=1.3)
    x = randn(1, (3, 2, 9, 64), dt).cuda()
    t = np.arange(9)
    for offset in (0, -5, 1 << 20, (1 << 31) - 1, -(1 << 31)):
        check(ofh, x, rotary, t[None, None] + offset, f"offset {offset}", dt=dt, got=rotary(x, offset=offset))
    rng = np.random.default_rng(0)
    pos = rng.integers(-100, 1 << 21, (3, 9)).astype(np.int32)
    pos[0, 0], pos[1, 3], pos[2, 8] = (1 << 31) - 1, -(1 << 31), 0
    p = torch.from_numpy(pos).cuda()
    check(ofh, x, rotary, pos[:, None], "positions", dt=dt, got=rotary(x, positions=p))
    check(ofh, x, rotary, pos[:1, None], "positions [T]", dt=dt, got=rotary(x, positions=p[0]))
    check(ofh, x, rotary, pos[:1, None], "positions expanded", dt=dt, got=rotary(x, positions=p[:1].expand(3, 9)))
    wide = torch.zeros((3, 20), dtype=torch.int32).cuda()
    wide[:, 4:13] = p
    check(ofh, x, rotary, pos[:, None], "positions strided", dt=dt, got=rotary(x, positions=wide[:, 4:13]))
    lengths = [9, 700, 3]  # (the last has fewer tokens than rows: positions from -6)
    at = np.array(lengths)[:, None] - 9 + t
    check(ofh, x, rotary, at[:, None], "lengths", dt=dt,
          got=rotary(x, lengths=torch.tensor(lengths, dtype=torch.int32).cuda()))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_layouts(ofh, dt, interleaved):
    D = 64
    rotary = ofh.Rotary(D, rotary_dim=48, interleaved=interleaved)
    at = np.arange(21)[None, None]
    base = randn(3, (2, 21, 5, D), dt).cuda()
    token_major = base.transpose(1, 2)
    check(ofh, token_major, rotary, at, "token major", dt=dt, got=rotary(token_major))
    wide = randn(4, (2, 5, 21, D + 9), dt).cuda()
    odd = wide[..., 3:3 + D]  # rows at odd addresses
    check(ofh, odd, rotary, at, "odd rows", dt=dt, got=rotary(odd))
    out = torch.full((2, 5, 21, D + 9), 7.0, dtype=TYPES[dt]).cuda()
    got = rotary(token_major, out=out[..., 1:1 + D])
    check(ofh, token_major, rotary, at, "odd out", dt=dt, got=got)
    assert (out[..., :1] == 7).all() and (out[..., 1 + D:] == 7).all()
    every = base[:, :, :1].transpose(1, 2).expand(2, 5, 21, D)  # one head for all
    check(ofh, every, rotary, at, "broadcast", dt=dt, got=rotary(every))
    for x in (token_major.clone(memory_format=torch.preserve_format), odd):
        want = rotary(x.clone())
        got = rotary(x, out=x)
        assert got is x and torch.equal(got, want)
    one = randn(5, (1, 1, 1, D), dt).cuda()
    assert torch.equal(rotary(one, out=one, offset=5), rotary(randn(5, (1, 1, 1, D), dt).cuda(), offset=5))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(ofh, interleaved):
    """The transposed form is the gradient: <turn(x + d) - turn(x - d), y> / 2 = <d,
    back(y)>, the turn being linear, so that differences of any width are exact."""
    rotary = ofh.Rotary(80, rotary_dim=64, interleaved=interleaved, magnitude=1.1)
    x, d, y = (randn(i, (2, 3, 33, 80), "f32").cuda() for i in range(3))
    turn = lambda t: f64(rotary(t, offset=1000))
    left = ((turn(x + d) - turn(x - d)) / 2 * f64(y)).sum()
    back = f64(rotary(y, offset=1000, transpose=True))
    # each turned element is off by less than 8 u (|x| + |y|) m, x + d and x - d by u
    size = (np.abs(f64(x)).mean() + np.abs(f64(d)).mean()) * 2 * 1.1
    bound = 12 * 2.0 ** -24 * 2 * size * np.abs(f64(y)).sum()
    assert abs(left - (back * f64(d)).sum()) <= bound
    # and turning there and back scales by the magnitude's square
    both = f64(rotary(rotary(x, offset=7), offset=7, transpose=True))
    want = f64(x).copy()
    want[..., :64] *= float(np.float32(1.1)) ** 2
    assert np.abs(both - want).max() <= 2 * 1.21 * 16 * 2.0 ** -24 * 2 * np.abs(f64(x)).max()


def test_rotary_hidden_values(ofh):
    """A NaN or an infinity stays in its pair."""
    rotary = ofh.Rotary(16)
    x = randn(0, (1, 1, 3, 16), "f32").cuda()
    clean = rotary(x, offset=3)
    x[0, 0, 1, 2] = float("nan")
    x[0, 0, 1, 5] = float("inf")
    got = rotary(x, offset=3)
    bad = torch.zeros(16, dtype=torch.bool).cuda()
    bad[[2, 10, 5, 13]] = True
    assert not torch.isfinite(got[0, 0, 1, bad]).any()
    assert torch.equal(got[0, 0, 1, ~bad], clean[0, 0, 1, ~bad]) and torch.equal(got[0, 0, [0, 2]], clean[0, 0, [0, 2]])


def test_rotary_offsets_past_32_bits(ofh):
    """More than 2^32 bytes in a tensor, positions in the millions."""
    T, D = 9_000_001, 128
    rotary = ofh.Rotary(D)
    x = torch.empty((1, 2, T, D), dtype=torch.bfloat16, device="cuda")
    rows = [0, 1, T // 2, T - 2, T - 1]
    x[:, :, rows] = randn(1, (1, 2, len(rows), D), "bf16").cuda()
    got = rotary(x)
    check(ofh, x[:, :, rows], rotary, np.array(rows)[None, None], "far rows", dt="bf16", got=got[:, :, rows])


def test_rotary_refusals(ofh):
    rotary = ofh.Rotary(64)
    x = torch.zeros((2, 3, 4, 64), device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    for bad in (x.cpu(), x[0], x.double(), x[..., :62], x.transpose(2, 3), torch.zeros((2, 3, 0, 64), device="cuda")):
        with pytest.raises(ValueError):
            rotary(bad)
    for options in (dict(offset=1.0), dict(offset=1 << 31), dict(positions=torch.zeros((2, 5), **i32)),
                    dict(positions=torch.zeros((4,), dtype=torch.int64, device="cuda")),
                    dict(positions=torch.zeros((4,), dtype=torch.int32)), dict(positions=[0, 1, 2, 3]),
                    dict(lengths=torch.zeros((3,), **i32)), dict(lengths=torch.zeros((2,), **i32), offset=1),
                    dict(lengths=torch.zeros((2,), **i32), positions=torch.zeros((4,), **i32)),
                    dict(out=x[..., :62]), dict(out=x.half()), dict(out=x.cpu()),
                    dict(out=torch.zeros((2, 1, 4, 64), device="cuda").expand(2, 3, 4, 64))):
        with pytest.raises(ValueError):
            rotary(x, **options)
    y = torch.zeros((2, 4, 3, 64), device="cuda").transpose(1, 2)
    with pytest.raises(ValueError, match="in place"):  # same memory in another order
        rotary(y, out=y.as_strided((2, 3, 4, 64), (768, 256, 64, 1)))


# --- appending to a cache ----------------------------------------------------

def place_of(table, position, size):
    page, row = divmod(position, size)
    return None if position < 0 or page >= table.shape[1] else (page, row)


def check_append(F, dt, B, Hkv, H, T, D, Dv, size, lengths, counts=None, *, part=None, interleaved=False, seed=0,
                 pages=None, table=None, odd=False, in_place=False, token_major=True):
    part = D if part is None else part
    rotary = F.Rotary(D, rotary_dim=part, interleaved=interleaved, magnitude=1.25)
    per = max(1, -(-max(max(lengths), 1) // size))
    pages = B * per + 3 if pages is None else pages
    if table is None:
        order = np.random.default_rng(seed).permutation(pages)[:B * per].astype(np.int32).reshape(B, per)
        table = order
    pad = 3 if odd else 0
    new = lambda i, heads, dim: (randn(seed + i, (B, T, heads, dim + pad), dt).cuda()[..., pad:].transpose(1, 2) if token_major
                                 else randn(seed + i, (B, heads, T, dim + pad), dt).cuda()[..., pad:])
    k, v = new(1, Hkv, D), new(2, Hkv, Dv)
    q = new(3, H, D) if H else None
    k_pages = randn(seed + 4, (pages, Hkv, size, D), dt).cuda()
    v_pages = randn(seed + 5, (pages, Hkv, size, Dv), dt).cuda()
    want_k, want_v = k_pages.clone(), v_pages.clone()
    n = [T] * B if counts is None else [max(0, min(c, T)) for c in counts]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    label = f"append {dt} B{B} H{H}/{Hkv} T{T} D{D}/{Dv} part {part} {interleaved} page {size} {lengths} {counts}"
    # the rotation by itself is bit for bit the same; 64 bits below
    at = np.array([[lengths[b] - n[b] + t for t in range(T)] for b in range(B)], np.int32)
    turned = rotary(k, positions=torch.from_numpy(at).cuda())
    check(F, k, rotary, at[:, None], label, dt=dt, got=turned)
    for b in range(B):
        for t in range(n[b]):
            to = place_of(table, int(at[b, t]), size)
            if to is None or not 0 <= table[b, to[0]] < pages:
                continue
            want_k[table[b, to[0]], :, to[1]] = turned[b, :, t]
            want_v[table[b, to[0]], :, to[1]] = v[b, :, t]
    want_q = None
    if H:
        want_q = rotary(q, positions=torch.from_numpy(at).cuda())
        for b in range(B):
            want_q[b, :, n[b]:] = 0
    q_out = F.cache_append(k, v, k_pages, v_pages, torch.from_numpy(np.ascontiguousarray(table)).cuda(), i32(lengths),
                           rotary, q=q, q_out=q if in_place else None, counts=None if counts is None else i32(counts))
    assert torch.equal(k_pages, want_k) and torch.equal(v_pages, want_v), label
    assert (q_out is None) == (H == 0) and (H == 0 or torch.equal(q_out, want_q)), label


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_sizes(ofh, dt, interleaved):
    for i, (B, Hkv, H, T, D, Dv, part, size) in enumerate([
            (1, 1, 1, 1, 64, 64, 64, 16), (3, 2, 8, 1, 128, 128, 128, 16), (2, 8, 32, 1, 128, 64, 64, 32),
            (2, 2, 0, 5, 80, 80, 80, 16), (2, 1, 3, 40, 64, 40, 32, 64), (2, 3, 5, 7, 50, 34, 34, 16),
            (1, 1, 2, 3, 2, 1, 2, 16), (2, 2, 4, 33, 256, 256, 256, 128), (1, 1, 1, 2, 1024, 8, 1024, 16)]):
        check_append(ofh, dt, B, Hkv, H, T, D, Dv, size, [T + 9 * b + 4 for b in range(B)], part=part,
                     interleaved=interleaved, seed=10 * i)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_append_ragged(ofh, dt):
    lengths, counts = [40, 7, 100, 0, 3], [20, 7, 1, 0, 0]
    check_append(ofh, dt, 5, 2, 4, 20, 64, 64, 16, lengths, counts)
    check_append(ofh, dt, 5, 2, 4, 20, 64, 64, 16, lengths, [25, -3, 20, 0, 9], in_place=True)  # taken between 0 and T
    check_append(ofh, dt, 5, 2, 4, 20, 62, 64, 16, lengths, counts, odd=True, in_place=True)
    check_append(ofh, dt, 5, 2, 4, 20, 64, 64, 16, lengths, counts, token_major=False)
    check_append(ofh, dt, 3, 2, 4, 6, 64, 64, 16, [4, 6, 8])  # the first sequence's first tokens have no position


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_append_places(ofh, dt):
    """Entries outside the pool, and positions past the table, are not written."""
    table = np.array([[3, -1, 5], [0, 9, 1 << 30], [-5, 4, 2]], np.int32)
    for lengths in ([48, 48, 48], [30, 60, 33], [16, 17, 1000]):
        check_append(ofh, dt, 3, 2, 4, 30, 64, 64, 16, lengths, pages=9, table=table)


def test_append_many_tokens(ofh):
    """Four tokens per workgroup."""
    check_append(ofh, "bf16", 3, 2, 5, 1500, 64, 64, 32, [1500, 1800, 2000], [1500, 700, 1399])
    check_append(ofh, "f16", 3, 8, 16, 1399, 128, 128, 16, [1399, 1800, 2000], part=64, interleaved=True)


def test_append_pools_with_strides(ofh):
    """Layers in one tensor, pages of token-major rows."""
    F = ofh
    pools = torch.zeros((2, 7, 16, 3, 2, 64), dtype=torch.bfloat16, device="cuda")  # layer, page, row, head, k and v, D
    k_pages, v_pages = (pools[1, :, :, :, i].transpose(1, 2) for i in range(2))
    k, v = (randn(i, (2, 3, 4, 64), "bf16").cuda() for i in range(2))
    table = torch.tensor([[5, 1], [2, 0]], dtype=torch.int32).cuda()
    lengths = torch.tensor([20, 6], dtype=torch.int32).cuda()
    rotary = F.Rotary(64)
    assert F.cache_append(k, v, k_pages, v_pages, table, lengths, rotary) is None
    turned = rotary(k, lengths=lengths)
    assert torch.equal(k_pages[1, :, 0:4], turned[0]) and torch.equal(k_pages[2, :, 2:6], turned[1])
    assert torch.equal(v_pages[1, :, 0:4], v[0]) and torch.equal(v_pages[2, :, 2:6], v[1])
    assert int((pools != 0).any(-1).sum()) == 2 * 3 * 4 * 2


def test_append_refusals(ofh):
    F = ofh
    k = torch.zeros((2, 3, 4, 64), dtype=torch.bfloat16, device="cuda")
    pages = torch.zeros((5, 3, 16, 64), dtype=torch.bfloat16, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    table, lengths = torch.zeros((2, 2), **i32), torch.full((2,), 4, **i32)
    rotary = F.Rotary(64)
    for r in (None, F.Rotary(32), rotary.frequencies):
        with pytest.raises(ValueError, match="rotary"):
            F.CacheAppender(pages, pages.clone(), table, lengths, r)
    append = F.CacheAppender(pages, pages.clone(), table, lengths, rotary)
    q = torch.zeros((2, 6, 4, 64), dtype=torch.bfloat16, device="cuda")
    for args, options in (((k, k[:, :, :2]), {}), ((k.half(), k), {}), ((k, k, q[:, :, :3]), {}), ((k, k, q.float()), {}),
                          ((k, k, q[..., :32]), {}), ((k, k, q.cpu()), {}), ((k, k), dict(q_out=q)),
                          ((k, k, q), dict(q_out=q[:, :3])), ((k, k, q), dict(q_out=q.float())),
                          ((k, k, q), dict(q_out=q[:, :1].expand(2, 6, 4, 64)))):
        with pytest.raises(ValueError):
            append(*args, **options)
    assert not pages.any()


def test_append_streams_and_graphs(ofh):
    """A captured step replayed with new inputs, eager calls in between, another
    stream, and two threads at once."""
    F = ofh
    B, Hkv, H, D, size = 4, 2, 8, 64, 16
    rotary = F.Rotary(D)
    table = torch.arange(B * 4, dtype=torch.int32).reshape(B, 4).cuda()
    lengths = torch.tensor([1, 5, 16, 17], dtype=torch.int32).cuda()
    pools = [torch.zeros((B * 4, Hkv, size, D), dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    append = F.CacheAppender(pools[0], pools[1], table, lengths, rotary)
    eager = F.CacheAppender(pools[2], pools[3], table, lengths, rotary)
    k, v, q = (randn(i, (B, h, 1, D), "bf16").cuda() for i, h in enumerate((Hkv, Hkv, H)))
    append(k, v, q)
    eager(k, v, q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = append(k, v, q)
    for i in range(5):
        lengths += 3
        for j, t in enumerate((k, v, q)):
            t.copy_(randn(100 * i + j, t.shape, "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager(k, v, q))
        assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = eager(k, v, q)
    got = append(k, v, q, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    results = {}

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            x = randn(i, (2, 3, 50, D), "bf16").cuda()
            for _ in range(20):
                results[i] = (x, rotary(x, offset=i))
            s.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert torch.equal(results[i][1], rotary(results[i][0], offset=i))


def test_cache_batch_append(ofh):
    """A layer's step through the cache's own calls is rotary, write and attend."""
    from onednn_flash_cache import PagedCache
    F = ofh
    cache = PagedCache(layers=2, num_pages=20, page_size=16, kv_heads=2, head_dim=64)
    other = PagedCache(layers=2, num_pages=20, page_size=16, kv_heads=2, head_dim=64)
    rotary = F.Rotary(64)
    for c in (cache, other):
        c.seqs = [c.add() for _ in range(3)]
    for step, counts in enumerate(([7, 30, 16], [1, 1, 1], [2, 2, 2])):
        T = max(counts)
        k, v, q = (randn(step * 3 + i, (3, h, T, 64), "bf16").cuda() for i, h in enumerate((2, 2, 4)))
        a, b = cache.extend(cache.seqs, counts), other.extend(other.seqs, counts)
        got = a.append(1, k, v, rotary, q)
        at = (b.lengths - b.counts)[:, None] + torch.arange(T, dtype=torch.int32, device="cuda")
        b.write(1, rotary(k, positions=at), v)
        want = rotary(q, positions=at)
        for i, n in enumerate(counts):
            assert torch.equal(got[i, :, :n], want[i, :, :n]) and not got[i, :, n:].any()
        assert torch.equal(cache.k_pages, other.k_pages) and torch.equal(cache.v_pages, other.v_pages)
        if min(counts) == T:
            assert torch.equal(a.attend(1, got), b.attend(1, want))
    assert a.append(0, k, v, rotary) is None
    with pytest.raises(ValueError, match="new ones"):
        a.append(0, k[:, :, :1], v[:, :, :1], rotary)
