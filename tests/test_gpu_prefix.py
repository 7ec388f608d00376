"""GPU parity of attention over shared prefixes against the plain 64-bit
implementation of serving_ref.py, within the bound that it derives."""

from __future__ import annotations

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


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def make(seed, dt, groups, lengths, Hkv, D, Dv, size, spare=2):
    """Pools and table of a batch in groups; pages in no order, the rest of a row -1."""
    per = [-(-n // size) for n in lengths]
    total = sum(tokens // size for _, tokens in groups) + sum(per) + spare
    order = np.random.default_rng(seed).permutation(total)
    table = np.full((len(lengths), max(max(per), max(t // size for _, t in groups), 1)), -1, np.int32)
    at = row = 0
    for count, tokens in groups:
        shared = order[at:at + tokens // size]
        at += shared.size
        for _ in range(count):
            table[row, :shared.size] = shared
            mine = max(0, per[row] - shared.size)
            table[row, shared.size:shared.size + mine] = order[at:at + mine]
            at += mine
            row += 1
    return (randn(seed + 1, (total, Hkv, size, D), dt), randn(seed + 2, (total, Hkv, size, Dv), dt), table)


def gather(pages, table, b, h):
    """Rows of sequence b (entries outside the pool: row 0, listed as hidden)."""
    ids = table[b]
    ok = (ids >= 0) & (ids < pages.shape[0])
    rows = pages[np.where(ok, ids, 0), h].reshape(-1, pages.shape[-1])
    return rows, np.flatnonzero(~np.repeat(ok, pages.shape[2]))


def check(F, dt, groups, lengths, H, Hkv, T, D, Dv=None, *, size=16, seed=0, slopes=False, out_f32=False, rows=48,
          pools=None, heads=5, **options):
    Dv = Dv or D
    k_pages, v_pages, table = make(seed, dt, groups, lengths, Hkv, D, Dv, size) if pools is None else pools
    B = len(lengths)
    q = randn(seed + 3, (B, H, T, D), dt)
    alibi = 2.0 ** -torch.arange(1.0, H + 1) if slopes else None
    out = F.shared_prefix_attention(
        q.cuda(), k_pages.cuda(), v_pages.cuda(), torch.from_numpy(table).cuda(), i32(lengths), groups=groups,
        alibi_slopes=None if alibi is None else alibi.cuda(), out_dtype=torch.float32 if out_f32 else None, **options)
    got, kp, vp, qn = f64(out), f64(k_pages), f64(v_pages), f64(q)
    rng = np.random.default_rng(seed)
    all_rows = [(b, h, t) for b in range(B) for h in range(H) for t in range(T)]
    some = [all_rows[i] for i in sorted({0, len(all_rows) - 1, *rng.integers(0, len(all_rows), rows)})]
    worst = 0.0
    label = f"prefix {dt} {groups} {lengths[:6]} H{H}/{Hkv} T{T} D{D}/{Dv} {options}"
    for b, h, t in some:
        k, hidden = gather(kp, table, b, h * Hkv // H)
        v, _ = gather(vp, table, b, h * Hkv // H)
        n = max(0, min(lengths[b], table.shape[1] * size))
        ref, bound = attend_row(qn[b, h, t], k, v, n - T + t, n, window=options.get("window", 0),
                                sinks=options.get("sink_tokens", 0), scale=options.get("scale"),
                                slope=float(alibi[h]) if slopes else 0.0, softcap=options.get("softcap", 0.0), dtype=dt,
                                out_dtype="f32" if out_f32 else dt, hidden=hidden)
        assert np.isfinite(got[b, h, t]).all(), f"{label}: row {b, h, t} is not finite"
        off = np.abs(got[b, h, t] - ref)
        worst = max(worst, float((off / (bound + 1e-300)).max()))
        assert (off <= bound).all(), f"{label}: row {b, h, t} off by {off.max():.3e}, bound {bound[off.argmax()]:.3e}"
    assert np.isfinite(got).all(), label
    print(f"{label}: at most {worst:.2f} of the bound", flush=True)
    return out


GROUPS = [[(1, 0)], [(3, 32)], [(1, 16)], [(2, 64), (1, 0), (3, 16)], [(1, 0), (4, 48), (1, 32)]]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("groups", GROUPS)
def test_prefix_groups(ofh, dt, groups):
    shared = [t for n, t in groups for _ in range(n)]
    for i, T in enumerate([1, 2, 5]):
        lengths = [s + T + 7 * b + i for b, s in enumerate(shared)]
        check(ofh, dt, groups, lengths, 8, 2, T, 64, seed=10 * i)
        check(ofh, dt, groups, lengths, 3, 3, T, 128, seed=10 * i + 1, out_f32=True)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D,Dv", [(8, 8), (32, 40), (64, 64), (80, 80), (96, 128), (128, 64), (136, 136), (192, 128), (256, 256)])
def test_prefix_head_dims(ofh, dt, D, Dv):
    check(ofh, dt, [(3, 48), (2, 96)], [50, 60, 49, 110, 97], 6, 2, 1, D, Dv, seed=D)
    check(ofh, dt, [(20, 160)], [161 + b for b in range(20)], 8, 1, 2, D, Dv, seed=D + 1, size=32)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lengths", [[0, 0, 0], [1, 40, 64], [64, 64, 64], [3, 63, 70], [65, 0, 200], [-4, 80, 1 << 30]])
def test_prefix_short_sequences(ofh, dt, lengths):
    """Sequences that end within what their group shares."""
    held = [max(0, min(n, 208)) for n in lengths]
    pools = make(5, dt, [(3, 64)], held, 2, 64, 64, 16)
    if lengths[2] == 1 << 30:  # taken as the table's tokens
        lengths = lengths[:2] + [pools[2].shape[1] * 16 + 5]
    for T in (1, 3):
        check(ofh, dt, [(3, 64)], lengths, 8, 2, T, 64, pools=pools, rows=72)
        check(ofh, dt, [(3, 64)], lengths, 8, 2, T, 64, pools=pools, rows=72, window=33, sink_tokens=5)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (20, 0), (20, 3), (100, 70), (100, 200), (4096, 4)])
def test_prefix_windows(ofh, dt, window, sinks):
    for T, D in ((1, 64), (4, 128)):
        check(ofh, dt, [(3, 128), (2, 64)], [129 + T, 150, 300, 70, 64 + T], 4, 2, T, D, window=window, sink_tokens=sinks,
              seed=window + T)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_prefix_scores(ofh, dt):
    for i, options in enumerate([dict(softcap=3.0), dict(slopes=True), dict(slopes=True, softcap=20.0), dict(scale=0.7),
                                 dict(scale=-0.2), dict(scale=0.0), dict(softcap=1000.0)]):
        check(ofh, dt, [(20, 96), (5, 32)], [97 + b for b in range(20)] + [33, 40, 50, 60, 70], 8, 2, 2, 64, seed=i, **options)
        check(ofh, dt, [(9, 96)], [97 + b for b in range(9)], 4, 4, 1, 128, seed=i + 50, **options)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("size", [16, 32, 64, 256])
def test_prefix_page_sizes(ofh, dt, D, size):
    """Pages within, of and past the keys of a step; pools with strides; a last step that
    is not full."""
    shared = max(size, 1200 // size * size)
    lengths = [shared + 1 + 11 * b for b in range(21)]
    k, v, table = make(D, dt, [(21, shared)], lengths, 4, D, D, size)
    wide = torch.zeros((k.shape[0], size, 4, D + 8), dtype=k.dtype)[..., :D].transpose(1, 2)  # token-major pages
    wide.copy_(k)
    check(ofh, dt, [(21, shared)], lengths, 16, 4, 1, D, pools=(wide, v, table), size=size, seed=size)
    check(ofh, dt, [(21, shared)], lengths, 16, 4, 1, D, pools=(k, v, table), size=size, seed=size, softcap=20.0, slopes=True)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefix_many_rows(ofh, dt, D):
    """Several tiles of rows, several parts of keys, tiles that end inside a sequence."""
    rng = np.random.default_rng(D)
    lengths = [1024 + int(x) for x in rng.integers(1, 90, 33)]
    check(ofh, dt, [(33, 1024)], lengths, 8, 2, 1, D, seed=D, rows=60)
    check(ofh, dt, [(20, 1024), (13, 512)], lengths, 12, 4, 3, D, seed=D + 1, rows=60, size=64)
    check(ofh, dt, [(33, 1024)], lengths, 40, 1, 1, D, seed=D + 2, rows=60, max_key_splits=1)
    check(ofh, dt, [(33, 1024)], lengths, 10, 2, 1, D, seed=D + 3, rows=60, max_key_splits=3, window=700, sink_tokens=40)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_prefix_many_groups(ofh, dt):
    """More groups than a wavefront has lanes, some of which share nothing."""
    groups = [(1 + i % 3, 16 * (i % 4)) for i in range(150)]
    shared = [t for n, t in groups for _ in range(n)]
    check(ofh, dt, groups, [s + 1 + b % 20 for b, s in enumerate(shared)], 4, 2, 1, 64, rows=200)
    check(ofh, dt, groups, [s + 2 + b % 40 for b, s in enumerate(shared)], 16, 1, 2, 128, rows=200, seed=1)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_prefix_beside_single_sequences(ofh, dt):
    """A large group and small ones among sequences that share nothing."""
    groups = [(1, 0)] * 20 + [(40, 512)] + [(1, 0)] * 9 + [(2, 1024)] + [(3, 0)]
    shared = [t for n, t in groups for _ in range(n)]
    check(ofh, dt, groups, [s + 1 + 5 * (b % 13) for b, s in enumerate(shared)], 8, 2, 1, 128, rows=150)
    check(ofh, dt, groups, [s + 2 + 5 * (b % 13) for b, s in enumerate(shared)], 4, 4, 2, 64, rows=150, seed=1)
    check(ofh, dt, [(1, 0)] * 70, [1 + 5 * b for b in range(70)], 4, 2, 1, 64, rows=100, seed=2)  # nothing is shared


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefix_parts(ofh, dt, D):
    """The shared keys in as many parts as the call's own tiles leave room for: none
    (own tiles for every place), few, and the most."""
    check(ofh, dt, [(72, 512)], [513 + 7 * i for i in range(72)], 8, 8, 1, D, rows=32, seed=D)
    check(ofh, dt, [(6, 512), (5, 256)], [600 + 3 * i for i in range(11)], 8, 4, 2, D, rows=32, seed=D + 1)
    check(ofh, dt, [(3, 4096)], [4097, 4300, 4096], 2, 1, 1, D, rows=6, seed=D + 2)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_prefix_widest_window(ofh, dt):
    """Positions before the sequence, and a window wider than any of them."""
    for n in (1, 5):
        check(ofh, dt, [(3 * n, 64)], [0, 2, 80] * n, 4, 2, 5, 64, window=(1 << 30) - 1, sink_tokens=1, rows=60, seed=n)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n", [3, 12, 40])
def test_prefix_workspace_contents(ofh, dt, n):
    """What the workspace held before does not matter: NaN in all of it."""
    F = ofh
    groups = [(n, 400), (2, 0)]
    lengths = [3 if b % 5 == 4 else 401 + 30 * b for b in range(n)] + [50, 0]
    k, v, table = make(4, dt, groups, [max(x, 401) for x in lengths], 2, 64, 64, 16)
    q = randn(5, (n + 2, 8, 1, 64), dt).cuda()
    for options in (dict(), dict(window=100, sink_tokens=20), dict(softcap=10.0)):
        a = F.SharedPrefixAttention(k.cuda(), v.cuda(), torch.from_numpy(table).cuda(), i32(lengths), groups=groups, heads=8,
                                    **options)
        outs = [a(q, workspace=torch.full((a.workspace_bytes,), x, dtype=torch.uint8, device="cuda")) for x in (0, 255, 127)]
        assert all(torch.equal(o, outs[0]) for o in outs) and torch.isfinite(outs[0]).all()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_prefix_pages_outside(ofh, dt):
    """Keys of entries outside the pool are not seen."""
    for n, T in ((3, 1), (40, 2)):
        lengths = [100 + b for b in range(n)]
        k, v, table = make(1, dt, [(n, 80)], lengths, 2, 64, 64, 16)
        table[:, 1], table[:, 3] = -1, k.shape[0]
        table[1, 5] = 1 << 30
        check(ofh, dt, [(n, 80)], lengths, 8, 2, T, 64, pools=(k, v, table), rows=100)
        table[:] = -7
        out = check(ofh, dt, [(n, 80)], lengths, 8, 2, T, 64, pools=(k, v, table))
        assert not out.any()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bad", [NAN, float("inf")])
def test_prefix_hidden_values(ofh, dt, D, bad):
    """What a row does not see does not reach it: shared keys past a short
    sequence's end or behind a window, rows of pages past a sequence's end."""
    n, T, H, Hkv = 18, 2, 8, 2
    lengths = [40 if b % 3 == 0 else 70 + b for b in range(n)]
    k, v, table = make(3, dt, [(n, 64)], lengths, Hkv, D, D, 16)
    q = randn(4, (n, H, T, D), dt).cuda()
    for options in (dict(), dict(window=30, sink_tokens=3)):
        run = lambda a, b: f64(ofh.shared_prefix_attention(q, a.cuda(), b.cuda(), torch.from_numpy(table).cuda(), i32(lengths),
                                                          groups=[(n, 64)], **options))
        clean = run(k, v)
        for pools in ("v", "kv"):
            k2, v2 = k.clone(), v.clone()
            v2[table[0, 3], :, 2, 1] = bad  # key 50
            if pools == "kv":
                k2[table[0, 3], :, 2, 1] = bad
            for b in range(n):  # past the end
                v2[table[b, (lengths[b] - 1) // 16], :, (lengths[b] - 1) % 16 + 1:] = bad if lengths[b] > 64 else 0
            out = run(k2, v2)
            worst = 0.0
            for b in range(n):
                for t in range(T):
                    p = lengths[b] - T + t
                    if p >= 50 and ("window" not in options or p - 50 < 30):
                        assert not np.isfinite(out[b, :, t, 1]).any()
                    elif lengths[b] > 64 or lengths[b] == 40:
                        worst = max(worst, np.abs(out[b, :, t] - clean[b, :, t]).max())
            # (other tiles may form their sums in another order)
            assert worst <= (1e-5 if dt == "f32" else 2.0 ** -6) * np.abs(clean).max()


def test_prefix_agrees_with_paged(ofh):
    """The same call without groups, over lengths that change between calls."""
    F = ofh
    k, v, table = make(9, "bf16", [(16, 512)], [700] * 16, 4, 128, 128, 16)
    k, v, table = k.cuda(), v.cuda(), torch.from_numpy(table).cuda()
    lengths = torch.full((16,), 513, dtype=torch.int32).cuda()
    shared = F.SharedPrefixAttention(k, v, table, lengths, groups=[(16, 512)], heads=16, query_tokens=2)
    plain = F.PagedAttention(k, v, table, lengths, heads=16, query_tokens=2)
    for n in (514, 600, 3, 700):
        lengths.fill_(n)
        q = randn(n, (16, 16, 2, 128), "bf16").cuda()
        a, b = shared(q), plain(q)
        # each is within a few 2^-8 of the exact row
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -5 * b.float().abs().max()
        ws = torch.empty(shared.workspace_bytes, dtype=torch.uint8, device="cuda")
        assert torch.equal(shared(q, workspace=ws), a)
        with pytest.raises(F.OfhError) as e:
            shared(q, workspace=ws[:-256])
        assert e.value.code == F.OFH_ERROR_WORKSPACE_TOO_SMALL
        out = torch.full((16, 2, 16, 130), 7.0, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
        with pytest.raises(F.OfhError):  # rows that are not 16-byte aligned
            shared(q, out=out[..., 1:129])
        tokens = q.transpose(1, 2).contiguous().transpose(1, 2)
        assert torch.equal(shared(tokens, out=torch.empty_like(tokens)), a)


def test_prefix_refusals(ofh):
    F = ofh
    k = torch.zeros((9, 2, 16, 64), dtype=torch.bfloat16, device="cuda")
    table, lengths = torch.zeros((3, 4), dtype=torch.int32).cuda(), torch.zeros(3, dtype=torch.int32).cuda()
    for groups in ([(2, 16)], [(4, 16)], [(3, 15)], [(3, 80)], [], [(3,)], [(0, 16), (3, 16)], [(3, -16)], [(3, 16.0)],
                   [(True, 16), (2, 16)]):
        with pytest.raises(ValueError):
            F.SharedPrefixAttention(k, k, table, lengths, groups=groups, heads=4)
    with pytest.raises(ValueError, match="whole pages"):
        F.PrefixGroups([(3, 24)], page_size=16)
    with pytest.raises(ValueError, match="whole pages"):  # made for pages of another size
        F.SharedPrefixAttention(torch.zeros((9, 2, 64, 64), device="cuda"), torch.zeros((9, 2, 64, 64), device="cuda"), table,
                                lengths, groups=F.PrefixGroups([(3, 16)], page_size=16), heads=4)
    with pytest.raises(ValueError, match="on cuda"):
        F.SharedPrefixAttention(k, k, table, lengths, groups=F.PrefixGroups([(3, 16)], page_size=16, device="cpu"), heads=4)


def test_prefix_graphs_and_streams(ofh):
    """Captured calls replayed with other inputs; two graphs; a side stream; two threads."""
    F = ofh
    k, v, table = make(2, "f16", [(12, 256), (4, 64)], [400] * 12 + [200] * 4, 2, 64, 64, 16)
    k, v, table = k.cuda(), v.cuda(), torch.from_numpy(table).cuda()
    lengths = i32([300] * 12 + [100] * 4)
    attend = F.SharedPrefixAttention(k, v, table, lengths, groups=[(12, 256), (4, 64)], heads=8)
    qs = [randn(i, (16, 8, 1, 64), "f16").cuda() for i in range(2)]
    for q in qs:
        attend(q)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(attend(q))
        graphs.append(graph)
    for step in range(4):
        lengths += 5
        for i, q in enumerate(qs):
            q.copy_(randn(10 * step + i, q.shape, "f16"))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for q, out in zip(qs, outs):
            assert torch.equal(out, attend(q))
    side = torch.cuda.Stream()
    want = attend(qs[0])
    side.wait_stream(torch.cuda.current_stream())
    got = [attend(qs[0], stream=s) for s in (side, side.cuda_stream)]
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)
    results = [None, None]

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                results[i] = attend(qs[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for q, r in zip(qs, results):
        assert torch.equal(r, attend(q))


def test_cache_batch_attend_shared(ofh):
    """Forks of a cache's sequences find their groups by themselves."""
    from onednn_flash_cache import PagedCache
    F = ofh
    cache = PagedCache(layers=1, num_pages=200, page_size=16, kv_heads=2, head_dim=64)
    rotary = F.Rotary(64)

    def step(seqs, counts, seed, attend):
        T = max(counts)
        batch = cache.extend(seqs, counts)
        k, v, q = (randn(seed + i, (len(seqs), h, T, 64), "bf16").cuda() for i, h in enumerate((2, 2, 8)))
        q = batch.append(0, k, v, rotary, q)
        if attend:
            return batch, batch.attend_shared(0, q), batch.attend(0, q)
        return batch, None, None

    roots = [cache.add(), cache.add()]
    step(roots, [100, 41], 0, False)
    seqs = [roots[0]] + [cache.fork(roots[0]) for _ in range(4)] + [roots[1]] + [cache.fork(roots[1]) for _ in range(2)]
    seqs.append(cache.add())
    for i in range(3):
        batch, a, b = step(seqs, [1 + i] * len(seqs), 10 * i, True)
        assert batch.groups.groups == [(5, 96), (3, 32), (1, 0)]
        assert (a.float() - b.float()).abs().max() <= 2.0 ** -5 * b.float().abs().max()
    with pytest.raises(ValueError, match="new ones"):
        batch.attend_shared(0, torch.zeros((9, 8, 9, 64), dtype=torch.bfloat16, device="cuda"))
