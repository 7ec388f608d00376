"""GPU parity of page bounds, of the selection of pages, and of attention over
selected pages, against plain implementations in 64 bits (serving_ref.py has the
attention's error bound)."""

from __future__ import annotations

import numpy as np
import pytest

from serving_ref import attend_row

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NAN, INF = float("nan"), float("inf")


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
    return torch.tensor(np.asarray(x), dtype=torch.int32).cuda()


def make_table(seed, lengths, size, width=None, spare=3):
    per = [-(-max(n, 0) // size) for n in lengths]
    total = sum(per) + spare
    order = np.random.default_rng(seed).permutation(total)
    table = np.full((len(lengths), width or max(max(per), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


# --- bounds -----------------------------------------------------------------

def bounds_ref(k, bounds, table, lengths, counts, size):
    """k [P,Hkv,S,D], bounds [P,Hkv,2,D] (numpy, of any type): renewed in place."""
    for b, n in enumerate(lengths):
        count = counts[b]
        if count <= 0:
            continue
        for place in range(max(0, n - count) // size, min(table.shape[1], -(-n // size))):
            page = table[b, place]
            if not 0 <= page < k.shape[0]:
                continue
            rows = k[page, :, :min(size, n - place * size)]
            bounds[page, :, 0], bounds[page, :, 1] = rows.min(1), rows.max(1)  # (a NaN stays)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [8, 24, 64, 80, 128, 136, 256])
@pytest.mark.parametrize("size", [16, 64, 128])
def test_bounds(ofh, dt, D, size):
    lengths = [1, size, size + 1, 5 * size - 3, 0, 3, 2 * size + 7]
    table, pages = make_table(D, lengths, size)
    k = randn(D, (pages, 3, size, D), dt)
    for i, (tokens, counts) in enumerate([(1, None), (size, None), (3 * size + 1, None), (7 * size, None),
                                          (2 * size, [1, 0, -1, 2 * size, 5, 3, 99 * size])]):
        bounds = randn(i, (pages, 3, 2, D), dt)
        want = f64(bounds)
        n = [tokens] * 7 if counts is None else [max(0, min(c, tokens)) for c in counts]
        bounds_ref(f64(k), want, table, lengths, n, size)
        got = bounds.cuda()
        ofh.page_bounds(k.cuda(), got, i32(table), i32(lengths), tokens=tokens, counts=None if counts is None else i32(counts))
        np.testing.assert_array_equal(f64(got), want)


def test_bounds_values_and_places(ofh):
    """NaN and infinities, pages outside the pool, sequences longer than the table, pools with strides."""
    lengths = [40, 100, -5, 33]
    table = np.array([[2, -1, 4], [0, 9, 1], [3, 5, 6], [8, 7, 1 << 30]], np.int32)
    k = randn(0, (9, 2, 16, 64), "bf16")
    k[2, 0, 5, 7], k[0, 1, 2, 3], k[0, 1, 4, 3], k[4, 0, 8, 1] = NAN, INF, -INF, NAN  # (row 8 of page 4 is past the end)
    bounds = torch.full((9, 2, 2, 64), 5.0, dtype=torch.bfloat16)
    want = f64(bounds)
    bounds_ref(f64(k), want, table, lengths, [1000] * 4, 16)
    assert np.isnan(want).sum() == 2
    wide = torch.full((3, 9, 2, 2, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    ofh.page_bounds(k.cuda(), wide[1], i32(table), i32(lengths))
    np.testing.assert_array_equal(f64(wide[1]), want)
    assert (wide[0] == 5).all() and (wide[2] == 5).all()
    rows = torch.zeros((9, 16, 2, 64), dtype=torch.bfloat16, device="cuda")  # token-major pages
    rows.copy_(k.transpose(1, 2))
    again = torch.full_like(wide[1], 5.0)
    ofh.page_bounds(rows.transpose(1, 2), again, i32(table), i32(lengths), tokens=1000)
    np.testing.assert_array_equal(f64(again), want)


def test_bounds_refusals(ofh):
    F = ofh
    k = torch.zeros((9, 2, 16, 64), dtype=torch.bfloat16, device="cuda")
    table, lengths = i32(np.zeros((3, 4))), i32([1, 2, 3])
    good = torch.zeros((9, 2, 2, 64), dtype=torch.bfloat16, device="cuda")
    for bounds in (good[:8], good.float(), good[..., :32], good[:, :, :1], good.cpu(), good[:, :1].expand(9, 2, 2, 64)):
        with pytest.raises(ValueError):
            F.PageBounds(k, bounds, table, lengths, tokens=1)
    for options in (dict(tokens=0), dict(tokens=1.0), dict(tokens=1, counts=i32([1, 2])), dict(tokens=1, counts=[1, 2, 3])):
        with pytest.raises(ValueError):
            F.PageBounds(k, good, table, lengths, **options)


# --- selection --------------------------------------------------------------

def rank(x):
    """Numbers in the order of scores: NaN above all, -0 as 0."""
    return np.where(np.isnan(x), np.inf, x), np.isnan(x)


def select_ref(q, bounds, table, lengths, T, pages, first, recent, size, negative=False):
    B, H = q.shape[:2]
    Hkv = bounds.shape[1]
    out = np.full((B, Hkv, T, pages), -1, np.int32)
    if negative:
        q = -q
    for b in range(B):
        for h in range(Hkv):
            for t in range(T):
                n = max(0, min(lengths[b], table.shape[1] * size))
                have = -(-max(0, n - T + t + 1) // size)
                if have <= pages:
                    out[b, h, t, :have] = np.arange(have)
                    continue
                ids = table[b, first:have - recent]
                ok = (ids >= 0) & (ids < bounds.shape[0])
                bd = bounds[np.where(ok, ids, 0), h]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = np.stack([(r * np.where(r > 0, bd[:, 1], bd[:, 0])).sum(-1).astype(np.float32)
                                  for r in q[b, h * H // Hkv:(h + 1) * H // Hkv, t]])
                    nan = np.isnan(s).any(0)
                    s = np.where(np.isnan(s), -np.inf, s).max(0)
                order = sorted(range(len(ids)), key=lambda i: (not ok[i], not nan[i], -s[i], i))
                mid = sorted(order[:pages - first - recent])
                out[b, h, t] = [*range(first), *(first + i for i in mid), *range(have - recent, have)]
    return out


def check_select(F, dt, lengths, H, Hkv, T, D, size, pages, first=1, recent=2, *, seed=0, k=None, q=None, table=None,
                 width=None, attend=True, bounds=None, **options):
    B = len(lengths)
    if table is None:
        table, total = make_table(seed, lengths, size, width)
    else:
        total = k.shape[0]
    k = randn(seed + 1, (total, Hkv, size, D), dt) if k is None else k
    v = randn(seed + 2, (total, Hkv, size, D), dt)
    q = randn(seed + 3, (B, H, T, D), dt) if q is None else q
    if bounds is None:
        bounds = torch.zeros((total, Hkv, 2, D), dtype=TYPES[dt], device="cuda")
        F.page_bounds(k.cuda(), bounds, i32(table), i32(lengths))
    a = F.SelectedAttention(k.cuda(), v.cuda(), bounds, i32(table), i32(lengths), heads=H, pages=pages, first_pages=first,
                            recent_pages=recent, query_tokens=T, **options)
    got = a.select(q.cuda())
    want = select_ref(f64(q), f64(bounds), table, lengths, T, pages, first, recent, size, options.get("scale", 1.0) < 0)
    label = f"select {dt} {lengths[:6]} H{H}/{Hkv} T{T} D{D} page {size} {first}+{pages}+{recent} {options}"
    np.testing.assert_array_equal(got.cpu().numpy(), want, err_msg=label)
    if attend:
        out = a(q.cuda())
        assert torch.equal(out, a(q.cuda(), selected=got)), label
        check_rows(label, out, q, k, v, table, lengths, want, size, dt, **options)
    return got, a


def check_rows(label, out, q, k, v, table, lengths, selected, size, dt, rows=40, **options):
    B, H, T, _ = q.shape
    Hkv = k.shape[1]
    got, qn, kn, vn = f64(out), f64(q), f64(k), f64(v)
    every = [(b, h, t) for b in range(B) for h in range(H) for t in range(T)]
    rng = np.random.default_rng(len(every))
    worst = 0.0
    for b, h, t in [every[i] for i in sorted({0, len(every) - 1, *rng.integers(0, len(every), rows)})]:
        n = max(0, min(lengths[b], table.shape[1] * size))
        ids = table[b]
        ok = (ids >= 0) & (ids < k.shape[0])
        place = np.where(ok, ids, 0)
        ks, vs = (x[place, h * Hkv // H].reshape(-1, x.shape[-1]) for x in (kn, vn))
        mine, before = set(), -1
        for s in selected[b, h * Hkv // H, t].tolist():  # ascending entries within the row
            if before < s < table.shape[1]:
                mine.add(s)
            before = s
        hidden = [j for j in range(len(ks)) if j // size not in mine or not ok[j // size]]
        ref, bound = attend_row(qn[b, h, t], ks, vs, n - T + t, n, scale=options.get("scale"),
                                softcap=options.get("softcap", 0.0), dtype=dt, out_dtype=dt, hidden=hidden)
        assert np.isfinite(got[b, h, t]).all(), f"{label}: row {b, h, t} is not finite"
        off = np.abs(got[b, h, t] - ref)
        worst = max(worst, float((off / (bound + 1e-300)).max()))
        assert (off <= bound).all(), f"{label}: row {b, h, t} off by {off.max():.3e}, bound {bound[off.argmax()]:.3e}"
    print(f"{label}: at most {worst:.2f} of the bound", flush=True)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [8, 24, 64, 80, 128, 136, 256])
def test_select_head_dims(ofh, dt, D):
    check_select(ofh, dt, [300, 17, 64, 65, 0, 1000], 6, 2, 1, D, 16, 5, seed=D)
    check_select(ofh, dt, [900, 640], 3, 3, 2, D, 32, 8, seed=D + 1)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (5, 1), (40, 1), (16, 8), (64, 2)])
def test_select_head_groups(ofh, dt, H, Hkv):
    check_select(ofh, dt, [500, 333], H, Hkv, 1, 64, 16, 7, seed=H)
    check_select(ofh, dt, [400], H, Hkv, 3, 256, 16, 6, seed=H + 1)  # more heads than fit the kept queries at once


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("pages,first,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (2, 1, 1), (3, 1, 2), (4, 0, 0), (9, 3, 2),
                                                (64, 1, 2), (200, 100, 99)])
def test_select_counts(ofh, dt, pages, first, recent):
    check_select(ofh, dt, [16 * pages, 16 * pages + 1, 16 * pages + 17, 5000, 3, 0], 4, 2, 2, 64, 16, pages, first, recent,
                 seed=pages)


def test_select_options(ofh):
    for i, options in enumerate([dict(scale=-0.1), dict(softcap=5.0), dict(scale=0.3), dict(max_key_splits=1),
                                 dict(max_key_splits=4)]):
        check_select(ofh, "bf16", [2000, 700], 8, 2, 1, 128, 16, 30, seed=i, **options)
        check_select(ofh, "f32", [2000, 700], 8, 2, 2, 64, 64, 9, seed=i, **options)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_select_ties(ofh, dt):
    """Few different scores: ties go to the lower page."""
    lengths = [3000, 1601]
    table, total = make_table(1, lengths, 16)
    k = torch.from_numpy(np.random.default_rng(0).integers(-1, 2, (total, 2, 16, 32))).to(TYPES[dt])
    k[:, :, :, 1:] = 0
    q = torch.from_numpy(np.random.default_rng(1).integers(-1, 2, (2, 4, 3, 32))).to(TYPES[dt])
    check_select(ofh, dt, lengths, 4, 2, 3, 32, 16, 20, k=k, q=q, table=table)
    check_select(ofh, dt, lengths, 4, 2, 3, 32, 16, 20, 0, 0, k=torch.zeros_like(k), q=q, table=table)
    # sums of both signs of zero are one score
    k = torch.zeros_like(k)
    k[::2] = -0.0
    check_select(ofh, dt, lengths, 4, 2, 3, 32, 16, 20, 2, 1, k=k, q=q, table=table, attend=False)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_select_values(ofh, dt):
    """NaN scores are above all, infinite ones above and below; pages outside the
    pool are below all."""
    lengths = [800, 640]
    table, total = make_table(2, lengths, 16)
    k = randn(3, (total, 2, 16, 64), dt)
    bounds = torch.zeros((total, 2, 2, 64), dtype=TYPES[dt], device="cuda")
    ofh.page_bounds(k.cuda(), bounds, i32(table), i32(lengths))
    bounds[table[0, 30], :, :, 3] = NAN
    bounds[table[0, 35], :, 1, 5] = INF
    bounds[table[1, 20], 0, 0, 6] = -INF
    bounds[table[1, 7], :, 0] = -INF
    bounds[table[1, 7], :, 1] = -INF
    table[0, 10:20] = -1
    table[1, 33] = total
    for pages in (6, 34, 39):
        check_select(ofh, dt, lengths, 4, 2, 1, 64, 16, pages, k=k, table=table, bounds=bounds, attend=False)
    check_select(ofh, dt, lengths, 4, 2, 1, 64, 16, 45, k=k, table=table, bounds=bounds)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_select_many_pages(ofh, dt):
    """More candidates than a workgroup keeps, and many pages chosen."""
    check_select(ofh, dt, [16 * 20011 - 5, 16 * 16391], 2, 1, 1, 8, 16, 50, attend=False)
    check_select(ofh, dt, [16 * 20011 - 5], 2, 1, 1, 8, 16, 18000, 7, 9, attend=False)
    check_select(ofh, dt, [16 * 5000], 2, 1, 1, 16, 16, 700)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_selected_lists(ofh, dt):
    """Lists of the program's own making: empty, short, with entries that select nothing."""
    F = ofh
    lengths, size, T, H, Hkv, D = [200, 90, 16, 0], 16, 2, 8, 2, 64
    table, total = make_table(4, lengths, size)
    table[0, 5] = -1
    k, v, q = randn(0, (total, Hkv, size, D), dt), randn(1, (total, Hkv, size, D), dt), randn(2, (4, H, T, D), dt)
    bounds = torch.zeros((total, Hkv, 2, D), dtype=TYPES[dt], device="cuda")
    a = F.SelectedAttention(k.cuda(), v.cuda(), bounds, i32(table), i32(lengths), heads=H, pages=6, query_tokens=T)
    lists = np.full((4, Hkv, T, 6), -1, np.int32)
    lists[0, 0, 0] = [0, 3, 5, 12, 13, 100]     # 13 and 100: past the table's row
    lists[0, 0, 1] = [2, 2, 2, 4, 4, 7]         # each once
    lists[0, 1, 0] = [-1, -1, -1, -1, -1, -1]
    lists[0, 1, 1] = [12, -1, -1, -1, -1, -1]
    lists[1, :, :] = [0, 1, 2, 3, 4, 5]
    lists[2, :, :, 0] = 0
    lists[3, :, :, 0] = 0
    out = a(q.cuda(), selected=i32(lists))
    check_rows("lists", out, q, k, v, table, lengths, lists, size, dt, rows=200)
    assert not out[0, 4:, 0].any() and not out[3].any()


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [NAN, INF])
def test_selected_hidden_values(ofh, dt, bad):
    """Pages that are not selected, and rows past the end of one that is, do not reach a row."""
    F = ofh
    lengths, size, H, Hkv, D = [200, 90], 32, 4, 2, 128
    table, total = make_table(4, lengths, size)
    k, v, q = randn(0, (total, Hkv, size, D), dt), randn(1, (total, Hkv, size, D), dt), randn(2, (2, H, 1, D), dt)
    bounds = torch.zeros((total, Hkv, 2, D), dtype=TYPES[dt], device="cuda")
    lists = i32([[[[0, 4, 6]]] * 2, [[[1, 2, -1]]] * 2])
    run = lambda: F.SelectedAttention(k.cuda(), v.cuda(), bounds, i32(table), i32(lengths), heads=H, pages=3)(
        q.cuda(), selected=lists)
    clean = run()
    for t in (k, v):
        t[table[0, 5]], t[table[1, 0]], t[table[0, 6], :, 8:], t[table[1, 2], :, 26:] = bad, bad, bad, bad
    assert torch.equal(run(), clean)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_select_workspace_contents(ofh, dt):
    """What the workspaces held before does not matter."""
    F = ofh
    lengths = [900, 0, 16, 500, 3000]
    table, total = make_table(9, lengths, 16)
    k, v, q = randn(0, (total, 2, 16, 64), dt).cuda(), randn(1, (total, 2, 16, 64), dt).cuda(), randn(2, (5, 8, 2, 64), dt).cuda()
    bounds = torch.zeros((total, 2, 2, 64), dtype=TYPES[dt], device="cuda")
    F.page_bounds(k, bounds, i32(table), i32(lengths))
    a = F.SelectedAttention(k, v, bounds, i32(table), i32(lengths), heads=8, pages=70, query_tokens=2)
    assert a.workspace_bytes > 0 and a.select_workspace_bytes > 0
    fill = lambda n, x: torch.full((n,), x, dtype=torch.uint8, device="cuda")
    lists = [a.select(q, workspace=fill(a.select_workspace_bytes, x)) for x in (0, 255, 127)]
    assert all(torch.equal(x, lists[0]) for x in lists)
    outs = [a(q, selected=lists[0], workspace=fill(a.workspace_bytes, x)) for x in (0, 255, 127)]
    assert all(torch.equal(x, outs[0]) for x in outs) and torch.isfinite(outs[0]).all()


def test_selected_long_lists(ofh):
    """Lists longer than the 64 entries that are looked up at once, with gaps."""
    F = ofh
    lengths, size = [16 * 400 - 3, 16 * 250], 16
    table, total = make_table(5, lengths, size)
    k, v, q = randn(0, (total, 2, size, 64), "bf16"), randn(1, (total, 2, size, 64), "bf16"), randn(2, (2, 4, 1, 64), "bf16")
    bounds = torch.zeros((total, 2, 2, 64), dtype=torch.bfloat16, device="cuda")
    lists = np.full((2, 2, 1, 200), -1, np.int32)
    for b in range(2):
        for h in range(2):
            pick = np.sort(np.random.default_rng(2 * b + h).permutation(-(-lengths[b] // size))[:200 - 30 * h])
            lists[b, h, 0, :pick.size] = pick
    for splits in (0, 1, 5):
        a = F.SelectedAttention(k.cuda(), v.cuda(), bounds, i32(table), i32(lengths), heads=4, pages=200, max_key_splits=splits)
        check_rows(f"long lists {splits}", a(q.cuda(), selected=i32(lists)), q, k, v, table, lengths, lists, size, "bf16")


def test_select_refusals(ofh):
    F = ofh
    k = torch.zeros((9, 2, 16, 64), dtype=torch.bfloat16, device="cuda")
    bounds = torch.zeros((9, 2, 2, 64), dtype=torch.bfloat16, device="cuda")
    table, lengths = i32(np.zeros((3, 4))), i32([1, 2, 3])
    make = lambda b=bounds, **o: F.SelectedAttention(k, k, b, table, lengths, **(dict(heads=4, pages=4) | o))
    for options in (dict(pages=0), dict(pages=2), dict(first_pages=3), dict(recent_pages=-1), dict(pages=4.0), dict(heads=3),
                    dict(query_tokens=0)):
        with pytest.raises(ValueError):
            make(**options)
    for b in (bounds[:8], bounds.float(), bounds[:, :, :1], bounds.cpu()):
        with pytest.raises(ValueError):
            make(b)
    a = make()
    q = torch.zeros((3, 4, 1, 64), dtype=torch.bfloat16, device="cuda")
    for bad in (q[:2], q.float(), q.cpu(), q[..., :32]):
        with pytest.raises(ValueError):
            a.select(bad)
        with pytest.raises(ValueError):
            a(bad)
    for selected in (i32(np.zeros((3, 2, 1, 5))), i32(np.zeros((3, 2, 1, 4))).long(), i32(np.zeros((3, 2, 1, 4))).cpu(),
                     i32(np.zeros((4, 1, 2, 3))).permute(3, 2, 1, 0)):
        with pytest.raises(ValueError):
            a(q, selected=selected)
        with pytest.raises(ValueError):
            a.select(q, out=selected)
    wide = F.SelectedAttention(k, k, bounds, table, lengths, heads=4, pages=3)
    assert wide.select_workspace_bytes > 0 and a.select_workspace_bytes == 0
    with pytest.raises(F.OfhError) as e:
        wide.select(q, workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))
    assert e.value.code == F.OFH_ERROR_WORKSPACE_TOO_SMALL


def test_select_graphs_and_streams(ofh):
    """A captured selection and its attention replayed, beside another graph and eager calls."""
    F = ofh
    lengths = i32([900, 800, 333])
    table, total = make_table(7, [1000, 1000, 500], 16)
    k, v = (randn(i, (total, 2, 16, 64), "bf16").cuda() for i in range(2))
    bounds = torch.zeros((total, 2, 2, 64), dtype=torch.bfloat16, device="cuda")
    F.page_bounds(k, bounds, i32(table), i32([1000, 1000, 500]))
    t = i32(table)
    a = F.SelectedAttention(k, v, bounds, t, lengths, heads=8, pages=12)
    qs = [randn(i, (3, 8, 1, 64), "bf16").cuda() for i in range(2)]
    for q in qs:
        a(q)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            selected = a.select(q)
            outs.append((selected, a(q, selected=selected), a(q)))
        graphs.append(graph)
    for step in range(4):
        lengths += 9
        for i, q in enumerate(qs):
            q.copy_(randn(10 * step + i, q.shape, "bf16"))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for q, (selected, x, y) in zip(qs, outs):
            assert torch.equal(selected, a.select(q)) and torch.equal(x, a(q)) and torch.equal(x, y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want, got = a(qs[0]), a(qs[0], stream=side)
    side.synchronize()
    assert torch.equal(got, want)


def test_cache_batch_attend_selected(ofh):
    """A cache keeps its bounds as its sequences grow, fork, shrink and move."""
    from onednn_flash_cache import PagedCache
    F = ofh
    cache = PagedCache(layers=2, num_pages=120, page_size=16, kv_heads=2, head_dim=64, bounds=True)
    rotary = F.Rotary(64)

    def step(seqs, counts, seed):
        T = max(counts)
        batch = cache.extend(seqs, counts)
        for layer in range(2):
            k, v, q = (randn(seed + 3 * layer + i, (len(seqs), h, T, 64), "bf16").cuda() for i, h in enumerate((2, 2, 8)))
            q = batch.append(layer, k, v, rotary, q)
            fresh = cache.k_bounds[layer].clone()
            F.page_bounds(cache.k_pages[layer], fresh, batch.page_table, batch.lengths)
            assert torch.equal(fresh, cache.k_bounds[layer])
        return batch, q

    seqs = [cache.add(), cache.add()]
    step(seqs, [300, 41], 0)
    seqs.append(cache.fork(seqs[0]))
    batch, q = step(seqs, [1, 1, 1], 10)
    out = batch.attend_selected(1, q, pages=6)
    assert torch.equal(batch.attend_selected(1, q, pages=6, selected=F.SelectedAttention(
        cache.k_pages[1], cache.v_pages[1], cache.k_bounds[1], batch.page_table, batch.lengths, heads=8, pages=6).select(q)), out)
    # with every page selected it is attention over all of them
    a, b = batch.attend_selected(1, q, pages=30), batch.attend(1, q)
    assert (a.float() - b.float()).abs().max() <= 2.0 ** -5 * b.float().abs().max()
    cache.truncate(seqs[0], 290)
    cache.free(seqs[1])
    cache.compact()
    batch, q = step([seqs[0], seqs[2]], [3, 3], 20)
    a, b = batch.attend_selected(1, q, pages=30), batch.attend(1, q)
    assert (a.float() - b.float()).abs().max() <= 2.0 ** -5 * b.float().abs().max()
    with pytest.raises(ValueError, match="bounds"):
        plain = PagedCache(layers=1, num_pages=4, page_size=16, kv_heads=2, head_dim=64)
        other = plain.extend([plain.add()], [1])
        other.attend_selected(0, q[:1, :, :1], pages=4)
