"""Selected pages at the edge of what the entries take, against the references of
test_gpu_select.py."""

from __future__ import annotations

import numpy as np
import pytest

from serving_ref import attend_row
from test_gpu_select import INF, TYPES, bounds_ref, check_select, f64, i32, make_table, randn

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [8, 24, 40, 64, 80, 96, 136, 192, 248])
@pytest.mark.parametrize("bad", [INF, -INF])
def test_infinite_queries(ofh, dt, D, bad):
    """An infinity in one of q's columns, the last among them, ranks pages by the sign
    of that column's bound, also where a row does not fill the words of its lanes."""
    lengths = [700, 333]
    table, total = make_table(D, lengths, 16)
    for column in (D - 1, 0):
        k = randn(1, (total, 2, 16, D), dt)
        sign = torch.from_numpy(np.random.default_rng(D).choice([-1.0, 1.0], (total, 2, 1))).to(TYPES[dt])
        k[..., column] = (k[..., column].abs() + 0.25) * sign
        for H in (2, 6):
            q = randn(2, (2, H, 2, D), dt)
            q[:, ::3, :, column] = bad  # (the first head of each key-value head)
            for scale in (1.0, -1.0):
                check_select(ofh, dt, lengths, H, 2, 2, D, 16, 9, k=k, q=q, table=table, scale=scale, attend=False)


def test_workspace_of_a_batch(ofh):
    """A cache's batch takes the attention's workspace, as its other attentions do."""
    from onednn_flash_cache import PagedCache
    F = ofh
    cache = PagedCache(layers=1, num_pages=150, page_size=16, kv_heads=2, head_dim=64, bounds=True)
    seqs = [cache.add(), cache.add()]
    batch = cache.extend(seqs, [1200, 1000])
    k, q = randn(0, (2, 2, 1200, 64), "bf16").cuda(), randn(1, (2, 8, 1, 64), "bf16").cuda()
    batch.write(0, k, k)
    a = F.SelectedAttention(cache.k_pages[0], cache.v_pages[0], cache.k_bounds[0], batch.page_table, batch.lengths, heads=8,
                            pages=70)
    assert a.workspace_bytes > 0
    workspace = torch.full((a.workspace_bytes,), 255, dtype=torch.uint8, device="cuda")
    assert torch.equal(batch.attend_selected(0, q, pages=70, workspace=workspace), a(q))
    assert not (workspace == 255).all()
    with pytest.raises(F.OfhError) as e:
        batch.attend_selected(0, q, pages=70, workspace=workspace[:16])
    assert e.value.code == F.OFH_ERROR_WORKSPACE_TOO_SMALL


def check_lists(F, dt, lengths, H, Hkv, T, D, Dv, size, pages, *, slopes=False, out_f32=False, seed=0, rows=40, **options):
    """Attention over lists of the program's own making, one per token and key-value head."""
    B = len(lengths)
    table, total = make_table(seed, lengths, size)
    k, v, q = randn(seed + 1, (total, Hkv, size, D), dt), randn(seed + 2, (total, Hkv, size, Dv), dt), randn(seed + 3, (B, H, T, D), dt)
    alibi = 2.0 ** -torch.arange(4.0, H + 4) if slopes else None
    a = F.SelectedAttention(k.cuda(), v.cuda(), torch.zeros((total, Hkv, 2, D), dtype=TYPES[dt], device="cuda"), i32(table),
                            i32(lengths), heads=H, query_tokens=T, pages=pages, first_pages=0, recent_pages=0,
                            alibi_slopes=None if alibi is None else alibi.cuda(), out_dtype=torch.float32 if out_f32 else None,
                            **options)
    rng = np.random.default_rng(seed)
    lists = np.full((B, Hkv, T, pages), -1, np.int32)
    for b in range(B):
        for h in range(Hkv):
            for t in range(T):
                pick = np.sort(rng.permutation(-(-lengths[b] // size))[:rng.integers(1, pages + 1)])
                lists[b, h, t, :pick.size] = pick
    out = a(q.cuda(), selected=i32(lists))
    assert out.shape == (B, H, T, Dv) and out.dtype == (torch.float32 if out_f32 else TYPES[dt])
    got, qn, kn, vn = f64(out), f64(q), f64(k), f64(v)
    every = [(b, h, t) for b in range(B) for h in range(H) for t in range(T)]
    label = f"lists {dt} H{H}/{Hkv} T{T} D{D}/{Dv} {slopes} {out_f32} {options}"
    for b, h, t in [every[i] for i in sorted({0, len(every) - 1, *rng.integers(0, len(every), rows)})]:
        ids = table[b][:-(-lengths[b] // size)]
        ks, vs = (x[ids, h * Hkv // H].reshape(-1, x.shape[-1]) for x in (kn, vn))
        hidden = np.flatnonzero(~np.isin(np.arange(len(ks)) // size, lists[b, h * Hkv // H, t]))
        ref, bound = attend_row(qn[b, h, t], ks, vs, lengths[b] - T + t, lengths[b], scale=options.get("scale"),
                                slope=float(alibi[h]) if slopes else 0.0, softcap=options.get("softcap", 0.0), dtype=dt,
                                out_dtype="f32" if out_f32 else dt, hidden=hidden)
        assert np.isfinite(got[b, h, t]).all(), f"{label}: row {b, h, t} is not finite"
        off = np.abs(got[b, h, t] - ref)
        assert (off <= bound).all(), f"{label}: row {b, h, t} off by {off.max():.3e}, bound {bound[off.argmax()]:.3e}"


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D,Dv", [(64, 64), (64, 32), (40, 128), (128, 64), (128, 256), (256, 96), (192, 8)])
@pytest.mark.parametrize("out_f32", [False, True])
def test_selected_head_dims_and_outputs(ofh, dt, D, Dv, out_f32):
    """Values of another head dim than the keys', 32-bit output; whole tiles and parts of them."""
    check_lists(ofh, dt, [300, 65, 16], 6, 2, 2, D, Dv, 16, 9, out_f32=out_f32, seed=D)
    check_lists(ofh, dt, [3000], 8, 1, 1, D, Dv, 32, 70, out_f32=out_f32, seed=D + 1)
    check_lists(ofh, dt, [700, 900], 4, 4, 3, D, Dv, 64, 9, out_f32=out_f32, seed=D + 2, max_key_splits=1)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("options", [dict(), dict(softcap=6.0), dict(softcap=900.0), dict(scale=-0.3), dict(out_f32=True)])
def test_selected_slopes(ofh, dt, D, options):
    """ALiBi goes by the keys' places in the sequence, not in the list."""
    check_lists(ofh, dt, [333, 40, 200], 8, 2, 3, D, D, 16, 7, slopes=True, seed=D, **options)
    check_lists(ofh, dt, [4000], 16, 2, 1, D, D, 16, 150, slopes=True, seed=D + 1, **options)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_bounds_of_small_values(ofh, dt):
    """Subnormals and zeros of both signs are values as any other."""
    info = torch.finfo(TYPES[dt])
    small = info.tiny * info.eps  # the least subnormal
    values = torch.tensor([small, -small, 3 * small, -info.tiny, info.tiny, 0.0, info.max, info.min, -5 * small], dtype=TYPES[dt])
    assert (values != 0).sum() == 8
    lengths = [50, 16, 7]
    table, total = make_table(1, lengths, 16)
    pick = torch.from_numpy(np.random.default_rng(0).integers(0, 9, (total, 2, 16, 64)))
    k = values[pick]
    k[0] = k[0].abs().clamp(max=float(info.tiny))  # (a page of subnormals alone)
    bounds = torch.ones((total, 2, 2, 64), dtype=TYPES[dt])
    want = f64(bounds)
    bounds_ref(f64(k), want, table, lengths, lengths, 16)
    got = bounds.cuda()
    ofh.page_bounds(k.cuda(), got, i32(table), i32(lengths))
    np.testing.assert_array_equal(f64(got), want)
