"""Shared prefixes: what rows do not see, in every kernel that reads the shared
keys and at every place of the ring that stages them."""

from __future__ import annotations

import numpy as np
import pytest

from hidden_values import check_rows
from test_gpu_prefix import NAN, f64, gather, i32, make, randn

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

INF = float("inf")


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def check_hidden(F, dt, n, H, Hkv, T, D, lengths, shared, key, bad, where, *, splits=1, slopes=False, seed=0, **options):
    """`n` sequences that share `shared` keys, of which one holds `bad`."""
    k, v, table = make(seed, dt, [(n, shared)], lengths, Hkv, D, D, 16)
    page, row = table[0, key // 16], key % 16
    v[page, :, row, 1] = bad
    if where == "kv":
        k[page, :, row, 1] = bad
    for b in range(n):  # past a sequence's end, in pages of its own
        if lengths[b] > shared and lengths[b] % 16:
            v[table[b, lengths[b] // 16], :, lengths[b] % 16:] = bad
            k[table[b, lengths[b] // 16], :, lengths[b] % 16:] = bad
    q = randn(seed + 3, (n, H, T, D), dt)
    alibi = 2.0 ** -torch.arange(4.0, H + 4) if slopes else None
    out = F.shared_prefix_attention(q.cuda(), k.cuda(), v.cuda(), torch.from_numpy(table).cuda(), i32(lengths),
                                    groups=[(n, shared)], max_key_splits=splits,
                                    alibi_slopes=None if alibi is None else alibi.cuda(), **options)
    kn, vn = f64(k), f64(v)
    ref = {"sinks" if x == "sink_tokens" else x: y for x, y in options.items()}
    label = f"{dt} n{n} H{H}/{Hkv} T{T} D{D} key {key} {bad} in {where} {options}"
    heads = sorted({0, H // 2, H - 1}) if not slopes else [H - 1]
    if slopes:
        ref["slope"] = float(alibi[H - 1])
    return check_rows(label, f64(out), f64(q), lambda b, h: [gather(x, table, b, h * Hkv // H)[0] for x in (kn, vn)],
                      lambda b, t: lengths[b] - T + t, lambda b: lengths[b], [[key]] * n, 1, dtype=dt, heads=heads, **ref)


# rows of a key-value head: through LDS 128 and 64 at a time, streaming 32 and 16
SIZES = [(20, 8, 2, 2), (6, 8, 2, 2), (4, 8, 2, 2), (3, 4, 2, 2)]


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("n,H,Hkv,T", SIZES)
@pytest.mark.parametrize("options", [dict(), dict(window=300, sink_tokens=5), dict(softcap=8.0), dict(slopes=True, softcap=9.0)])
def test_hidden_shared_keys(ofh, dt, D, n, H, Hkv, T, options):
    """More steps of shared keys than the ring has places for, in one workgroup; the
    key in the first of them, in those whose K is at the ring's last place and V at its
    first, and in the last. A third of the sequences ends just before it, one some steps
    before."""
    shared, step = 1024, 32 if D == 256 else 64
    for i, (at, bad, where) in enumerate([(0, NAN, "v"), (2, INF, "kv"), (4, NAN, "kv"), (7, INF, "v"), (13, NAN, "v"),
                                          (1024 // step - 1, INF, "v")]):
        key = at * step + 29
        lengths = [key - b % 7 if b % 3 == 0 else max(T, key - 100 - b) if b % 3 == 1 else shared + 1 + 9 * b for b in range(n)]
        touched, clean = check_hidden(ofh, dt, n, H, Hkv, T, D, lengths, shared, key, bad, where, seed=i, **options)
        assert clean > 0 and (touched > 0 or "window" in options)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,H,Hkv,T", SIZES)
def test_hidden_behind_windows(ofh, dt, D, n, H, Hkv, T):
    """Shared keys that the later sequences' windows have left behind, in a step that the
    earlier ones still see; the steps before it are first tokens'."""
    shared = 640
    for i, (key, bad) in enumerate([(70, NAN), (517, INF), (620, NAN)]):
        lengths = [shared + 1 + (97 * b + 60 * (b % 2)) % 500 for b in range(n)]
        touched, clean = check_hidden(ofh, dt, n, H, Hkv, T, D, lengths, shared, key, bad, "v", splits=0, seed=i, window=210,
                                      sink_tokens=33)
        assert clean > 0 and (touched > 0 or key == 70)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,H,Hkv,T", [(20, 8, 2, 3), (6, 8, 2, 3), (3, 4, 2, 3)])
def test_hidden_own_keys(ofh, dt, D, n, H, Hkv, T):
    """A new token's key that the tokens before it do not see."""
    for bad in (NAN, INF):
        k, v, table = make(1, dt, [(n, 64)], [100 + b for b in range(n)], Hkv, D, D, 16)
        lengths = [100 + b for b in range(n)]
        keys = [x - 1 - b % 2 for b, x in enumerate(lengths)]
        for b, key in enumerate(keys):
            v[table[b, key // 16], :, key % 16, 1] = bad
        q = randn(4, (n, H, T, D), dt)
        out = ofh.shared_prefix_attention(q.cuda(), k.cuda(), v.cuda(), torch.from_numpy(table).cuda(), i32(lengths),
                                          groups=[(n, 64)])
        kn, vn = f64(k), f64(v)
        touched, clean = check_rows(f"{dt} own {bad}", f64(out), f64(q),
                                    lambda b, h: [gather(x, table, b, h * Hkv // H)[0] for x in (kn, vn)],
                                    lambda b, t: lengths[b] - T + t, lambda b: lengths[b], [[x] for x in keys], 1, dtype=dt)
        assert touched > 0 and clean > 0
