"""Rotary positions and appending: rows that hold a NaN or an infinity."""

from __future__ import annotations

import pytest

from test_gpu_rotary import TYPES, randn

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def bits(t):
    return t.contiguous().view(torch.int32 if t.dtype == torch.float32 else torch.int16)


def pairs(columns, part, interleaved):
    """The columns that those turn with."""
    out = set()
    for c in columns:
        out |= {c} if c >= part else {c, c ^ 1} if interleaved else {c, (c + part // 2) % part}
    return sorted(out)


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,part", [(64, 64), (80, 48), (50, 34)])  # words, words and copied columns, single columns
@pytest.mark.parametrize("T", [3, 5000])  # four wavefronts per token, one
def test_rows_with_bad_values(ofh, dt, interleaved, D, part, T):
    """A bad value stays in its pair, or its column past rotary_dim; everything else is
    bit for bit what it was."""
    rotary = ofh.Rotary(D, rotary_dim=part, interleaved=interleaved)
    columns = [2, part // 2 + 5, D - 1]
    spoilt = pairs(columns, part, interleaved)
    for bad in (NAN, INF, -INF):
        for transpose in (False, True):
            x = randn(0, (1, 2, T, D), dt).cuda()
            clean = rotary(x, offset=3, transpose=transpose)
            x[0, 1, T - 2, columns] = bad
            got = rotary(x, offset=3, transpose=transpose)
            row = got[0, 1, T - 2]
            assert not torch.isfinite(row[spoilt]).any()
            if part < D:
                assert torch.equal(bits(row[D - 1:]), bits(x[0, 1, T - 2, D - 1:]))
            row[spoilt] = clean[0, 1, T - 2][spoilt]
            assert torch.equal(bits(got), bits(clean))


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,part", [(64, 64), (80, 48), (50, 34)])
@pytest.mark.parametrize("T", [3, 1500])
def test_appended_bad_values(ofh, dt, interleaved, D, part, T):
    """As above, on the way into a cache; rows of padding, whatever they hold, leave pages
    as they were and queries 0."""
    B, H, Hkv, size = 4, 4, 2, 16
    rotary = ofh.Rotary(D, rotary_dim=part, interleaved=interleaved)
    counts = [T, 1, 0, T - 1]
    lengths = [c + 5 + b for b, c in enumerate(counts)]
    per = -(-max(lengths) // size)
    table = torch.randperm(B * per, generator=torch.Generator().manual_seed(0)).to(torch.int32).reshape(B, per).cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32).cuda()

    def run(k, v, q):
        pages = [torch.full((B * per, Hkv, size, D), 3.0, dtype=TYPES[dt], device="cuda") for _ in range(2)]
        out = ofh.cache_append(k, v, *pages, table, i32(lengths), rotary, q=q, counts=i32(counts))
        return (*pages, out)

    k, v, q = (randn(i, (B, h, T, D), dt).cuda() for i, h in enumerate((Hkv, Hkv, H)))
    clean = run(k, v, q)
    columns = [2, part // 2 + 5, D - 1]
    spoilt = pairs(columns, part, interleaved)
    for bad in (NAN, INF, -INF):
        k2, v2, q2 = k.clone(), v.clone(), q.clone()
        t = T - 2  # a token of sequences 0 and 3
        k2[0, 1, t, columns] = v2[0, 1, t, columns] = q2[3, 2, t, columns] = bad
        for x in (k2, v2, q2):  # padding
            for b, c in enumerate(counts):
                x[b, :, c:] = bad
        got = run(k2, v2, q2)
        position = lengths[0] - counts[0] + t
        page, row = int(table[0, position // size]), position % size
        assert not torch.isfinite(got[0][page, 1, row][spoilt]).any()
        assert torch.equal(bits(got[1][page, 1, row]), bits(v2[0, 1, t]))
        assert not torch.isfinite(got[2][3, 2, t][spoilt]).any()
        got[0][page, 1, row, spoilt] = clean[0][page, 1, row, spoilt]
        got[1][page, 1, row] = clean[1][page, 1, row]
        got[2][3, 2, t, spoilt] = clean[2][3, 2, t, spoilt]
        for x, y in zip(got, clean):
            assert torch.equal(bits(x), bits(y))
        assert not got[2][2].any() and not got[2][1, :, 1:].any()
