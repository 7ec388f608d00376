"""Selected pages at the edge of what the entries take, against the references of
test_gpu_select.py."""

from __future__ import annotations

import numpy as np
import pytest

from test_gpu_select import INF, TYPES, check_select, make_table, randn

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
