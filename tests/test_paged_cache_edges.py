"""PagedCache calls that are refused before they reach a kernel: on the CPU."""

from __future__ import annotations

import pytest

import onednn_flash_cache as C

torch = pytest.importorskip("torch")


def cache(**other):
    return C.PagedCache(**(dict(layers=1, num_pages=8, page_size=16, kv_heads=2, head_dim=8, device="cpu") | other))


def test_queries_of_a_batch_with_uneven_counts():
    """Rows laid out as write takes them (from the front) would be attended at
    positions from the back."""
    c = cache()
    a, b = c.add(), c.add()
    c.extend([a, b], [20, 20])
    batch = c.extend([a, b], [3, 1])
    for T in (2, 3):
        with pytest.raises(ValueError, match=f"q has {T} tokens per sequence, the batch 1 new"):
            batch.attend(0, torch.zeros(2, 4, T, 8))
    with pytest.raises(ValueError, match="GPU tensor"):  # the last token of each: to the kernel's own checks
        batch.attend(0, torch.zeros(2, 4, 1, 8))
    with pytest.raises(ValueError, match="GPU tensor"):
        c.extend([a, b], [3, 3]).attend(0, torch.zeros(2, 4, 3, 8))


def test_rows_missing_from_a_write():
    """A write that has fewer rows than the batch made room for would fill the last
    places and leave the others as they were."""
    c = cache()
    a, b = c.add(), c.add()
    batch = c.extend([a, b], [3, 1])
    for T in (1, 2):
        rows = torch.zeros(2, 2, T, 8)
        with pytest.raises(ValueError, match=f"k has {T} tokens per sequence, the batch 3 new"):
            batch.write(0, rows, rows)
    rows = torch.zeros(2, 2, 4, 8)
    with pytest.raises(ValueError, match="GPU tensor"):  # padded: to the kernel's own checks
        batch.write(0, rows, rows)


@pytest.mark.parametrize("size", [1, 8, 24, 48])
def test_page_sizes_that_no_kernel_takes(size):
    with pytest.raises(ValueError, match="power of two, 16 or more"):
        cache(page_size=size)
    assert cache(page_size=64).pool.page_size == 64


def test_arguments_of_selected_attention(monkeypatch):
    """A batch passes a call's tensors on: the workspace among them."""
    made, called = [], []

    class Attention:
        def __init__(self, *args, **options):
            made.append(options)

        def __call__(self, q, **options):
            called.append(options)

    monkeypatch.setattr(C.F, "SelectedAttention", Attention)
    c = cache(bounds=True)
    batch = c.extend([c.add()], [1])
    call = dict(selected=1, out=2, workspace=3, stream=None)
    batch.attend_selected(0, torch.zeros(1, 4, 1, 8), pages=4, recent_pages=1, **call)
    assert made == [dict(heads=4, query_tokens=1, pages=4, recent_pages=1)] and called == [call]


@pytest.mark.parametrize("dtype,good,bad", [(torch.float32, (4, 20, 256), (2, 66, 260)), (torch.bfloat16, (8, 24, 256), (4, 20, 264)),
                                            (torch.float16, (8, 136), (12, 260))])
def test_head_dims_of_a_cache_with_bounds(dtype, good, bad):
    """The bounds' kernels take rows of 16-byte words up to 256 columns: others are refused
    when the cache is made, not by a write whose rows are then in their pages."""
    for D in good:
        assert cache(head_dim=D, dtype=dtype, bounds=True).k_bounds.shape == (1, 8, 2, 2, D)
    for D in bad:
        with pytest.raises(ValueError, match="a cache with bounds needs"):
            cache(head_dim=D, dtype=dtype, bounds=True)
        assert cache(head_dim=D, dtype=dtype).k_bounds is None
