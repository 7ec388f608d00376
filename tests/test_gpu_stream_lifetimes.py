"""Device tensors of the library's own, read on a stream other than the one they
were made on by an object that is dropped at once: their memory is not given to
the next tensor while the call may still read it."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def busy_stream():
    """A side stream with work ahead of the calls, 40 ms. (Copies to the device may wait
    for it: objects are made before.)"""
    torch.cuda.current_stream().synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)
    return side


def reused(ptrs, nbytes):
    """Whether tensors of the current stream get this memory now."""
    held = [torch.empty(nbytes, dtype=torch.uint8, device="cuda") for _ in range(64)]
    return any(t.data_ptr() in ptrs for t in held)


def pools():
    k = torch.randn(40, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    table = torch.arange(4, dtype=torch.int32, device="cuda").repeat(8, 1)
    return k, torch.randn_like(k), table, torch.full((8,), 64, dtype=torch.int32, device="cuda")


def spy(monkeypatch, F):
    """Addresses of the tensors that the library keeps from here on."""
    ptrs = set()
    plain = F._Kept.__init__

    def init(self, torch, *tensors):
        plain(self, torch, *tensors)
        ptrs.update(t.data_ptr() for t in tensors)

    monkeypatch.setattr(F._Kept, "__init__", init)
    return ptrs


@pytest.mark.parametrize("handle", [False, True])
def test_groups_of_one_call(ofh, monkeypatch, handle):
    k, v, table, lengths = pools()
    q = torch.randn(8, 8, 1, 64, device="cuda", dtype=torch.bfloat16)
    want = ofh.shared_prefix_attention(q, k, v, table, lengths, groups=[(8, 48)])
    ptrs, busy = spy(monkeypatch, ofh), busy_stream()
    out = ofh.shared_prefix_attention(q, k, v, table, lengths, groups=[(8, 48)], stream=busy.cuda_stream if handle else busy)
    assert len(ptrs) == 2 and not reused(ptrs, 64)
    busy.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("current", [False, True])
def test_groups_of_a_dropped_object(ofh, monkeypatch, current):
    k, v, table, lengths = pools()
    q = torch.randn(8, 8, 1, 64, device="cuda", dtype=torch.bfloat16)
    want = ofh.shared_prefix_attention(q, k, v, table, lengths, groups=[(8, 48)])
    ptrs = spy(monkeypatch, ofh)
    attend = ofh.SharedPrefixAttention(k, v, table, lengths, groups=[(8, 48)], heads=8)
    busy = busy_stream()
    if current:
        with torch.cuda.stream(busy):
            out = attend(q)
    else:
        out = attend(q, stream=busy)
    del attend
    assert len(ptrs) == 2 and not reused(ptrs, 64) and not busy.query()
    busy.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("current", [False, True])
def test_frequencies_of_a_dropped_rotary(ofh, monkeypatch, current):
    x = torch.randn(2, 4, 5, 64, device="cuda")
    want = ofh.Rotary(64)(x, offset=9)
    ptrs = spy(monkeypatch, ofh)
    rotary = ofh.Rotary(64)
    busy = busy_stream()
    if current:
        with torch.cuda.stream(busy):
            out = rotary(x, offset=9)
    else:
        out = rotary(x, offset=9, stream=busy)
    del rotary
    assert len(ptrs) == 1 and not reused(ptrs, 256) and not busy.query()
    busy.synchronize()
    assert torch.equal(out, want)


def test_frequencies_of_a_dropped_appender(ofh, monkeypatch):
    k_pages, v_pages, table, lengths = pools()
    table = torch.arange(32, dtype=torch.int32, device="cuda").reshape(8, 4)
    k, q = (torch.randn(8, h, 1, 64, device="cuda", dtype=torch.bfloat16) for h in (2, 8))
    want = ofh.cache_append(k, k, k_pages, v_pages, table, lengths, ofh.Rotary(64), q=q)
    ptrs = spy(monkeypatch, ofh)
    append = ofh.CacheAppender(k_pages, v_pages, table, lengths, ofh.Rotary(64))
    busy = busy_stream()
    out = append(k, k, q, stream=busy)
    del append
    assert len(ptrs) == 1 and not reused(ptrs, 256) and not busy.query()
    busy.synchronize()
    assert torch.equal(out, want)


def test_frequencies_from_a_device_are_there(ofh, monkeypatch):
    """A Rotary made from a device tensor is ready when its constructor returns: what
    was looked at last is its own copy, not the tensor before it was copied."""
    seen, plain = [], torch.isfinite
    monkeypatch.setattr(torch, "isfinite", lambda t: seen.append(t.data_ptr()) or plain(t))
    given = torch.rand(32, dtype=torch.float64, device="cuda")
    rotary = ofh.Rotary(64, frequencies=given)
    assert seen == [rotary.frequencies.data_ptr()] and rotary.frequencies.data_ptr() != given.data_ptr()
    given[3] = float("nan")
    with pytest.raises(ValueError, match="finite"):
        ofh.Rotary(64, frequencies=given)


@pytest.mark.parametrize("method", ["attend", "attend_shared", "attend_selected", "write", "append"])
def test_tables_of_a_dropped_batch(ofh, monkeypatch, method):
    """A cache's batch is dropped with the next step's, and its tables with it."""
    from onednn_flash_cache import PagedCache
    cache = PagedCache(layers=1, num_pages=40, page_size=16, kv_heads=2, head_dim=64, bounds=True)
    seqs = [cache.add() for _ in range(4)]
    k, q = (torch.randn(4, h, 40, 64, device="cuda", dtype=torch.bfloat16) for h in (2, 8))
    cache.extend(seqs, [40] * 4).write(0, k, k)
    rotary = ofh.Rotary(64)
    ptrs = spy(monkeypatch, ofh)
    batch = cache.extend(seqs, [1] * 4)
    k, q = k[:, :, :1].contiguous(), q[:, :, :1].contiguous()
    batch.write(0, k, k)
    call = {"attend": lambda **o: batch.attend(0, q, **o), "attend_shared": lambda **o: batch.attend_shared(0, q, **o),
            "attend_selected": lambda **o: batch.attend_selected(0, q, pages=3, first_pages=0, **o),
            "write": lambda: batch.write(0, k, k), "append": lambda: batch.append(0, k, k, rotary, q)}[method]
    want = call()  # (also makes the batch's groups)
    pages = cache.k_pages.clone()
    for current in (True, False) if method.startswith("attend") else (True,):
        busy = busy_stream()
        if current:
            with torch.cuda.stream(busy):
                out = call()
        else:
            out = call(stream=busy)
    del batch, call
    assert len(ptrs) == (5 if method == "attend_shared" else 3) and not reused(ptrs, 64) and not busy.query()
    busy.synchronize()
    assert torch.equal(cache.k_pages, pages) and (want is None or torch.equal(out, want))
