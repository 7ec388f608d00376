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


@pytest.fixture
def busy():
    """A side stream with work ahead of the calls, a few tens of milliseconds."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(50_000_000)
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
def test_groups_of_one_call(ofh, monkeypatch, busy, handle):
    k, v, table, lengths = pools()
    q = torch.randn(8, 8, 1, 64, device="cuda", dtype=torch.bfloat16)
    want = ofh.shared_prefix_attention(q, k, v, table, lengths, groups=[(8, 48)])
    torch.cuda.current_stream().synchronize()
    ptrs = spy(monkeypatch, ofh)
    out = ofh.shared_prefix_attention(q, k, v, table, lengths, groups=[(8, 48)], stream=busy.cuda_stream if handle else busy)
    assert len(ptrs) == 2 and not reused(ptrs, 64)
    busy.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("current", [False, True])
def test_groups_of_a_dropped_object(ofh, monkeypatch, busy, current):
    k, v, table, lengths = pools()
    q = torch.randn(8, 8, 1, 64, device="cuda", dtype=torch.bfloat16)
    want = ofh.shared_prefix_attention(q, k, v, table, lengths, groups=[(8, 48)])
    torch.cuda.current_stream().synchronize()
    ptrs = spy(monkeypatch, ofh)
    attend = ofh.SharedPrefixAttention(k, v, table, lengths, groups=[(8, 48)], heads=8)
    if current:
        with torch.cuda.stream(busy):
            out = attend(q)
    else:
        out = attend(q, stream=busy)
    del attend
    assert len(ptrs) == 2 and not busy.query() and not reused(ptrs, 64)
    busy.synchronize()
    assert torch.equal(out, want)
