"""On which streams the library's own device tensors are made and read, so that
their memory is not given away while a kernel may still read it: on the CPU, with
stand-ins for torch's streams."""

from __future__ import annotations

import contextlib
import types

import pytest

import onednn_flash_hip as F

torch = pytest.importorskip("torch")


class Stream:
    def __init__(self, handle):
        self.cuda_stream = handle


class ExternalStream(Stream):
    pass


class Tensor:
    def __init__(self, index=0):
        self.device = types.SimpleNamespace(index=index)
        self.recorded = []

    def record_stream(self, stream):
        self.recorded.append(stream.cuda_stream)


class Torch:
    """What _Kept asks of torch; `current` is the current stream."""

    def __init__(self):
        self.current = Stream(0)
        self._C = types.SimpleNamespace(_cuda_getCurrentRawStream=lambda index: self.current.cuda_stream)
        self.cuda = types.SimpleNamespace(Stream=Stream, ExternalStream=ExternalStream, current_stream=lambda index: self.current)


def test_kept_tensors_know_their_streams():
    t = Torch()
    tensors = Tensor(), Tensor()
    kept = F._Kept(t, *tensors)
    kept.used(None)         # the stream that they were made on
    kept.used(Stream(0))
    kept.used(7)            # a handle: the caller keeps the object
    kept.used(ExternalStream(9))
    assert all(x.recorded == [] for x in tensors)
    kept.used(Stream(3))
    kept.used(Stream(3))    # (known by now)
    t.current = Stream(5)
    kept.used(None)
    kept.used(None)
    assert all(x.recorded == [3, 5] for x in tensors)
    on_cpu = F._Kept(t, Tensor(None))
    on_cpu.used(None)
    on_cpu.used(Stream(3))
    assert on_cpu.tensors[0].recorded == []


def test_groups_of_a_list_are_made_on_the_calls_stream(monkeypatch):
    """They are freed when the call returns, so they belong to the stream that reads them."""
    now, made = [None], []

    @contextlib.contextmanager
    def on_stream(torch, device, stream):
        now[0] = stream
        yield
        now[0] = None

    class Attention:
        def __init__(self, *args, **options):
            made.append(now[0])

        def __call__(self, q, *, stream=None, **options):
            return stream

    monkeypatch.setattr(F, "_on_stream", on_stream, raising=False)
    monkeypatch.setattr(F, "SharedPrefixAttention", Attention)
    q = torch.zeros(1, 1, 1, 8)
    for stream in (None, 7, Stream(3)):
        assert F.shared_prefix_attention(q, q, q, q, q, groups=[(1, 0)], stream=stream) is stream
        assert made[-1] is stream


def test_on_stream_of_the_cpu():
    with F._on_stream(torch, torch.device("cpu"), 7):
        pass


def test_batches_tell_their_tables(monkeypatch):
    import onednn_flash_cache as C
    cache = C.PagedCache(layers=1, num_pages=8, page_size=16, kv_heads=2, head_dim=8, device="cpu", bounds=True)
    batch = cache.extend([cache.add()], [1])
    assert [id(t) for t in batch._kept.tensors] == [id(t) for t in (batch.page_table, batch.lengths, batch.counts)]
    told = []
    monkeypatch.setattr(batch._kept, "used", told.append)
    side, q, k = Stream(3), torch.zeros(1, 4, 1, 8), torch.zeros(1, 2, 1, 8)
    for call in (lambda: batch.write(0, k, k), lambda: batch.append(0, k, k, None), lambda: batch.attend(0, q),
                 lambda: batch.attend(0, q, stream=side), lambda: batch.attend_shared(0, q, stream=side),
                 lambda: batch.attend_selected(0, q, pages=4, stream=side)):
        with pytest.raises(ValueError, match="GPU"):  # (past what a cache on the CPU can do)
            call()
    assert told == [None, None, None, side, side, side]
