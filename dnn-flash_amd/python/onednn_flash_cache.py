"""A paged key-value cache on the operators of onednn_flash_hip.

PagePool is the host bookkeeping (the library's ofh_page_pool): which sequence
holds which pages. PagedCache adds the K and V pools of a model's layers on a
GPU. A decode step of a program that serves sequences:

    cache = PagedCache(layers=L, num_pages=P, page_size=16, kv_heads=8, head_dim=128)
    seqs = [cache.add() for _ in prompts]
    batch = cache.extend(seqs, [1] * len(seqs))       # room for one token each
    for layer in range(L):
        batch.write(layer, k, v)                      # [B,Hkv,1,D]
        out = batch.attend(layer, q)                  # [B,H,1,D]

`fork` shares pages until one of the sequences grows; `free` and `truncate`
give them back; `compact` moves what is in use to the front of the pools.
"""

from __future__ import annotations

import ctypes
import weakref

import onednn_flash_hip as F

_I32 = ctypes.c_int32
_I64 = ctypes.c_int64
_SZ = ctypes.c_size_t


def _fit(name, x, kind):
    """x as a C integer (ctypes itself drops the bits that do not fit)."""
    c = kind(x)
    if c.value != x:
        raise ValueError(f"{name} is out of range")
    return c


def _row(name, xs, kind):
    """A C array of the integers xs, of one element at least."""
    xs = list(xs)
    row = (kind * max(len(xs), 1))(*xs)
    if any(a != b for a, b in zip(row, xs)):
        raise ValueError(f"{name} are out of range")
    return row


class PagePool:
    """Which sequences hold which of num_pages pages of page_size tokens."""

    def __init__(self, num_pages: int, page_size: int):
        for name, x in (("num_pages", num_pages), ("page_size", page_size)):
            if isinstance(x, bool) or not isinstance(x, int) or x <= 0:
                raise ValueError(f"{name} must be a positive integer")
        self.num_pages, self.page_size = num_pages, page_size
        self._lib = F.lib()
        handle = ctypes.c_void_p()
        F.check(self._lib.ofh_page_pool_create(_fit("num_pages", num_pages, _SZ), _fit("page_size", page_size, _SZ),
                                               ctypes.byref(handle)))
        self._handle = handle
        weakref.finalize(self, self._lib.ofh_page_pool_destroy, handle)

    def add(self) -> int:
        """A new sequence without tokens."""
        seq = _I64()
        F.check(self._lib.ofh_page_pool_add(self._handle, ctypes.byref(seq)))
        return seq.value

    def extend(self, sequences, tokens) -> tuple[list[int], list[int]]:
        """Room for tokens[i] more tokens in sequences[i]: all of it, or an
        OfhError (code OFH_ERROR_OUT_OF_PAGES) and nothing changed. Returns the
        pages (src, dst) to copy before the new tokens are written."""
        n = len(sequences)
        if len(tokens) != n or any(isinstance(t, bool) or int(t) != t or t < 0 for t in tokens):
            raise ValueError("tokens must be a non-negative integer per sequence")
        src, dst, copies = (_I32 * max(n, 1))(), (_I32 * max(n, 1))(), _SZ()
        F.check(self._lib.ofh_page_pool_extend(self._handle, _row("sequences", sequences, _I64),
                                               _row("tokens", tokens, _SZ), n, src, dst, ctypes.byref(copies)))
        return list(src[:copies.value]), list(dst[:copies.value])

    def fork(self, sequence: int) -> int:
        """A new sequence with the same tokens."""
        child = _I64()
        F.check(self._lib.ofh_page_pool_fork(self._handle, _fit("sequence", sequence, _I64), ctypes.byref(child)))
        return child.value

    def truncate(self, sequence: int, length: int) -> None:
        """Drops the tokens of a sequence from `length` on."""
        if length < 0:
            raise ValueError("length must be non-negative")
        F.check(self._lib.ofh_page_pool_truncate(self._handle, _fit("sequence", sequence, _I64),
                                                 _fit("length", length, _SZ)))

    def free(self, sequence: int) -> None:
        F.check(self._lib.ofh_page_pool_free(self._handle, _fit("sequence", sequence, _I64)))

    def compact(self, most: int | None = None) -> tuple[list[int], list[int]]:
        """Moves used pages (at most `most`) to the lowest numbers. Returns the
        pages (src, dst) to copy."""
        n = self.num_pages // 2 if most is None else min(most, self.num_pages // 2)
        if n < 0:
            raise ValueError("most must be non-negative")
        src, dst, copies = (_I32 * max(n, 1))(), (_I32 * max(n, 1))(), _SZ()
        F.check(self._lib.ofh_page_pool_compact(self._handle, src, dst, n, ctypes.byref(copies)))
        return list(src[:copies.value]), list(dst[:copies.value])

    def table(self, sequences, max_pages: int) -> tuple[list[list[int]], list[int]]:
        """Page table rows (unused entries -1) and lengths."""
        n = len(sequences)
        if max_pages < 0:
            raise ValueError("max_pages must be non-negative")
        rows, lengths = (_I32 * max(n * max_pages, 1))(), (_I32 * max(n, 1))()
        F.check(self._lib.ofh_page_pool_table(self._handle, _row("sequences", sequences, _I64), n, rows,
                                              _fit("max_pages", max_pages, _SZ), lengths))
        return [list(rows[i * max_pages:(i + 1) * max_pages]) for i in range(n)], list(lengths[:n])

    @property
    def pages_in_use(self) -> int:
        used = _SZ()
        F.check(self._lib.ofh_page_pool_info(self._handle, ctypes.byref(used), None))
        return used.value

    def length(self, sequence: int) -> int:
        n = _SZ()
        F.check(self._lib.ofh_page_pool_length(self._handle, _fit("sequence", sequence, _I64), ctypes.byref(n)))
        return n.value


class PagedCache:
    """The K and V pools of `layers` layers, [layers, P, Hkv, S, D], and the
    sequences in them. Copies run on the current stream; a program that uses the
    cache from several streams orders them itself."""

    def __init__(self, *, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                 value_dim: int | None = None, dtype=None, device="cuda"):
        import torch
        self._torch = torch
        self.pool = PagePool(num_pages, page_size)
        if page_size < 16 or page_size & (page_size - 1):  # (what the kernels read and write)
            raise ValueError("page_size must be a power of two, 16 or more")
        dtype = torch.bfloat16 if dtype is None else dtype
        shape = (layers, num_pages, kv_heads, page_size)
        # (zeros: what a page holds past its tokens is never seen, but a program may look)
        self.k_pages = torch.zeros((*shape, head_dim), dtype=dtype, device=device)
        self.v_pages = torch.zeros((*shape, head_dim if value_dim is None else value_dim), dtype=dtype, device=device)

    def add(self) -> int:
        return self.pool.add()

    def fork(self, sequence: int) -> int:
        return self.pool.fork(sequence)

    def truncate(self, sequence: int, length: int) -> None:
        self.pool.truncate(sequence, length)

    def free(self, sequence: int) -> None:
        self.pool.free(sequence)

    def _copy(self, src, dst):
        if src:
            for pages in (self.k_pages, self.v_pages):
                F.copy_pages(list(pages.unbind(0)), src, dst)

    def compact(self, most: int | None = None) -> int:
        """Moves pages in use to the front of the pools; returns how many moved.
        Batches made before hold the old places."""
        src, dst = self.pool.compact(most)
        self._copy(src, dst)
        return len(src)

    def extend(self, sequences, tokens) -> "CacheBatch":
        """Room for tokens[i] new tokens in sequences[i], whose K and V the
        batch's write brings."""
        if not sequences:
            raise ValueError("a batch needs a sequence")
        self._copy(*self.pool.extend(sequences, tokens))
        return CacheBatch(self, sequences, tokens)


class CacheBatch:
    """Sequences of a cache as one batch: page table, lengths and counts on the
    GPU, as of its making."""

    def __init__(self, cache: PagedCache, sequences, tokens):
        torch = cache._torch
        self.cache = cache
        self._fewest, self._most = min(tokens), max(tokens)
        size = cache.pool.page_size
        longest = max(cache.pool.length(s) for s in sequences)
        rows, lengths = cache.pool.table(sequences, max(1, -(-longest // size)))
        device = cache.k_pages.device
        self.page_table = torch.tensor(rows, dtype=torch.int32, device=device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.counts = torch.tensor(list(tokens), dtype=torch.int32, device=device)

    def write(self, layer: int, k, v) -> None:
        """k: [B,Hkv,T,D], v: [B,Hkv,T,Dv]; the first tokens[i] rows of each sequence."""
        if k.dim() == 4 and k.shape[2] < self._most:  # (their places would keep what the pages held)
            raise ValueError(f"k has {k.shape[2]} tokens per sequence, the batch {self._most} new ones")
        F.cache_write(k, v, self.cache.k_pages[layer], self.cache.v_pages[layer], self.page_table, self.lengths,
                      counts=self.counts)

    def attend(self, layer: int, q, **options):
        """q: [B,H,T,D], the last T of the batch's new tokens of each sequence; options as
        paged_attention. A sequence with fewer than T new tokens is refused: rows
        laid out as write takes them, from the front, would be attended at positions
        from the back (such batches go in parts of one T, or prompts through
        window_attention with the batch's lengths)."""
        if q.dim() == 4 and q.shape[2] > self._fewest:
            raise ValueError(f"q has {q.shape[2]} tokens per sequence, the batch {self._fewest} new ones for some")
        return F.paged_attention(q, self.cache.k_pages[layer], self.cache.v_pages[layer], self.page_table,
                                 self.lengths, **options)
