"""A paged key-value cache on the operators of onednn_flash_hip.

PagePool is the host bookkeeping (the library's ofh_page_pool): which sequence
holds which pages. PagedCache adds the K and V pools of a model's layers on a
GPU. A decode step of a program that serves sequences:

    cache = PagedCache(layers=L, num_pages=P, page_size=16, kv_heads=8, head_dim=128)
    seqs = [cache.add() for _ in prompts]
    rotary = F.Rotary(128)
    batch = cache.extend(seqs, [1] * len(seqs))       # room for one token each
    for layer in range(L):
        q = batch.append(layer, k, v, rotary, q)      # [B,Hkv,1,D]; turned by their positions
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


def _common_pages(a, b, most):
    """Pages that two table rows begin with alike, `most` at most. (Slices compare
    quicker than pages one by one.)"""
    low, high = 0, most
    if a[:most] == b[:most]:
        low = most
    while low < high:
        mid = (low + high + 1) // 2
        if a[low:mid] == b[low:mid]:
            low = mid
        else:
            high = mid - 1
    return a.index(-1, 0, low) if -1 in a[:low] else low


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
    sequences in them; with `bounds` also the bounds of the pages' keys, [layers, P,
    Hkv, 2, D], which batches keep up to date and attend_selected reads. Copies run on
    the current stream; a program that uses the cache from several streams orders them
    itself."""

    def __init__(self, *, layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                 value_dim: int | None = None, dtype=None, device="cuda", bounds: bool = False):
        import torch
        self._torch = torch
        self.pool = PagePool(num_pages, page_size)
        if page_size < 16 or page_size & (page_size - 1):  # (what the kernels read and write)
            raise ValueError("page_size must be a power of two, 16 or more")
        dtype = torch.bfloat16 if dtype is None else dtype
        step = 16 // dtype.itemsize
        if bounds and (head_dim % step or not 0 < head_dim <= 256):  # (refused later, a batch would have written its rows)
            raise ValueError(f"a cache with bounds needs a head_dim that is a multiple of {step} up to 256")
        shape = (layers, num_pages, kv_heads, page_size)
        # (zeros: what a page holds past its tokens is never seen, but a program may look)
        self.k_pages = torch.zeros((*shape, head_dim), dtype=dtype, device=device)
        self.v_pages = torch.zeros((*shape, head_dim if value_dim is None else value_dim), dtype=dtype, device=device)
        self.k_bounds = None
        if bounds:
            self.k_bounds = torch.zeros((layers, num_pages, kv_heads, 2, head_dim), dtype=dtype, device=device)

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
            for pages in (self.k_pages, self.v_pages, self.k_bounds):
                if pages is not None:
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
        self._rows, self._groups = rows, None
        self.page_table = torch.tensor(rows, dtype=torch.int32, device=device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.counts = torch.tensor(list(tokens), dtype=torch.int32, device=device)
        self._kept = F._Kept(torch, self.page_table, self.lengths, self.counts)

    def _check_tokens(self, k) -> None:
        if k.dim() == 4 and k.shape[2] < self._most:  # (their places would keep what the pages held)
            raise ValueError(f"k has {k.shape[2]} tokens per sequence, the batch {self._most} new ones")

    def write(self, layer: int, k, v) -> None:
        """k: [B,Hkv,T,D], v: [B,Hkv,T,Dv]; the first tokens[i] rows of each sequence."""
        self._check_tokens(k)
        self._kept.used(None)
        F.cache_write(k, v, self.cache.k_pages[layer], self.cache.v_pages[layer], self.page_table, self.lengths,
                      counts=self.counts)
        self._renew_bounds(layer)

    def _renew_bounds(self, layer: int) -> None:
        if self.cache.k_bounds is not None and self._most > 0:
            F.page_bounds(self.cache.k_pages[layer], self.cache.k_bounds[layer], self.page_table, self.lengths,
                          tokens=self._most, counts=self.counts)

    def append(self, layer: int, k, v, rotary, q=None):
        """`write` with K turned by `rotary` (a Rotary) on the way. Returns q
        [B,H,T,D], the queries of the same tokens, turned too (None without)."""
        self._check_tokens(k)
        self._kept.used(None)
        q = F.cache_append(k, v, self.cache.k_pages[layer], self.cache.v_pages[layer], self.page_table, self.lengths,
                           rotary, q=q, counts=self.counts)
        self._renew_bounds(layer)
        return q

    def attend(self, layer: int, q, **options):
        """q: [B,H,T,D], the last T of the batch's new tokens of each sequence; options as
        paged_attention. A sequence with fewer than T new tokens is refused: rows
        laid out as write takes them, from the front, would be attended at positions
        from the back (such batches go in parts of one T, or prompts through
        window_attention with the batch's lengths)."""
        self._check_queries(q)
        self._kept.used(options.get("stream"))
        return F.paged_attention(q, self.cache.k_pages[layer], self.cache.v_pages[layer], self.page_table,
                                 self.lengths, **options)

    def _check_queries(self, q) -> None:
        if q.dim() == 4 and q.shape[2] > self._fewest:
            raise ValueError(f"q has {q.shape[2]} tokens per sequence, the batch {self._fewest} new ones for some")

    @property
    def groups(self) -> F.PrefixGroups:
        """Neighbouring sequences that begin with the same pages (forks), in groups
        that together save the most reading: a sequence joins the group before it when
        the group's shared pages, times the sequences after its first, do not get
        fewer by it."""
        if self._groups is None:
            size, groups = self.cache.pool.page_size, []
            first, count, shared = self._rows[0], 1, None
            for row in self._rows[1:]:
                common = _common_pages(first, row, len(row) if shared is None else shared)
                if common > 0 and (shared is None or count * common >= (count - 1) * shared):
                    count, shared = count + 1, common
                else:
                    groups.append((count, (shared or 0) * size))
                    first, count, shared = row, 1, None
            groups.append((count, (shared or 0) * size))
            self._groups = F.PrefixGroups(groups, page_size=size, device=self.page_table.device)
        return self._groups

    def attend_shared(self, layer: int, q, **options):
        """`attend`, with the pages that forks share read once for all of them."""
        self._check_queries(q)
        self._kept.used(options.get("stream"))
        return F.shared_prefix_attention(q, self.cache.k_pages[layer], self.cache.v_pages[layer], self.page_table,
                                         self.lengths, groups=self.groups, **options)

    def attend_selected(self, layer: int, q, *, pages: int, selected=None, out=None, workspace=None, stream=None,
                        **options):
        """`attend` over `pages` of each sequence's pages, of a cache with bounds;
        options as SelectedAttention, which the other arguments are passed to."""
        self._check_queries(q)
        if self.cache.k_bounds is None:
            raise ValueError("the cache has no bounds (PagedCache(bounds=True))")
        if q.dim() != 4:
            raise ValueError("q must be a rank-4 tensor")
        self._kept.used(stream)
        attend = F.SelectedAttention(self.cache.k_pages[layer], self.cache.v_pages[layer], self.cache.k_bounds[layer],
                                     self.page_table, self.lengths, heads=q.shape[1], query_tokens=q.shape[2], pages=pages,
                                     **options)
        return attend(q, selected=selected, out=out, workspace=workspace, stream=stream)
