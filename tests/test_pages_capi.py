"""Argument checks of attention over shared prefixes and selected pages, of page
bounds and of the selection: refused on the host, before any device work."""

from __future__ import annotations

import ctypes

import pytest

from test_serving_capi import ALIGNED, paged, params, status

A = ALIGNED


def groups(F, **fields):
    base = dict(groups=1, starts=A, shared_tokens=A, least_shared=32, most_shared=32)
    return params(F, F.PrefixGroupsParams, "ofh_prefix_groups_init", **(base | fields))


def bounds(F, **fields):
    base = dict(batch=2, kv_heads=2, tokens=3, head_dim=64, num_pages=10, page_size=16, max_pages=5, dtype=F.DTYPE_BF16,
                page_table=A, lengths=A)
    return params(F, F.PageBoundsParams, "ofh_page_bounds_params_init", **(base | fields))


def select(F, **fields):
    base = dict(batch=2, heads=8, kv_heads=2, head_dim=64, num_pages=10, page_size=16, max_pages=5, dtype=F.DTYPE_BF16,
                page_table=A, lengths=A, pages=4, first_pages=1, recent_pages=2)
    return params(F, F.SelectParams, "ofh_select_params_init", **(base | fields))


PAGED = [
    (dict(batch=0), 1, "attention dimensions must be non-zero"),
    (dict(heads=7), 1, "heads must be a multiple of kv_heads"),
    (dict(dtype=3), 1, "unknown dtype"),
    (dict(head_dim=60), 2, "multiples of 8 up to 256"),
    (dict(page_size=24), 2, "page_size must be a power of two"),
    (dict(max_pages=0), 1, "num_pages and max_pages must be non-zero"),
    (dict(struct_size=8), 1, "struct_size mismatch"),
    (dict(batch=1 << 16, heads=1 << 10, query_tokens=1 << 6), 2, "32-bit index range"),
]


@pytest.mark.parametrize("fields,code,text", PAGED)
def test_paged_refusals(ofh, fields, code, text):
    L, n = ofh.lib(), ctypes.c_size_t()
    p, g = paged(ofh, **fields), groups(ofh)
    at, ag = ctypes.addressof(p), ctypes.addressof(g)
    status(ofh, L.ofh_shared_prefix_attention_fwd(at, ag, A, A, A, A, None, 0, None), code, text)
    status(ofh, L.ofh_shared_prefix_workspace_bytes(at, ag, ctypes.byref(n)), code, text)
    status(ofh, L.ofh_selected_attention_fwd(at, A, 4, A, A, A, A, None, 0, None), code, text)
    status(ofh, L.ofh_selected_attention_workspace_bytes(at, 4, ctypes.byref(n)), code, text)


@pytest.mark.parametrize("fields,code,text", [
    (dict(struct_size=8), 1, "struct_size mismatch"),
    (dict(groups=0), 1, "groups must be 1 to batch"),
    (dict(groups=3), 1, "groups must be 1 to batch"),
    (dict(least_shared=48), 1, "in this order"),
    (dict(most_shared=96), 1, "within the table's tokens"),
    (dict(sharing_groups=2), 1, "within the batch's"),
    (dict(sharing_sequences=3), 1, "within the batch's"),
    (dict(most_sequences=3), 1, "within the batch's"),
])
def test_group_refusals(ofh, fields, code, text):
    L, n = ofh.lib(), ctypes.c_size_t()
    p, g = paged(ofh), groups(ofh, **fields)
    at, ag = ctypes.addressof(p), ctypes.addressof(g)
    status(ofh, L.ofh_shared_prefix_attention_fwd(at, ag, A, A, A, A, None, 0, None), code, text)
    status(ofh, L.ofh_shared_prefix_workspace_bytes(at, ag, ctypes.byref(n)), code, text)


def test_prefix_pointers(ofh):
    L, n = ofh.lib(), ctypes.c_size_t()
    p = paged(ofh)
    at = ctypes.addressof(p)
    for fields in (dict(starts=None), dict(shared_tokens=None)):
        g = groups(ofh, **fields)
        status(ofh, L.ofh_shared_prefix_attention_fwd(at, ctypes.addressof(g), A, A, A, A, None, 0, None), 1,
               "starts and shared_tokens must be non-null")
    status(ofh, L.ofh_shared_prefix_attention_fwd(at, None, A, A, A, A, None, 0, None), 1, "groups must be non-null")
    g = groups(ofh)
    status(ofh, L.ofh_shared_prefix_attention_fwd(None, ctypes.addressof(g), A, A, A, A, None, 0, None), 1,
           "params must be non-null")
    status(ofh, L.ofh_shared_prefix_workspace_bytes(at, ctypes.addressof(g), None), 1, "bytes must be non-null")
    for i in range(4):
        args = [A] * 4
        args[i] = None
        status(ofh, L.ofh_shared_prefix_attention_fwd(at, ctypes.addressof(g), *args, None, 0, None), 1, "must be non-null")
        args[i] = A + 2
        status(ofh, L.ofh_shared_prefix_attention_fwd(at, ctypes.addressof(g), *args, None, 0, None), 2, "16-byte aligned")
    # scratch of every call: an empty or unaligned workspace is refused
    assert L.ofh_shared_prefix_workspace_bytes(at, ctypes.addressof(g), ctypes.byref(n)) == 0 and n.value > 0
    status(ofh, L.ofh_shared_prefix_attention_fwd(at, ctypes.addressof(g), A, A, A, A, A, n.value - 1, None), 4,
           "workspace too small")
    status(ofh, L.ofh_shared_prefix_attention_fwd(at, ctypes.addressof(g), A, A, A, A, A + 8, n.value, None), 2,
           "workspace must be 16-byte aligned")


def test_selected_refusals(ofh):
    L, n = ofh.lib(), ctypes.c_size_t()
    p = paged(ofh)
    at = ctypes.addressof(p)
    status(ofh, L.ofh_selected_attention_fwd(at, A, 0, A, A, A, A, None, 0, None), 1, "pages must be non-zero")
    status(ofh, L.ofh_selected_attention_fwd(at, None, 4, A, A, A, A, None, 0, None), 1, "selected must be non-null")
    status(ofh, L.ofh_selected_attention_fwd(at, A, 1 << 27, A, A, A, A, None, 0, None), 2, "32-bit index range")
    status(ofh, L.ofh_selected_attention_workspace_bytes(at, 4, None), 1, "bytes must be non-null")
    windowed = paged(ofh, window=10)
    status(ofh, L.ofh_selected_attention_fwd(ctypes.addressof(windowed), A, 4, A, A, A, A, None, 0, None), 2, "take no window")
    assert L.ofh_selected_attention_workspace_bytes(at, 4, ctypes.byref(n)) == 0


SHARED = [
    (dict(batch=0), 1, "cache dimensions must be non-zero"),
    (dict(kv_heads=0), 1, "cache dimensions must be non-zero"),
    (dict(head_dim=0), 1, "cache dimensions must be non-zero"),
    (dict(head_dim=60), 2, "multiple of 8 up to 256"),
    (dict(head_dim=264), 2, "multiple of 8 up to 256"),
    (dict(dtype=0, head_dim=62), 2, "multiple of 4 up to 256"),
    (dict(dtype=5), 1, "unknown dtype"),
    (dict(page_size=8), 2, "page_size must be a power of two"),
    (dict(num_pages=0), 1, "num_pages and max_pages must be non-zero"),
    (dict(max_pages=1 << 30), 2, "pages exceed"),
    (dict(page_table=None), 1, "page_table and lengths must be non-null"),
    (dict(lengths=None), 1, "page_table and lengths must be non-null"),
    (dict(table_stride=-1), 1, "table_stride must be non-negative"),
    (dict(bounds_strides=(512, 128, -64)), 1, "bounds strides must be non-negative"),
    (dict(bounds_strides=(512, 128, 60)), 2, "bounds strides must be multiples of 16 bytes"),
    (dict(batch=1 << 31), 2, "32-bit index range"),
    (dict(struct_size=8), 1, "struct_size mismatch"),
]


@pytest.mark.parametrize("fields,code,text", SHARED + [
    (dict(tokens=0), 1, "cache dimensions must be non-zero"),
    (dict(tokens=1 << 31), 2, "32-bit index range"),
    (dict(k_page_strides=(2048, 1024, 60)), 2, "k_pages strides must be multiples of 16 bytes"),
    (dict(batch=1 << 20, kv_heads=1 << 20, tokens=1 << 20), 2, "launch range"),
])
def test_bounds_refusals(ofh, fields, code, text):
    p = bounds(ofh, **fields)
    status(ofh, ofh.lib().ofh_page_bounds(ctypes.addressof(p), A, A, None), code, text)


def test_bounds_pointers(ofh):
    L, p = ofh.lib(), bounds(ofh)
    status(ofh, L.ofh_page_bounds(None, A, A, None), 1, "params must be non-null")
    for k, b in ((None, A), (A, None)):
        status(ofh, L.ofh_page_bounds(ctypes.addressof(p), k, b, None), 1, "must be non-null")
    for k, b in ((A + 8, A), (A, A + 8)):
        status(ofh, L.ofh_page_bounds(ctypes.addressof(p), k, b, None), 2, "16-byte aligned")


@pytest.mark.parametrize("fields,code,text", SHARED + [
    (dict(heads=0), 1, "attention dimensions must be non-zero"),
    (dict(query_tokens=0), 1, "attention dimensions must be non-zero"),
    (dict(heads=7), 1, "heads must be a multiple of kv_heads"),
    (dict(pages=0), 1, "pages must be non-zero"),
    (dict(first_pages=3), 1, "at most pages together"),
    (dict(first_pages=5, recent_pages=0), 1, "at most pages together"),
    (dict(recent_pages=(1 << 64) - 1), 1, "at most pages together"),
    (dict(pages=1 << 31), 2, "32-bit index range"),
    (dict(batch=1 << 16, heads=1 << 10, query_tokens=1 << 6), 2, "32-bit index range"),
    (dict(q_strides=(512, -64, 64)), 1, "q strides must be non-negative"),
    (dict(batch=1 << 12, heads=1 << 12, kv_heads=1 << 12, max_pages=1 << 20, page_size=16), 2, "launch range"),
])
def test_select_refusals(ofh, fields, code, text):
    p = select(ofh, **fields)
    status(ofh, ofh.lib().ofh_select_pages(ctypes.addressof(p), A, A, A, None, 0, None), code, text)


def test_select_pointers(ofh):
    L, p, n = ofh.lib(), select(ofh), ctypes.c_size_t()
    at = ctypes.addressof(p)
    status(ofh, L.ofh_select_pages(None, A, A, A, None, 0, None), 1, "params must be non-null")
    for i in range(3):
        args = [A] * 3
        args[i] = None
        status(ofh, L.ofh_select_pages(at, *args, None, 0, None), 1, "must be non-null")
    status(ofh, L.ofh_select_pages(at, A + 1, A, A, None, 0, None), 2, "aligned to their elements")
    status(ofh, L.ofh_select_pages(at, A, A + 2, A, None, 0, None), 2, "16-byte aligned")
    status(ofh, L.ofh_select_pages(at, A, A, A + 2, None, 0, None), 2, "aligned to their elements")
    # scores for a table of more pages than are taken
    assert L.ofh_select_pages_workspace_bytes(at, ctypes.byref(n)) == 0 and n.value > 0
    status(ofh, L.ofh_select_pages(at, A, A, A, A, n.value - 1, None), 4, "workspace too small")
    p.pages = 5
    assert L.ofh_select_pages_workspace_bytes(at, ctypes.byref(n)) == 0 and n.value == 0
