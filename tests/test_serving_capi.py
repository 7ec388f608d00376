"""Argument checks of the serving entry points: everything here is refused (or
answered) on the host, before any device work."""

from __future__ import annotations

import ctypes

import pytest

ALIGNED = 0x1000  # stands for a device address: no call below reaches the device


def params(F, cls, init, **fields):
    p = cls()
    getattr(F.lib(), init)(ctypes.addressof(p))
    for name, value in fields.items():
        if isinstance(value, tuple):
            getattr(p, name)[:] = value
        else:
            setattr(p, name, value)
    return p


def window(F, **fields):
    base = dict(batch=2, heads=8, kv_heads=2, query_tokens=33, key_tokens=40, head_dim=64, value_dim=64,
                dtype=F.DTYPE_BF16, out_dtype=F.DTYPE_BF16)
    return params(F, F.WindowParams, "ofh_window_params_init", **(base | fields))


def paged(F, **fields):
    base = dict(batch=2, heads=8, kv_heads=2, head_dim=64, value_dim=64, num_pages=10, page_size=16, max_pages=5,
                dtype=F.DTYPE_BF16, out_dtype=F.DTYPE_BF16, page_table=ALIGNED, lengths=ALIGNED)
    return params(F, F.PagedParams, "ofh_paged_params_init", **(base | fields))


def write(F, **fields):
    base = dict(batch=2, kv_heads=2, tokens=3, head_dim=64, value_dim=64, num_pages=10, page_size=16, max_pages=5,
                dtype=F.DTYPE_BF16, page_table=ALIGNED, lengths=ALIGNED)
    return params(F, F.CacheWriteParams, "ofh_cache_write_params_init", **(base | fields))


def status(F, rc, code, text):
    assert rc == code and text in F.lib().ofh_last_error().decode(), (rc, F.lib().ofh_last_error())


SHARED = [
    (dict(batch=0), 1, "attention dimensions must be non-zero"),
    (dict(kv_heads=0), 1, "attention dimensions must be non-zero"),
    (dict(heads=7), 1, "heads must be a multiple of kv_heads"),
    (dict(dtype=3), 1, "unknown dtype"),
    (dict(out_dtype=2), 1, "out_dtype must equal dtype or be f32"),
    (dict(scale=float("inf")), 1, "scale must be finite"),
    (dict(softcap=-1.0), 1, "softcap must be finite and >= 0"),
    (dict(softcap=float("nan")), 1, "softcap must be finite and >= 0"),
    (dict(max_key_splits=-1), 1, "max_key_splits must be >= 0"),
    (dict(sink_tokens=4), 1, "sink_tokens need a window"),
    (dict(head_dim=60), 2, "multiples of 8 up to 256"),
    (dict(value_dim=264), 2, "multiples of 8 up to 256"),
    (dict(dtype=0, out_dtype=0, head_dim=62), 2, "multiples of 4 up to 256"),
    (dict(query_tokens=1 << 31), 2, "32-bit index range"),
    (dict(window=1 << 31), 2, "32-bit index range"),
    (dict(heads=1 << 20, kv_heads=2, query_tokens=1 << 20), 2, "32-bit index range"),
    (dict(q_strides=(4096, 64, -64)), 1, "q strides must be non-negative"),
    (dict(q_strides=(4096, 64, 60)), 2, "q strides must be multiples of 16 bytes"),
    (dict(k_strides=(4096, 64, 1 << 27)), 2, "token stride is too large"),
]


@pytest.mark.parametrize("fields,code,text", SHARED + [
    (dict(key_tokens=0), 1, "attention dimensions must be non-zero"),
    (dict(key_tokens=1 << 31), 2, "32-bit index range"),
    (dict(query_offset=1 << 31), 2, "32-bit index range"),
    (dict(struct_size=8), 1, "struct_size mismatch"),
])
def test_window_refusals(ofh, fields, code, text):
    p = window(ofh, **fields)
    L = ofh.lib()
    status(ofh, L.ofh_window_attention_fwd(ctypes.addressof(p), ALIGNED, ALIGNED, ALIGNED, ALIGNED, None, 0, None),
           code, text)
    n = ctypes.c_size_t()
    status(ofh, L.ofh_window_attention_workspace_bytes(ctypes.addressof(p), ctypes.byref(n)), code, text)


@pytest.mark.parametrize("fields,code,text", SHARED + [
    (dict(num_pages=0), 1, "must be non-zero"),
    (dict(max_pages=0), 1, "must be non-zero"),
    (dict(page_size=8), 2, "power of two, 16 or more"),
    (dict(page_size=24), 2, "power of two, 16 or more"),
    (dict(max_pages=1 << 27), 2, "2^30 tokens"),
    (dict(num_pages=1 << 31), 2, "32-bit index range"),
    (dict(table_stride=-1), 1, "table_stride must be non-negative"),
    (dict(struct_size=8), 1, "struct_size mismatch"),
])
def test_paged_refusals(ofh, fields, code, text):
    p = paged(ofh, **fields)
    L = ofh.lib()
    status(ofh, L.ofh_paged_attention_fwd(ctypes.addressof(p), ALIGNED, ALIGNED, ALIGNED, ALIGNED, None, 0, None),
           code, text)
    n = ctypes.c_size_t()
    status(ofh, L.ofh_paged_attention_workspace_bytes(ctypes.addressof(p), ctypes.byref(n)), code, text)


def test_window_query_offset_does_not_wrap(ofh):
    """A position of 2^64 - 5 + 33 wraps to 28: refused for what it is."""
    lib, need = ofh.lib(), ctypes.c_size_t()
    p = window(ofh, query_offset=(1 << 64) - 5)
    status(ofh, lib.ofh_window_attention_workspace_bytes(ctypes.addressof(p), ctypes.byref(need)), 2,
           "32-bit index range")


def test_pointers_are_checked(ofh):
    L = ofh.lib()
    for p, fwd in ((window(ofh), L.ofh_window_attention_fwd), (paged(ofh), L.ofh_paged_attention_fwd)):
        for i in range(4):
            args = [ALIGNED] * 4
            args[i] = None
            status(ofh, fwd(ctypes.addressof(p), *args, None, 0, None), 1, "must be non-null")
            args[i] = ALIGNED + 8
            status(ofh, fwd(ctypes.addressof(p), *args, None, 0, None), 2, "must be 16-byte aligned")
    for name in ("page_table", "lengths"):
        p = paged(ofh, **{name: None})
        status(ofh, L.ofh_paged_attention_fwd(ctypes.addressof(p), *[ALIGNED] * 4, None, 0, None), 1, "non-null")
        p = write(ofh, **{name: None})
        status(ofh, L.ofh_cache_write(ctypes.addressof(p), *[ALIGNED] * 4, None), 1, "non-null")
    for fwd in (L.ofh_window_attention_fwd, L.ofh_paged_attention_fwd):
        status(ofh, fwd(None, *[ALIGNED] * 4, None, 0, None), 1, "params must be non-null")


def test_workspace(ofh):
    """A split's partial rows: within the bytes that the call asks for, which a
    smaller workspace is refused for."""
    L = ofh.lib()
    n = ctypes.c_size_t()
    for p, query, fwd in (
            (paged(ofh, batch=1, max_pages=512), L.ofh_paged_attention_workspace_bytes, L.ofh_paged_attention_fwd),
            (window(ofh, batch=1, query_tokens=1, key_tokens=8192, query_offset=8191),
             L.ofh_window_attention_workspace_bytes, L.ofh_window_attention_fwd)):
        assert query(ctypes.addressof(p), ctypes.byref(n)) == 0 and n.value > 0
        status(ofh, fwd(ctypes.addressof(p), *[ALIGNED] * 4, ALIGNED, n.value - 1, None), 4,
               f"need {n.value} bytes")
        status(ofh, fwd(ctypes.addressof(p), *[ALIGNED] * 4, ALIGNED + 4, n.value, None), 2,
               "workspace must be 16-byte aligned")
        p.max_key_splits = 1
        assert query(ctypes.addressof(p), ctypes.byref(n)) == 0 and n.value == 0
        assert query(ctypes.addressof(p), None) == 1


@pytest.mark.parametrize("fields,code,text", [
    (dict(tokens=0), 1, "cache dimensions must be non-zero"),
    (dict(head_dim=0), 1, "cache dimensions must be non-zero"),
    (dict(dtype=7), 1, "unknown dtype"),
    (dict(page_size=17), 2, "power of two, 16 or more"),
    (dict(num_pages=0), 1, "must be non-zero"),
    (dict(k_strides=(1, -1, 1)), 1, "cache strides must be non-negative"),
    (dict(v_page_strides=(-1, 1, 1)), 1, "cache strides must be non-negative"),
    (dict(tokens=1 << 31), 2, "32-bit index range"),
    (dict(tokens=1 << 28, batch=1 << 10), 2, "launch range"),
    (dict(struct_size=8), 1, "struct_size mismatch"),
])
def test_cache_write_refusals(ofh, fields, code, text):
    p = write(ofh, **fields)
    status(ofh, ofh.lib().ofh_cache_write(ctypes.addressof(p), *[ALIGNED] * 4, None), code, text)


def test_cache_write_pointers(ofh):
    p = write(ofh)
    for i in range(4):
        args = [ALIGNED] * 4
        args[i] = None
        status(ofh, ofh.lib().ofh_cache_write(ctypes.addressof(p), *args, None), 1, "must be non-null")


@pytest.mark.parametrize("src,dst,text", [
    ([0, 1], [5, 5], "copied to twice"),
    ([0, 1], [1, 2], "both copied from and copied to"),
    ([3], [3], "both copied from and copied to"),
    ([-1], [2], "within the pool"),
    ([1], [8], "within the pool"),
])
def test_copy_pages_refusals(ofh, src, dst, text):
    pools = (ctypes.c_void_p * 1)(ALIGNED)
    n = len(src)
    args = ((ctypes.c_int32 * n)(*src), (ctypes.c_int32 * n)(*dst), n, None)
    status(ofh, ofh.lib().ofh_cache_copy_pages(pools, 1, 8, 64, 0, *args), 1, text)


def test_copy_pages_geometry(ofh):
    L = ofh.lib()
    pools = (ctypes.c_void_p * 2)(ALIGNED, None)
    one, two = (ctypes.c_int32 * 1)(0), (ctypes.c_int32 * 1)(1)
    status(ofh, L.ofh_cache_copy_pages(pools, 2, 8, 64, 0, one, two, 1, None), 1, "non-null")
    pools[1] = ALIGNED + 1
    status(ofh, L.ofh_cache_copy_pages(pools, 2, 8, 64, 0, one, two, 1, None), 2, "2-byte aligned")
    status(ofh, L.ofh_cache_copy_pages(pools, 1, 8, 64, 32, one, two, 1, None), 1, "must not overlap")
    status(ofh, L.ofh_cache_copy_pages(pools, 1, 8, 63, 0, one, two, 1, None), 2, "2-byte elements")
    status(ofh, L.ofh_cache_copy_pages(pools, 0, 8, 64, 0, one, two, 1, None), 1, "non-zero")
    status(ofh, L.ofh_cache_copy_pages(pools, 1, 8, 64, 0, None, two, 1, None), 1, "non-null")
    assert L.ofh_cache_copy_pages(pools, 1, 8, 64, 0, None, None, 0, None) == 0  # nothing to copy


def test_python_entries_refuse_before_a_launch(ofh):
    """Tensors that do not fit are refused with ValueError; on host tensors every
    call ends there."""
    torch = pytest.importorskip("torch")
    F = ofh
    q, k = torch.zeros(1, 4, 3, 64), torch.zeros(1, 2, 5, 64)
    with pytest.raises(ValueError, match="GPU tensor"):
        F.window_attention(q, k, k)
    with pytest.raises(ValueError, match="rank-4"):
        F.window_attention(q[0], k, k)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        F.window_attention(q.double(), k, k)
    with pytest.raises(ValueError, match="must not be empty"):
        F.window_attention(q[:, :, :0], k, k)
    with pytest.raises(ValueError, match="last axis"):
        F.window_attention(q.transpose(2, 3), k, k)
    pool = torch.zeros(8, 2, 16, 64)
    table, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):
        F.paged_attention(q, pool, pool, table, lengths)
    with pytest.raises(ValueError, match="GPU tensor"):
        F.cache_write(k, k, pool, pool, table, lengths)
    with pytest.raises(ValueError, match="GPU tensors"):
        F.copy_pages([pool], [0], [1])
    with pytest.raises(ValueError, match="pools must be"):
        F.copy_pages([], [0], [1])
