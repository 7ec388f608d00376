"""Frequencies of rotary positions, and argument checks of the rotation and of
appending to a cache: refused on the host, before any device work."""

from __future__ import annotations

import ctypes

import pytest

import rotary_ref

ALIGNED = 0x1000  # stands for a device address: no call below reaches the device


def fill(p, fields):
    for name, value in fields.items():
        at = p
        *path, last = name.split("__")
        for part in path:
            at = getattr(at, part)
        if isinstance(value, tuple):
            getattr(at, last)[:] = value
        else:
            setattr(at, last, value)
    return p


def rotary(F, **fields):
    p = F.RotaryParams()
    F.lib().ofh_rotary_params_init(ctypes.addressof(p))
    assert p.rotary.magnitude == 1.0
    base = dict(batch=2, heads=3, tokens=5, head_dim=64, dtype=F.DTYPE_BF16, rotary__frequencies=ALIGNED,
                rotary__rotary_dim=64)
    return fill(p, base | fields)


def append(F, **fields):
    p = F.CacheAppendParams()
    F.lib().ofh_cache_append_params_init(ctypes.addressof(p))
    assert p.rotary.magnitude == 1.0 and p.cache.struct_size == ctypes.sizeof(F.CacheWriteParams)
    base = dict(cache__batch=2, cache__kv_heads=2, cache__tokens=3, cache__head_dim=64, cache__value_dim=64,
                cache__num_pages=10, cache__page_size=16, cache__max_pages=5, cache__dtype=F.DTYPE_BF16,
                cache__page_table=ALIGNED, cache__lengths=ALIGNED, rotary__frequencies=ALIGNED, rotary__rotary_dim=64,
                heads=4)
    return fill(p, base | fields)


def status(F, rc, code, text):
    assert rc == code and text in F.lib().ofh_last_error().decode(), (rc, F.lib().ofh_last_error())


TURNS = [
    (dict(rotary__rotary_dim=0), 1, "rotary_dim must be even"),
    (dict(rotary__rotary_dim=63), 1, "rotary_dim must be even"),
    (dict(rotary__rotary_dim=66), 1, "rotary_dim must be even"),
    (dict(rotary__frequencies=None), 1, "frequencies must be non-null"),
    (dict(rotary__frequencies=ALIGNED + 4), 1, "frequencies must be aligned"),
    (dict(rotary__magnitude=float("nan")), 1, "magnitude must be finite"),
    (dict(rotary__magnitude=float("inf")), 1, "magnitude must be finite"),
    (dict(struct_size=8), 1, "struct_size mismatch"),
    (dict(o_strides=(64, 64, -2)), 1, "strides must be non-negative"),
]


@pytest.mark.parametrize("fields,code,text", TURNS + [
    (dict(batch=0), 1, "rotary dimensions must be non-zero"),
    (dict(heads=0), 1, "rotary dimensions must be non-zero"),
    (dict(tokens=0), 1, "rotary dimensions must be non-zero"),
    (dict(head_dim=0), 1, "rotary dimensions must be non-zero"),
    (dict(head_dim=1026), 2, "head_dim must be at most 1024"),
    (dict(dtype=7), 1, "unknown dtype"),
    (dict(tokens=1 << 31), 2, "32-bit index range"),
    (dict(tokens=1 << 30, batch=2), 2, "launch range"),
    (dict(heads=1 << 30), 2, "launch range"),
    (dict(x_strides=(64, -64, 64)), 1, "strides must be non-negative"),
    (dict(positions=ALIGNED, lengths=ALIGNED), 1, "either positions or lengths"),
    (dict(positions=ALIGNED, position_stride=-1), 1, "position_stride must be non-negative"),
    (dict(offset=1 << 31), 2, "offset exceeds"),
    (dict(offset=-(1 << 31) - 1), 2, "offset exceeds"),
])
def test_rotary_refusals(ofh, fields, code, text):
    p = rotary(ofh, **fields)
    status(ofh, ofh.lib().ofh_rotary_fwd(ctypes.addressof(p), ALIGNED, 2 * ALIGNED, None), code, text)


def test_rotary_pointers(ofh):
    L = ofh.lib()
    p = rotary(ofh)
    status(ofh, L.ofh_rotary_fwd(None, ALIGNED, ALIGNED, None), 1, "params must be non-null")
    status(ofh, L.ofh_rotary_fwd(ctypes.addressof(p), None, ALIGNED, None), 1, "must be non-null")
    status(ofh, L.ofh_rotary_fwd(ctypes.addressof(p), ALIGNED, None, None), 1, "must be non-null")
    status(ofh, L.ofh_rotary_fwd(ctypes.addressof(p), ALIGNED + 1, ALIGNED, None), 2, "aligned to their elements")
    p = rotary(ofh, x_strides=(960, 64, 192))
    status(ofh, L.ofh_rotary_fwd(ctypes.addressof(p), ALIGNED, ALIGNED, None), 1, "in place must keep its strides")


@pytest.mark.parametrize("fields,code,text", TURNS + [
    (dict(cache__struct_size=8), 1, "struct_size mismatch"),
    (dict(cache__batch=0), 1, "cache dimensions must be non-zero"),
    (dict(cache__tokens=0), 1, "cache dimensions must be non-zero"),
    (dict(cache__dtype=7), 1, "unknown dtype"),
    (dict(cache__head_dim=1026), 2, "head_dim must be at most 1024"),
    (dict(cache__page_size=24), 2, "page_size must be a power of two"),
    (dict(cache__page_table=None), 1, "page_table and lengths must be non-null"),
    (dict(cache__lengths=None), 1, "page_table and lengths must be non-null"),
    (dict(cache__k_page_strides=(1, -1, 1)), 1, "strides must be non-negative"),
    (dict(heads=1 << 31), 2, "32-bit index range"),
    (dict(heads=1 << 30), 2, "launch range"),
    (dict(q_strides=(64, -64, 64)), 1, "strides must be non-negative"),
])
def test_append_refusals(ofh, fields, code, text):
    p = append(ofh, **fields)
    A = ALIGNED
    status(ofh, ofh.lib().ofh_cache_append(ctypes.addressof(p), A, A, A, A, A, 2 * A, None), code, text)


def test_append_pointers(ofh):
    L, A = ofh.lib(), ALIGNED
    p = append(ofh)
    status(ofh, L.ofh_cache_append(None, A, A, A, A, A, A, None), 1, "params must be non-null")
    for i in range(6):
        args = [A] * 6
        args[i] = None
        status(ofh, L.ofh_cache_append(ctypes.addressof(p), *args, None), 1, "must be non-null")
        args[i] = A + 1
        status(ofh, L.ofh_cache_append(ctypes.addressof(p), *args, None), 2, "aligned to their elements")
    p = append(ofh, q_strides=(960, 64, 192))
    status(ofh, L.ofh_cache_append(ctypes.addressof(p), A, A, A, A, A, A, None), 1, "in place must keep its strides")


def test_frequencies(ofh):
    f = ofh.rotary_frequencies
    for part in (2, 6, 64, 128):
        assert f(part) == pytest.approx(rotary_ref.frequencies(part), rel=1e-15)
        assert f(part, base=5e5) == pytest.approx(rotary_ref.frequencies(part, 5e5), rel=1e-15)
        assert f(part, scaling={"type": "linear", "factor": 4}) == pytest.approx([x / 4 for x in f(part)], rel=1e-15)
        got = f(part, scaling={"type": "parts", "factor": 8, "original_tokens": 4096})
        assert got == pytest.approx(rotary_ref.parts(part, 8, 4096), rel=1e-14)
        got = f(part, base=5e5, scaling={"type": "parts", "factor": 8, "original_tokens": 8192, "low": 1, "high": 4})
        assert got == pytest.approx(rotary_ref.parts(part, 8, 8192, 1, 4, 5e5), rel=1e-14)
    # the fastest pair keeps its frequency, the slowest is divided by the factor
    plain, stretched = f(64), f(64, scaling={"type": "base", "factor": 4})
    assert stretched[0] == plain[0] and stretched[-1] == pytest.approx(plain[-1] / 4, rel=1e-13)


@pytest.mark.parametrize("args,kwargs", [
    ((0,), {}), ((7,), {}), ((-2,), {}), ((8.0,), {}), ((8,), dict(base=0.0)), ((8,), dict(base=float("inf"))),
    ((8,), dict(scaling={})), ((8,), dict(scaling={"type": "other", "factor": 2})),
    ((8,), dict(scaling={"type": "linear"})), ((8,), dict(scaling={"type": "linear", "factor": 0})),
    ((8,), dict(scaling={"type": "linear", "factor": 2, "low": 1})),
    ((2,), dict(scaling={"type": "base", "factor": 2})),
    ((8,), dict(scaling={"type": "parts", "factor": 2})),
    ((8,), dict(scaling={"type": "parts", "factor": 2, "original_tokens": 0})),
    ((8,), dict(scaling={"type": "parts", "factor": 2, "original_tokens": 10, "low": 4, "high": 4})),
])
def test_frequency_refusals(ofh, args, kwargs):
    with pytest.raises(ValueError):
        ofh.rotary_frequencies(*args, **kwargs)


@pytest.mark.parametrize("args,kwargs", [
    ((0,), {}), ((64.0,), {}), ((64,), dict(rotary_dim=65)), ((64,), dict(rotary_dim=66)), ((64,), dict(rotary_dim=0)),
    ((64,), dict(magnitude=float("nan"))), ((64,), dict(frequencies=[1.0] * 31)),
    ((4,), dict(frequencies=[1.0, float("inf")])), ((4,), dict(frequencies=[1.0, 2.0], scaling={"type": "linear", "factor": 2})),
    ((64,), dict(device="cpu")),
])
def test_rotary_constructor_refusals(ofh, args, kwargs):
    with pytest.raises(ValueError):
        ofh.Rotary(*args, **kwargs)
