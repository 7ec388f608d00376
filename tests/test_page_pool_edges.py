"""Numbers that the page pool's C interface has no place for."""

from __future__ import annotations

import pytest

import onednn_flash_cache as C
import onednn_flash_hip as F

WRAP = 1 << 64


def test_numbers_past_64_bits_are_refused():
    """Taken modulo 2^64 they would name another sequence, drop its tokens or make
    room for none."""
    pool = C.PagePool(8, 4)
    a = pool.add()
    pool.extend([a], [6])
    for call in (lambda: pool.length(WRAP + a), lambda: pool.extend([a], [WRAP]), lambda: pool.extend([a], [WRAP + 1]),
                 lambda: pool.extend([WRAP + a], [1]), lambda: pool.truncate(a, WRAP), lambda: pool.truncate(a, WRAP + 2),
                 lambda: pool.truncate(WRAP + a, 0), lambda: pool.fork(WRAP + a), lambda: pool.free(WRAP + a),
                 lambda: pool.free(a - WRAP), lambda: pool.table([WRAP + a], 2), lambda: pool.table([], WRAP + 1),
                 lambda: C.PagePool(WRAP + 4, 4), lambda: C.PagePool(4, WRAP + 4)):
        with pytest.raises(ValueError, match="out of range"):
            call()
        assert (pool.length(a), pool.pages_in_use) == (6, 2)


def test_a_table_has_no_negative_width():
    pool = C.PagePool(8, 4)
    a = pool.add()
    for width in (-1, -(1 << 40), -WRAP):
        for sequences in ([a], [], [a, a]):
            with pytest.raises(ValueError, match="max_pages must be non-negative"):
                pool.table(sequences, width)
    assert pool.table([a], 0) == ([[]], [0])
    pool.extend([a], [1])
    with pytest.raises(F.OfhError, match="holds 1 pages, a row 0"):
        pool.table([a], 0)


def test_integers_of_other_kinds_are_numbers():
    import numpy as np
    import torch
    pool = C.PagePool(8, 4)
    a = np.int64(pool.add())
    pool.extend([a], [np.int32(3)])
    pool.extend([torch.tensor(int(a))], torch.tensor([2]))
    pool.truncate(a, np.int64(4))
    assert pool.length(a) == 4 and pool.table([a], 2)[1] == [4]
