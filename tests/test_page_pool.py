"""Host bookkeeping of the paged cache against a plain model: random calls on
both, the pool's invariants after each, and its refusals."""

from __future__ import annotations

import random
import threading

import pytest

import onednn_flash_cache as C
import onednn_flash_hip as F


class Model:
    """Sequences as rows of token ids, and what each page's places hold."""

    def __init__(self, pages, size):
        self.size, self.place = size, [[None] * size for _ in range(pages)]
        self.tokens, self.next = {}, 0

    def copy(self, src, dst):
        assert len(src) == len(dst) and not set(src) & set(dst) and len(set(dst)) == len(dst)
        read = [list(self.place[s]) for s in src]
        for d, r in zip(dst, read):
            self.place[d] = r

    def check(self, pool):
        """Every sequence finds its tokens where its table says."""
        used = set()
        for seq, tokens in self.tokens.items():
            need = -(-len(tokens) // self.size)
            rows, lengths = pool.table([seq], need + 2)
            row = rows[0]
            assert lengths == [len(tokens)] and pool.length(seq) == len(tokens)
            assert row[need:] == [-1, -1] and all(0 <= p < len(self.place) for p in row[:need])
            assert len(set(row[:need])) == need
            for i, t in enumerate(tokens):
                assert self.place[row[i // self.size]][i % self.size] == t
            used |= set(row[:need])
        assert pool.pages_in_use == len(used)

    def write(self, pool, seq, n):
        old = len(self.tokens[seq])
        self.tokens[seq] += [f"{seq}.{self.next + i}" for i in range(n)]
        self.next += n
        rows, _ = pool.table([seq], len(self.place))
        for i in range(old, old + n):
            self.place[rows[0][i // self.size]][i % self.size] = self.tokens[seq][i]


@pytest.mark.parametrize("size,pages,seed", [(1, 9, 0), (4, 25, 1), (16, 12, 2), (3, 40, 3)])
def test_random_calls_match_a_plain_model(size, pages, seed):
    rng = random.Random(seed)
    pool, model = C.PagePool(pages, size), Model(pages, size)
    for _ in range(400):
        seqs = list(model.tokens)
        op = rng.choice(["add", "extend", "extend", "extend", "fork", "truncate", "free", "compact"])
        if op == "add" and len(seqs) < 8:
            model.tokens[pool.add()] = []
        elif op == "extend" and seqs:
            some = rng.sample(seqs, rng.randint(1, len(seqs)))
            counts = [rng.choice([0, 1, 1, rng.randint(0, 2 * size)]) for _ in some]
            before = pool.pages_in_use
            try:
                src, dst = pool.extend(some, counts)
            except F.OfhError as e:
                assert e.code == F.OFH_ERROR_OUT_OF_PAGES and pool.pages_in_use == before
                model.check(pool)
                continue
            model.copy(src, dst)
            for s, n in zip(some, counts):
                model.write(pool, s, n)
        elif op == "fork" and seqs and len(seqs) < 8:
            s = rng.choice(seqs)
            child = pool.fork(s)
            assert child not in model.tokens
            model.tokens[child] = list(model.tokens[s])
        elif op == "truncate" and seqs:
            s = rng.choice(seqs)
            n = rng.randint(0, len(model.tokens[s]))
            pool.truncate(s, n)
            del model.tokens[s][n:]
        elif op == "free" and seqs:
            s = rng.choice(seqs)
            pool.free(s)
            del model.tokens[s]
        elif op == "compact":
            most = rng.choice([None, None, 0, 1, 3])
            before = pool.pages_in_use
            src, dst = pool.compact(most)
            assert most is None or len(src) <= most
            model.copy(src, dst)
            assert pool.pages_in_use == before
            if most is None:
                for s, t in model.tokens.items():
                    assert all(p < before for p in pool.table([s], pages)[0][0])
        model.check(pool)
    for s in list(model.tokens):
        pool.free(s)
    assert pool.pages_in_use == 0


def test_pages_are_shared_until_written():
    pool = C.PagePool(8, 4)
    a = pool.add()
    assert pool.extend([a], [6]) == ([], [])
    b, c = pool.fork(a), pool.fork(a)
    assert pool.pages_in_use == 2
    # three hold page 1; of the two that grow together, each leaves it to the one that does not
    src, dst = pool.extend([a, b], [1, 1])
    assert src == [1, 1] and dst == [2, 3]
    assert pool.table([a, b, c], 2)[0] == [[0, 2], [0, 3], [0, 1]]
    # the last holder writes in place
    assert pool.extend([c], [1]) == ([], [])
    # a full last page is not written: nothing to copy
    d = pool.fork(a)
    pool.truncate(d, 4)
    assert pool.extend([d], [1]) == ([], [])
    # a sequence cut inside a page that its parent filled takes a copy
    e = pool.fork(a)
    pool.truncate(e, 2)
    src, dst = pool.extend([e], [1])
    assert src == [0] and dst == [5] and pool.length(e) == 3


def test_nothing_is_taken_when_pages_run_out():
    pool = C.PagePool(3, 4)
    a, b = pool.add(), pool.add()
    pool.extend([a], [6])
    with pytest.raises(F.OfhError) as e:
        pool.extend([a, b], [3, 1])
    assert e.value.code == F.OFH_ERROR_OUT_OF_PAGES
    assert (pool.length(a), pool.length(b), pool.pages_in_use) == (6, 0, 2)
    pool.extend([a, b], [2, 4])
    assert pool.pages_in_use == 3


def test_refusals():
    for args in ((0, 4), (4, 0), (-1, 4), (True, 4), (2.0, 4)):
        with pytest.raises(ValueError):
            C.PagePool(*args)
    with pytest.raises(F.OfhError):
        C.PagePool(4, (1 << 30) + 1)
    pool = C.PagePool(4, 4)
    a = pool.add()
    for call in (lambda: pool.extend([a + 1], [1]), lambda: pool.extend([a, a], [1, 1]), lambda: pool.fork(7),
                 lambda: pool.free(7), lambda: pool.truncate(a, 1), lambda: pool.truncate(9, 0),
                 lambda: pool.table([5], 1), lambda: pool.length(-1), lambda: pool.extend([a], [(1 << 30) + 1])):
        with pytest.raises(F.OfhError) as e:
            call()
        assert e.value.code == F.OFH_ERROR_INVALID_ARGUMENT
    for bad in ([1], [-1], [1.5], [True]):
        with pytest.raises(ValueError):
            pool.extend([a] if bad != [1] else [a, a], bad)
    with pytest.raises(ValueError):
        pool.truncate(a, -1)
    pool.extend([a], [9])
    with pytest.raises(F.OfhError) as e:
        pool.table([a], 2)
    assert "holds 3 pages, a row 2" in str(e.value)
    pool.free(a)
    with pytest.raises(F.OfhError):
        pool.free(a)
    L = F.lib()
    assert L.ofh_page_pool_add(None, None) == F.OFH_ERROR_INVALID_ARGUMENT
    assert L.ofh_page_pool_info(None, None, None) == F.OFH_ERROR_INVALID_ARGUMENT
    assert L.ofh_page_pool_destroy(None) == F.OFH_SUCCESS


def test_calls_from_several_threads():
    pool = C.PagePool(64, 4)

    def work():
        for _ in range(200):
            s = pool.add()
            pool.extend([s], [8])
            f = pool.fork(s)
            pool.free(s)
            pool.free(f)

    threads = [threading.Thread(target=work) for _ in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert pool.pages_in_use == 0
