"""Fork and truncate of the host-side page allocator (no GPU): shared full
pages, the private partly filled page, copy on truncate, compaction of shared
pages, refusals that change nothing, and a random soak against a model that
keeps every stream's tokens."""
import ctypes as C

import numpy as np
import pytest


def test_fork_shares_full_pages_and_copies_the_last(pkg):
    p = pkg.Pager(16, 16, 4, 8)
    a = p.open()
    p.append(a, 40)                       # pages 0, 1, 2 (8 tokens in the last)
    b, copy = p.fork(a, 40)
    assert p.pages(b) == [0, 1, 3] and copy == (2, 3) and p.length(b) == 40
    c, copy = p.fork(a, 32)               # a page boundary: nothing to copy
    assert p.pages(c) == [0, 1] and copy is None
    d, copy = p.fork(b, 0)
    assert p.pages(d) == [] and copy is None
    assert p.free_pages() == 12 and p.check() == 0
    assert p.append(c, 1) == 1 and p.pages(c)[:2] == [0, 1]
    p.close(a)
    assert p.free_pages() == 12 and p.check() == 0     # page 2 came back, page 4 went to c
    p.close(b)
    p.close(c)
    p.close(d)
    assert p.free_pages() == 16 and p.check() == 0


def test_fork_refusals_change_nothing(pkg):
    p = pkg.Pager(3, 16, 2, 8)
    a = p.open()
    p.append(a, 40)
    for tokens, code in ((41, 1), (-1, 1), (40, 2)):   # more than held, negative, no free page for the copy
        with pytest.raises(pkg.QkvError) as ei:
            p.fork(a, tokens)
        assert ei.value.code == code
    with pytest.raises(pkg.QkvError):
        p.fork(1, 0)                                   # not open
    b, _ = p.fork(a, 32)
    with pytest.raises(pkg.QkvError) as ei:
        p.fork(a, 16)                                  # no slot left
    assert ei.value.code == 3
    assert p.length(a) == 40 and p.pages(b) == p.pages(a)[:2] and p.check() == 0


def test_truncate_frees_and_unshares(pkg):
    p = pkg.Pager(8, 16, 3, 8)
    a = p.open()
    p.append(a, 64)
    b, _ = p.fork(a, 64)
    assert p.truncate(b, 64) is None and p.free_pages() == 4
    # 40 tokens: page 3 is given up by b (a holds it), page 2 is shared and now partly filled
    copy = p.truncate(b, 40)
    assert copy == (p.pages(a)[2], p.pages(b)[2]) and copy[0] != copy[1]
    assert p.pages(b)[:2] == p.pages(a)[:2] and p.free_pages() == 3 and p.check() == 0
    assert p.truncate(a, 40) is None                   # a's page 2 is its own again
    assert p.free_pages() == 4 and p.check() == 0
    assert p.truncate(a, 0) is None and p.pages(a) == [] and p.check() == 0
    for s, tokens in ((b, 41), (b, -1), (2, 0)):
        with pytest.raises(pkg.QkvError) as ei:
            p.truncate(s, tokens)
        assert ei.value.code == 1


def test_truncate_without_a_free_page(pkg):
    p = pkg.Pager(4, 16, 3, 8)
    a = p.open()
    p.append(a, 48)
    b, _ = p.fork(a, 48)
    p.append(b, 1)                                     # the fourth page
    with pytest.raises(pkg.QkvError) as ei:
        p.truncate(a, 40)                              # needs a page of its own; frees none
    assert ei.value.code == 2 and p.length(a) == 48 and p.check() == 0
    copy = p.truncate(b, 40)                           # its fourth page serves as the copy
    assert copy == (p.pages(a)[2], p.pages(b)[2]) and p.free_pages() == 0 and p.check() == 0


def test_compaction_moves_a_shared_page_once(pkg):
    p = pkg.Pager(12, 16, 4, 8)
    low = p.open()
    p.append(low, 64)
    a = p.open()
    p.append(a, 64)
    b, _ = p.fork(a, 64)
    p.append(b, 5)
    p.close(low)
    before = {s: p.pages(s) for s in (a, b)}
    moves = dict(p.compact())
    assert len(moves) == len(set(moves.values())) and p.check() == 0
    for s in (a, b):
        assert [moves.get(q, q) for q in before[s]] == p.pages(s)
        assert all(q < 5 for q in p.pages(s))
    assert p.pages(a) == p.pages(b)[:4]


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_random_streams_keep_their_tokens(pkg, seed):
    """Pages hold numbered tokens here; every operation is replayed on lists."""
    rng = np.random.default_rng(seed)
    p = pkg.Pager(90, 16, 10, 20, seed=seed)
    mem = np.full((90, 16), -1, np.int64)
    want, serial = {}, 0

    def read(s):
        n = p.length(s)
        return mem[p.pages(s)].reshape(-1)[:n].tolist() if n else []

    for step in range(2500):
        op = rng.integers(0, 12)
        s = int(rng.choice(list(want))) if want else None
        try:
            if op == 0:
                want[p.open()] = []
            elif s is None:
                continue
            elif op == 1:
                p.close(s)
                del want[s]
            elif op < 6:
                k = int(rng.integers(0, 40))
                p.append(s, k)
                pages, n0 = p.pages(s), len(want[s])
                for t in range(n0, n0 + k):
                    mem[pages[t // 16], t % 16] = serial
                    want[s].append(serial)
                    serial += 1
            elif op < 8:
                t = int(rng.integers(0, len(want[s]) + 1))
                new, copy = p.fork(s, t)
                if copy:
                    mem[copy[1]] = mem[copy[0]]
                want[new] = want[s][:t]
            elif op < 11:
                t = int(rng.integers(0, len(want[s]) + 1))
                copy = p.truncate(s, t)
                if copy:
                    mem[copy[1]] = mem[copy[0]]
                want[s] = want[s][:t]
            else:
                old = mem.copy()
                for a, b in p.compact():
                    mem[b] = old[a]
        except pkg.QkvError as e:
            assert e.code in (2, 3)
        if step % 25 == 0:
            assert p.check() == 0
            assert all(read(x) == w for x, w in want.items())
    assert p.check() == 0 and all(read(x) == w for x, w in want.items())


def test_null_arguments(pkg):
    p = pkg.Pager(4, 16, 2, 4)
    s = p.open()
    n = C.c_int32()
    assert pkg.lib.qkv_pager_fork(None, s, 0, C.byref(n), C.byref(n), C.byref(n)) == 1
    assert pkg.lib.qkv_pager_fork(p.p, s, 0, None, C.byref(n), C.byref(n)) == 1
    assert pkg.lib.qkv_pager_fork(p.p, s, 0, C.byref(n), None, C.byref(n)) == 1
    assert pkg.lib.qkv_pager_truncate(p.p, s, 0, C.byref(n), None) == 1
    for name, args in (("qkv_stream_fork", (None, 0, 0, C.byref(n), None)), ("qkv_stream_truncate", (None, 0, 0, None)),
                       ("qkv_pool_view_get", (None, None)), ("qkv_pages_copy", (None, 0, None, None, None)),
                       ("qkv_tokens_move", (None, 0) + (None,) * 5 + (0, None, None)),
                       ("qkv_chunk_append", (None, 0, 0, None, None, None, None, 0, None, None, 0, None)),
                       ("qkv_chunk_attend", (None, 0, 0, None, None, None, 0, None, None, None, None))):
        assert getattr(pkg.lib, name)(*args) == 1, name
    assert p.check() == 0
