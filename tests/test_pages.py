"""ftb.PagePool's account, on the CPU with a fake of the copies."""
import random

import pytest
import torch

import ftb
from ftb import pages


@pytest.fixture
def copied(monkeypatch):
    calls = []
    monkeypatch.setattr(pages, "copy_pages", lambda caches, src, dst: calls.append((src, dst)))
    return calls


def test_allocate_and_free():
    pool = ftb.PagePool(4, 16)
    a, b = pool.allocate(3), pool.allocate(1)
    assert a == [0, 1, 2] and b == [3] and pool.free_pages == 0
    with pytest.raises(MemoryError):
        pool.allocate(1)
    pool.free(a)
    assert a == [] and pool.free_pages == 3 and pool.allocate(2) == [0, 1]
    assert pool.allocate(0) == []


def test_fork_and_extend(copied):
    pool = ftb.PagePool(8, 4)
    a = []
    assert pool.extend([a], [0], [10]) == 0 and a == [0, 1, 2]
    b = pool.fork(a)
    assert b == a and b is not a and pool.holders(0) == 2 and pool.free_pages == 5
    assert pool.extend([a], [10], [0]) == 0 and copied == []  # no new token
    assert pool.extend([a, b], [10, 10], [1, 3]) == 1
    # a page is copied once: the last holder keeps it
    assert copied == [([2], [3])] and a == [0, 1, 3] and b == [0, 1, 2, 4]
    assert [pool.holders(i) for i in range(5)] == [2, 2, 1, 1, 1]
    pool.free(a)
    assert [pool.holders(i) for i in range(5)] == [1, 1, 1, 0, 1]


def test_a_shared_page_without_older_tokens_is_not_copied(copied):
    pool = ftb.PagePool(8, 4)
    a = pool.allocate(3)  # room for 12, none written behind 8
    b = pool.fork(a)
    assert pool.extend([b], [8], [2]) == 0 and copied == []
    assert b == [0, 1, 3] and pool.holders(2) == 1


def test_extend_without_room_changes_nothing(copied):
    pool = ftb.PagePool(4, 4)
    a = pool.allocate(3)
    b = pool.fork(a)
    with pytest.raises(MemoryError):
        pool.extend([a, b], [10, 10], [1, 3])  # a copy and a page: one is free
    assert a == b == [0, 1, 2] and [pool.holders(i) for i in range(4)] == [2, 2, 2, 0]
    assert copied == [] and pool.free_pages == 1


def test_compact(copied):
    pool = ftb.PagePool(10, 4)
    a, b, c = pool.allocate(3), pool.allocate(3), pool.allocate(2)
    d = pool.fork(c)
    pool.free(a)
    assert pool.compact([b, c, d]) == 3
    used = sorted(set(b + c))
    assert used == list(range(5)) and c == d and pool.free_pages == 5
    (src, dst), = copied
    assert not set(src) & set(dst) and all(s >= 5 > t for s, t in zip(src, dst))
    assert pool.compact([b, c, d]) == 0 and len(copied) == 1
    assert pool.allocate(5) == [5, 6, 7, 8, 9]


def test_refusals(copied):
    pool = ftb.PagePool(4, 16)
    a = pool.allocate(2)
    for call in (lambda: pool.free([3]), lambda: pool.free([0, 0]), lambda: pool.fork([2]),
                 lambda: pool.fork([9]), lambda: pool.allocate(-1), lambda: pool.compact([]),
                 lambda: pool.compact([a, list(a)]), lambda: pool.compact([a, a]),
                 lambda: pool.extend([a], [33], [1]), lambda: pool.extend([a], [-1], [1]),
                 lambda: pool.extend([a], [0], [-1]), lambda: pool.extend([a, a], [0, 0], [1, 1]),
                 lambda: pool.extend([a], [0, 1], [1]), lambda: ftb.PagePool(-1, 16),
                 lambda: ftb.PagePool(4, 0), lambda: ftb.PagePool(4, 16, [torch.zeros(3, 1)])):
        with pytest.raises(ValueError):
            call()
    assert a == [0, 1] and pool.free_pages == 2


@pytest.mark.parametrize("seed", range(20))
def test_sequences_keep_their_tokens(monkeypatch, seed):
    """Random forks, extensions, frees and compactions against a record of each sequence's tokens."""
    rng = random.Random(seed)
    page, count = rng.choice([1, 4, 16]), 60
    memory = [[None] * page for _ in range(count)]

    def move(caches, src, dst):
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for s, d in zip(src, dst):
            memory[d] = list(memory[s])

    monkeypatch.setattr(pages, "copy_pages", move)
    pool, seqs, serial = ftb.PagePool(count, page), [], 0
    for _ in range(300):
        act = rng.random()
        if act < 0.15:
            seqs.append(([], []))
        elif act < 0.3 and seqs:
            ids, tokens = rng.choice(seqs)
            seqs.append((pool.fork(ids), list(tokens)))
        elif act < 0.45 and seqs:
            pool.free(seqs.pop(rng.randrange(len(seqs)))[0])
        elif act < 0.5:
            pool.compact([ids for ids, _ in seqs])
            assert {i for ids, _ in seqs for i in ids} == set(range(count - pool.free_pages))
        elif seqs:
            some = rng.sample(seqs, rng.randint(1, len(seqs)))
            new = [rng.randint(0, 2 * page) for _ in some]
            try:
                pool.extend([s[0] for s in some], [len(s[1]) for s in some], new)
            except MemoryError:
                continue
            for (ids, tokens), n in zip(some, new):
                for _ in range(n):
                    memory[ids[len(tokens) // page]][len(tokens) % page] = serial
                    tokens.append(serial)
                    serial += 1
        for ids, tokens in seqs:
            assert [memory[ids[i // page]][i % page] for i in range(len(tokens))] == tokens
        assert sum(bool(pool.holders(i)) for i in range(count)) == count - pool.free_pages
