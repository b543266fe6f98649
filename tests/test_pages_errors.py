"""Errors of ftb.PagePool and ftb.copy_pages come before anything is changed. On the CPU, with fakes of the
copies and of the launch."""
import pytest
import torch

import ftb
from ftb import pages


def account(pool, *lists):
    return [list(x) for x in lists], [pool.holders(i) for i in range(pool.num_pages)], pool.free_pages


@pytest.mark.parametrize("error", [ValueError, RuntimeError, MemoryError, KeyboardInterrupt])
def test_an_extension_whose_copies_fail_changes_nothing(monkeypatch, error):
    def fail(caches, src, dst):
        raise error("no copy")

    pool = ftb.PagePool(9, 4)
    a = pool.allocate(3)
    b, c = pool.fork(a), pool.allocate(1)
    before = account(pool, a, b, c)
    monkeypatch.setattr(pages, "copy_pages", fail)
    with pytest.raises(error):
        pool.extend([a, c, b], [10, 4, 9], [1, 9, 5])  # a copy for a, new pages for b and c
    assert account(pool, a, b, c) == before
    copied = []
    monkeypatch.setattr(pages, "copy_pages", lambda caches, src, dst: copied.append((src, dst)))
    assert pool.extend([a, c, b], [10, 4, 9], [1, 9, 5]) == 1
    assert (a, c, b) == ([0, 1, 4], [3, 5, 6, 7], [0, 1, 2, 8]) and copied == [([2], [4])]
    assert account(pool)[1:] == ([2, 2] + [1] * 7, 0)


def test_an_extension_of_caches_that_cannot_be_copied_changes_nothing():
    """(tensors on the CPU: copy_pages refuses them)"""
    pool = ftb.PagePool(6, 4, [torch.zeros(6, 4)])
    a = pool.allocate(2)
    b = pool.fork(a)
    before = account(pool, a, b)
    with pytest.raises(ValueError, match="CUDA"):
        pool.extend([b], [6], [1])
    assert account(pool, a, b) == before


@pytest.fixture
def launched(monkeypatch):
    """Calls of the entry point, which copy nothing: the caches of each."""
    calls = []

    def call(entry, template, offsets, stream, *tensors):
        calls.append(len(tensors) - 2)
        return 0

    monkeypatch.setattr(pages, "require_cuda", lambda *t: t[0].device)
    monkeypatch.setattr(pages, "stream_handle", lambda device: 0)
    monkeypatch.setattr(pages, "caller", lambda device: call)
    monkeypatch.setattr(pages, "_ARGS", {})
    monkeypatch.setattr(pages, "remember", lambda key, args, *extra: pages._ARGS.setdefault(
        key, (bytes(args), *extra)))
    return calls


def test_caches_of_several_launches_are_checked_before_the_first(launched):
    """Whether or not a part of the caches is known from a call of its own."""
    many, fewer = [torch.zeros(6, 4) for _ in range(24)], [torch.zeros(5, 4) for _ in range(24)]
    bad = [torch.zeros(6, 4) for _ in range(3)] + [torch.zeros(6, 4, 4)[:, :, :2]]
    for caches in (many + fewer, many + bad, many + [torch.zeros(6, 4), torch.tensor(1.0)]):
        with pytest.raises(ValueError):
            ftb.copy_pages(caches, [0], [1])
    assert launched == []
    ftb.copy_pages(fewer, [0], [1])
    ftb.copy_pages(many, [0], [1])
    with pytest.raises(ValueError, match="6 pages"):
        ftb.copy_pages(many + fewer, [0], [1])
    assert launched == [24, 24]
    ftb.copy_pages(many + many[:5], [0], [1])
    assert launched == [24, 24, 24, 5]


def test_a_cache_without_a_dimension(launched):
    with pytest.raises(ValueError):
        ftb.copy_pages([torch.tensor(1.0)], [0], [1])
    assert launched == []
