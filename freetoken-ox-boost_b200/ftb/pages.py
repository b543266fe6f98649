"""Pages of a cache: copies of whole pages (``ftb_copy_pages`` in ``include/ftb.h``), and the host's
account of who holds which page.

  * ``copy_pages(caches, src, dst)``: page dst[i] of every cache becomes its page src[i];
  * ``PagePool``: allocating, sharing, extending (with a copy of a shared page before it is written),
    freeing and compacting the pages of sequences.
"""
from __future__ import annotations

import heapq
from collections import Counter

import torch

from . import _lib
from ._runtime import _ARGS, _pycall, caller, remember, require_cuda, stream_handle

_GROUP = 24  # caches of one launch (a call's signature holds that many of four dimensions)
_OFFSETS = tuple(_lib.PagesArgsStruct.caches.offset + 8 * i for i in range(_lib.FTB_PAGES_MAX))
_IDS = _lib.offsets(_lib.PagesArgsStruct, "src", "dst")


def _dense_page(t: torch.Tensor) -> bool:
    """Whether each page of [pages, ...] is one piece of memory, in any order of its dimensions."""
    run = 1
    for size, stride in sorted(zip(t.shape[1:], t.stride()[1:]), key=lambda d: d[1]):
        if size == 1:
            continue
        if stride != run:
            return False
        run *= size
    return True


def _copy_args(caches, src, dst):
    """The checks of a call, and its arguments without the pointers."""
    dev = require_cuda(*caches, src, dst)
    if src.dim() != 1 or src.shape != dst.shape or src.dtype != dst.dtype or src.dtype not in (
            torch.int32, torch.int64) or not src.is_contiguous() or not dst.is_contiguous():
        raise ValueError(f"src {tuple(src.shape)} {src.dtype}, dst {tuple(dst.shape)} {dst.dtype}: "
                         "expected contiguous int32 or int64 of one length")
    a = _lib.PagesArgsStruct(n=src.numel(), n_caches=len(caches), id64=src.dtype == torch.int64)
    for i, t in enumerate(caches):
        if t.dim() < 1 or t.shape[0] != caches[0].shape[0]:
            raise ValueError(f"cache {i}: {tuple(t.shape)} on {t.device}, expected the first one's "
                             f"{caches[0].shape[0] if caches[0].dim() else 0} pages in dimension 0")
        if not _dense_page(t):
            raise ValueError(f"cache {i}: a page of strides {t.stride()[1:]} and shape "
                             f"{tuple(t.shape[1:])} is not one piece of memory")
        size = t.element_size()
        a.page_bytes[i] = t[0].numel() * size if t.shape[0] else 0
        a.page_strides[i] = t.stride(0) * size if t.shape[0] > 1 else a.page_bytes[i]
        if a.page_strides[i] < a.page_bytes[i]:
            raise ValueError(f"cache {i}: pages {t.stride(0)} elements apart overlap")
    a.num_pages = caches[0].shape[0]
    return a


def _ids(x, name, num_pages, dev):
    """Page ids of a list, checked, as int32 on the device; a tensor as it is."""
    if isinstance(x, torch.Tensor):
        return x
    x = [int(i) for i in x]
    if any(i < -1 or i >= num_pages for i in x):
        raise ValueError(f"{name}: page ids outside the {num_pages} pages")
    return torch.tensor(x, dtype=torch.int32, device=dev)


def copy_pages(caches, src, dst) -> None:
    """Page ``dst[i]`` of every tensor of ``caches`` becomes its page ``src[i]``, on the current stream.

    ``caches``: tensors [pages, ...] of any dtypes that share their page ids, such as the keys, values
    and scales of every layer; a page is one piece of memory, its dimensions in any order. ``src``,
    ``dst``: int32 or int64 device tensors of one length, or lists of ids. A pair with an id outside
    the pages (-1: padding), or twice the same, copies nothing. The copies have no order: no page may be
    in ``dst`` twice, or in ``src`` and ``dst`` (lists are checked, tensors are not)."""
    if type(caches) is not list:
        caches = list(caches)
    if not caches:
        return
    if caches[0].dim() < 1:
        raise ValueError("cache 0 has no dimension of pages")
    if not isinstance(src, torch.Tensor) or not isinstance(dst, torch.Tensor):
        if not isinstance(src, torch.Tensor) and not isinstance(dst, torch.Tensor):
            src, dst = list(src), list(dst)
            to = [d for s, d in zip(src, dst) if s != d and s >= 0 and d >= 0]
            if len(src) != len(dst) or len(set(to)) != len(to) or set(to) & {
                    s for s, d in zip(src, dst) if s != d and d >= 0}:
                raise ValueError("src and dst differ in length, or a page is copied to twice, or copied "
                                 "both from and to")
        dev = require_cuda(caches[0])
        src = _ids(src, "src", caches[0].shape[0], dev)
        dst = _ids(dst, "dst", caches[0].shape[0], dev)
    step = _GROUP
    if len(caches) > step or sum(t.dim() for t in caches) > 4 * step:
        step = min(step, max(1, 120 // (1 + max(t.dim() for t in caches))))
    groups = []  # (all checked before the first launch)
    for at in range(0, len(caches), step):
        group = caches if len(caches) <= step else caches[at:at + step]
        if at and group[0].shape[:1] != caches[0].shape[:1]:
            raise ValueError(f"cache {at}: shape {tuple(group[0].shape)}, expected "
                             f"{caches[0].shape[0]} pages in dimension 0")
        key = _pycall.key(src, dst, *group)
        known = _ARGS.get(key)
        if known is None:
            known = remember(key, _copy_args(group, src, dst), _OFFSETS[:len(group)] + _IDS)
        groups.append((group, known))
    for group, known in groups:
        dev = group[0].device
        st = caller(dev)(_lib.entry("ftb_copy_pages"), known[0], known[1], stream_handle(dev), *group,
                         src, dst)
        if st:
            _lib.check("ftb_copy_pages", st)


class PagePool:
    """Which pages are held, and by how many sequences. ``caches``: tensors [pages, ...], or objects
    with ``tensors()`` (:class:`~ftb.PagedKvCache`), whose pages the ids name; copies go to the current
    stream. A sequence's pages are a list of ids, as :meth:`~ftb.AttnStep.build` takes them."""

    def __init__(self, num_pages: int, page: int, caches=()):
        if num_pages < 0 or page < 1:
            raise ValueError(f"num_pages={num_pages}, page={page}")
        self.num_pages, self.page = num_pages, page
        self.caches = [t for c in caches for t in ([c] if isinstance(c, torch.Tensor) else c.tensors())]
        for t in self.caches:
            if t.shape[0] != num_pages:
                raise ValueError(f"a cache of {t.shape[0]} pages, expected {num_pages}")
        self._held = [0] * num_pages  # by how many lists
        self._free = list(range(num_pages))  # a heap: the lowest ids go first

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def holders(self, page_id: int) -> int:
        """How many lists hold a page."""
        return self._held[page_id]

    def allocate(self, count: int) -> list:
        """``count`` pages that nobody holds; a MemoryError (and no page) where there are fewer."""
        if count < 0:
            raise ValueError(f"count={count}")
        if count > len(self._free):
            raise MemoryError(f"{count} pages wanted, {len(self._free)} of {self.num_pages} free")
        ids = [heapq.heappop(self._free) for _ in range(count)]
        for i in ids:
            self._held[i] = 1
        return ids

    def _check(self, ids):
        if len(set(ids)) != len(ids):
            raise ValueError("a page twice in one list")
        if any(not 0 <= i < self.num_pages or not self._held[i] for i in ids):
            raise ValueError("a page that nobody holds")

    def fork(self, ids: list) -> list:
        """A second list of the same pages. Nothing is copied until one of them is extended."""
        self._check(ids)
        for i in ids:
            self._held[i] += 1
        return list(ids)

    def free(self, ids: list) -> None:
        """Gives a sequence's pages back, and empties the list. A page is free again when its last
        holder has."""
        self._check(ids)
        for i in ids:
            self._held[i] -= 1
            if not self._held[i]:
                heapq.heappush(self._free, i)
        ids.clear()

    def extend(self, pages: list, past: list, new: list) -> int:
        """Makes room for ``new[b]`` tokens behind the ``past[b]`` of sequence b, whose list ``pages[b]``
        is changed in place: pages are added, and a page that others hold too and that the new tokens
        reach is replaced by one of its own (a copy where older tokens are in it). All sequences'
        copies are one call; an error changes nothing. Returns how many pages were copied."""
        if not len(pages) == len(past) == len(new):
            raise ValueError(f"{len(pages)} page lists, {len(past)} pasts, {len(new)} counts")
        if len({id(ids) for ids in pages}) != len(pages):
            raise ValueError("the same list twice")
        held = {}  # what the lists before leave of a page's holders
        plan, want = [], 0
        for ids, p, n in zip(pages, past, new):
            self._check(ids)
            if p < 0 or n < 0 or p > len(ids) * self.page:
                raise ValueError(f"{p} + {n} tokens in {len(ids)} pages of {self.page}")
            last = -(-(p + n) // self.page) if n else 0
            for j in range(p // self.page, min(last, len(ids))):
                count = held.get(ids[j], self._held[ids[j]])
                if count > 1:
                    held[ids[j]] = count - 1
                    plan.append((ids, j, j * self.page < p))
                    want += 1
            want += max(0, last - len(ids))
        fresh = self.allocate(want)
        copies = [(ids[j], to) for (ids, j, copied), to in zip(plan, fresh) if copied]
        if copies:
            try:  # (before anything is changed)
                copy_pages(self.caches, [s for s, _ in copies], [d for _, d in copies])
            except BaseException:
                self.free(fresh)
                raise
        fresh.reverse()
        for ids, j, _ in plan:
            self._held[ids[j]] -= 1
            ids[j] = fresh.pop()
        for ids, p, n in zip(pages, past, new):
            last = -(-(p + n) // self.page) if n else 0
            ids += [fresh.pop() for _ in range(max(0, last - len(ids)))]
        return len(copies)

    def compact(self, pages: list) -> int:
        """Moves the pages in use to the lowest ids, and changes the lists of all sequences (``pages``:
        every list that holds pages) in place. Returns how many pages were moved."""
        if len({id(ids) for ids in pages}) != len(pages):
            raise ValueError("the same list twice")
        used = Counter(i for ids in pages for i in ids)
        if used != {i: n for i, n in enumerate(self._held) if n}:
            raise ValueError("pages: expected every list that holds pages")
        n = len(used)
        src = sorted(i for i in used if i >= n)
        dst = [i for i in range(n) if not self._held[i]]
        if src:
            copy_pages(self.caches, src, dst)
        to = dict(zip(src, dst))
        for s, d in to.items():
            self._held[d], self._held[s] = self._held[s], 0
        for ids in pages:
            ids[:] = [to.get(i, i) for i in ids]
        self._free = list(range(n, self.num_pages))
        return len(src)
