"""ftb.copy_pages and ftb.PagePool on the GPU: copies are the same bytes, and nothing else changes."""
import pytest
import torch

import ftb

pytestmark = pytest.mark.gpu


def caches(pages, shapes, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randint(0, 256, (pages, *s), generator=g, device="cuda", dtype=torch.uint8)
            for s in shapes]


def want(t, src, dst):
    out = t.clone()
    for s, d in zip(src, dst):
        if 0 <= s < len(t) and 0 <= d < len(t):
            out[d] = t[s]
    return out


@pytest.mark.parametrize("shape", [(1,), (3,), (4,), (16,), (30,), (32,), (64, 4), (20, 52), (16, 3, 80),
                                   (8191,), (8192,), (8208,), (16384,), (16400,), (65536,), (70001,),
                                   (64, 8, 128), (1 << 20,)])
@pytest.mark.parametrize("count", [1, 2, 33])
def test_page_sizes(shape, count):
    pages = 2 * count + 1
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(count)).tolist()
    src, dst = order[:count], order[-count:]
    a, b = caches(pages, [shape, (5,)])
    after = want(a, src, dst), want(b, src, dst)
    ftb.copy_pages([a, b], src, dst)
    assert torch.equal(a, after[0]) and torch.equal(b, after[1])


@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
def test_many_caches_of_different_types(id_type):
    """More than one launch holds; ids on the device, with pairs that copy nothing."""
    pages = 40
    shapes = [(16, 2, 64), (4,), (7,), (8192 * 3,)] * 20
    all_ = caches(pages, shapes)
    views = [t.view({0: torch.bfloat16, 1: torch.float32}.get(i % 4, torch.uint8)) for i, t in
             enumerate(all_)]
    src = [3, -1, 4, 40, 5, 6, 7, 8]
    dst = [20, 21, -1, 22, 41, 23, 7, 24]
    after = [want(t, src, dst) for t in all_]
    ids = [torch.tensor(x, dtype=id_type, device="cuda") for x in (src, dst)]
    ftb.copy_pages(views, *ids)
    assert all(torch.equal(a, b) for a, b in zip(all_, after))


def test_strides_and_layouts():
    pages = 12
    fused = caches(pages, [(2, 16, 2, 64)])[0]
    k, v = fused[:, 0], fused[:, 1]  # pages further apart than they are long
    heads_first = caches(pages, [(4, 32, 16)], 1)[0].transpose(1, 2)
    odd = caches(1, [(pages * 100 + 3,)], 2)[0][0][3:].view(pages, 100)  # unaligned
    src, dst = [0, 5, 9], [1, 2, 11]
    after = [want(t, src, dst) for t in (fused[:, 0], fused[:, 1], heads_first, odd)]
    ftb.copy_pages([k, v, heads_first, odd], src, dst)
    assert all(torch.equal(a, b) for a, b in zip((k, v, heads_first, odd), after))


def test_one_page_to_several():
    a = caches(9, [(300,)])[0]
    after = want(a, [4] * 5, [0, 1, 2, 3, 8])
    ftb.copy_pages([a], [4] * 5, [0, 1, 2, 3, 8])
    assert torch.equal(a, after)


def test_nothing_to_copy():
    a = caches(3, [(300,)])[0]
    before = a.clone()
    ftb.copy_pages([a], [], [])
    ftb.copy_pages([], [0], [1])
    ftb.copy_pages([a], torch.empty(0, dtype=torch.int64, device="cuda"),
                   torch.empty(0, dtype=torch.int64, device="cuda"))
    ftb.copy_pages([a[:, :0]], [0], [1])
    ftb.copy_pages([a], [1, -1], [1, 0])
    assert torch.equal(a, before)


def test_offsets_past_32_bits():
    page = 1 << 20
    a = torch.empty(4200, page, dtype=torch.uint8, device="cuda")
    a[4199], a[1] = 7, 9
    ftb.copy_pages([a], [4199, 1], [0, 4198])
    assert (a[0] == 7).all() and (a[4198] == 9).all()


def test_captured():
    a = caches(20, [(4096,), (32,)])
    src, dst = (torch.tensor(x, device="cuda") for x in ([1, 2, 3], [11, 12, 13]))
    ftb.copy_pages(a, src, dst)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ftb.copy_pages(a, src, dst)
    src.copy_(torch.tensor([4, -1, 5], device="cuda"))
    after = [want(t, [4, -1, 5], [11, 12, 13]) for t in a]
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(a, after))


def test_refusals():
    a = caches(4, [(8, 8)])[0]
    for bad in (([a], [0, 1], [2, 2]), ([a], [0, 2], [2, 3]), ([a], [0], [4]), ([a], [0], [1, 2]),
                ([a[:, :, :4]], [0], [1]), ([a, a[:3]], [0], [1]), ([a, a.cpu()], [0], [1]),
                ([a], torch.tensor([0.0], device="cuda"), torch.tensor([1.0], device="cuda")),
                ([a], torch.tensor([0]), torch.tensor([1])),
                ([a[:1].expand(4, 8, 8)], [0], [1])):
        with pytest.raises(ValueError):
            ftb.copy_pages(*bad)


def test_pool_moves_what_it_says():
    """Sequences forked, extended and compacted: each keeps its own tokens."""
    page, cache = 16, ftb.PagedKvCache(24, 16, 2, 32, dtype=torch.float8_e4m3fn)
    pool = ftb.PagePool(24, page, [cache])
    k = cache.k.view(torch.uint8)

    def write(ids, at, value):
        for i, v in zip(at, value):
            k[ids[i // page], i % page] = v
            cache.v_scale[ids[i // page], 0] = v

    def read(ids, n):
        return [k[ids[i // page], i % page, 0, 0].item() for i in range(n)]

    a = []
    pool.extend([a], [0], [20])
    write(a, range(20), range(1, 21))
    b, c = pool.fork(a), pool.fork(a)
    assert pool.extend([a, b, c], [20, 20, 20], [1, 15, 1]) == 2
    for ids, v in ((a, 100), (b, 101), (c, 102)):
        write(ids, [20], [v])
        assert read(ids, 21) == [*range(1, 21), v]
    assert a[0] == b[0] == c[0] and len({a[1], b[1], c[1]}) == 3
    pool.free(a)
    assert pool.compact([b, c]) > 0 and max(b + c) == 3
    assert read(b, 21) == [*range(1, 21), 101] and read(c, 21) == [*range(1, 21), 102]
    assert cache.v_scale[b[1], 0, 0].item() == 101
