"""Pages of caches copied: what the copies hold, and that nothing else changes; forks and compactions of sequences that a
step then goes on with."""

import numpy as np
import pytest

import serving

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


def filled(fk, gpu, pages, heads, dim, seed):
    """A cache and a batch that reads all of it, in the order of its pages."""
    import torch
    cache = fk.PagedCache(pages, heads, dim, device=gpu)
    n = 64 * pages
    batch = fk.Batch(torch.tensor([0, n], dtype=torch.int32, device=gpu), torch.tensor([n], dtype=torch.int32, device=gpu),
                     torch.arange(pages, dtype=torch.int32, device=gpu).view(1, -1))
    g = torch.Generator().manual_seed(seed)
    cache.write(batch, torch.randn(n, heads, dim, generator=g).to(gpu), torch.randn(n, heads, dim, generator=g).to(gpu))
    return cache, batch


def contents(cache, batch):
    import torch
    n = 64 * cache.pages
    out = [torch.zeros(n, cache.kv_heads, cache.head_dim, device=cache.device) for _ in range(2)]
    cache.read(batch, *out)
    return [x.cpu().view(cache.pages, 64, cache.kv_heads, cache.head_dim) for x in out]


# heads of every padding, layers of different shapes, more of them than a launch takes
SHAPES = [[(1, 4)], [(2, 64)] * 3, [(4, 128), (4, 128), (1, 36), (3, 256), (4, 128)], [(5, 72)], [(2, 192)], [(1, 32)] * 130]


@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("count", [0, 1, 7, 30])
def test_copies(fk, gpu, shapes, count):
    import torch
    print(f"copy {len(shapes)} caches {shapes[0]} {count} pages", flush=True)
    pages = 64
    layers = [filled(fk, gpu, pages + i % 2, h, d, i) for i, (h, d) in enumerate(shapes)]
    before = [contents(*layer) for layer in layers]
    ids = np.random.default_rng(count).permutation(pages)
    sources, targets = ids[:count], ids[count:2 * count]
    for as_lists in (False, True):
        s, t = sources.tolist(), targets.tolist()
        if not as_lists:
            s, t = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in (s, t))
        fk.copy_pages([c for c, _ in layers], s, t)
        for layer, old in zip(layers, before):
            for got, want in zip(contents(*layer), old):
                want = want.clone()
                want[targets] = want[sources]
                assert torch.equal(got, want)


@pytest.mark.parametrize("heads,dim", [(1849, 32), (977, 64), (513, 128), (257, 256)])
def test_many_heads(fk, gpu, heads, dim):
    """Pages of so many pieces that what is left after dividing a page among them is more than none."""
    import torch
    print(f"copy {heads} heads of {dim}", flush=True)
    cache, batch = filled(fk, gpu, 3, heads, dim, 0)
    old = contents(cache, batch)
    fk.copy_pages([cache], [0], [2])
    for got, want in zip(contents(cache, batch), old):
        want[2] = want[0]
        assert torch.equal(got, want)


def test_ids_outside_and_pages_onto_themselves(fk, gpu):
    """Pairs that name no page change nothing, in the cache whose page it is not; one source for several targets."""
    import torch
    small, large = filled(fk, gpu, 8, 2, 64, 0), filled(fk, gpu, 12, 2, 64, 1)
    old = [contents(*small), contents(*large)]
    big = 2 ** 31 - 1
    sources = torch.tensor([0, 0, -1, 1, 10, big, 2, 3, -big - 1], dtype=torch.int32, device=gpu)
    targets = torch.tensor([4, 5, 6, 9, 7, 6, -5, 3, 2], dtype=torch.int32, device=gpu)
    fk.copy_pages([small[0], large[0]], sources, targets)
    for layer, want, pairs in ((small, old[0], [(0, 4), (0, 5)]), (large, old[1], [(0, 4), (0, 5), (1, 9), (10, 7)])):
        for got, x in zip(contents(*layer), want):
            x = x.clone()
            for s, t in pairs:
                x[t] = x[s]
            assert torch.equal(got, x)


def test_offsets_past_32_bits(fk, gpu):
    import torch
    pages = 17000  # of 8 x 33 KB: 4.5 GB
    cache = fk.PagedCache(pages, 8, 256, device=gpu)
    batch = lambda p: fk.Batch(torch.tensor([0, 64], dtype=torch.int32, device=gpu), torch.tensor([64], dtype=torch.int32, device=gpu),
                               torch.tensor([[p]], dtype=torch.int32, device=gpu))
    x = torch.randn(64, 8, 256, generator=torch.Generator().manual_seed(0)).to(gpu)
    cache.write(batch(3), x, -x)
    fk.copy_pages([cache], [3], [pages - 1])
    fk.copy_pages([cache], [pages - 1], [pages - 2])
    got = [torch.zeros_like(x) for _ in range(4)]
    cache.read(batch(3), *got[:2])
    cache.read(batch(pages - 2), *got[2:])
    assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3]) and bool(got[2].any())


def test_replays_with_other_ids(fk, gpu):
    import torch
    cache, batch = filled(fk, gpu, 20, 2, 64, 0)
    sources, targets = torch.zeros(3, dtype=torch.int32, device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu)
    fk.copy_pages([cache], sources, targets)  # pages onto themselves
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fk.copy_pages([cache], sources, targets)
    rng = np.random.default_rng(0)
    for _ in range(5):
        old = contents(cache, batch)
        ids = rng.permutation(20)
        sources.copy_(torch.from_numpy(ids[:3].astype(np.int32)))
        targets.copy_(torch.from_numpy(ids[3:6].astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        for got, want in zip(contents(cache, batch), old):
            want[ids[3:6]] = want[ids[:3]]
            assert torch.equal(got, want)


def test_streams_and_refusals(fk, gpu):
    import ctypes

    import torch
    cache, batch = filled(fk, gpu, 4, 2, 64, 0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    fk.copy_pages([cache], [0], [1], stream=side)
    side.synchronize()
    x = contents(cache, batch)[0]
    assert torch.equal(x[0], x[1]) and not torch.equal(x[0], x[2])
    one = torch.tensor([1], dtype=torch.int32, device=gpu)
    for s, t in ((one, one.long()), (one, one.cpu()), (one, one.view(1, 1)), (one, torch.zeros(2, dtype=torch.int32, device=gpu)),
                 (one, [2]), (torch.zeros(4, dtype=torch.int32, device=gpu)[::2], torch.zeros(2, dtype=torch.int32, device=gpu))):
        with pytest.raises(fk.ShapeError):
            fk.copy_pages([cache], s, t)
    with pytest.raises(fk.ShapeError):
        fk.copy_pages([cache], [1], [2, 3])
    device = ctypes.cast(cache.handle, ctypes.POINTER(ctypes.c_int))
    device[0] = 1
    try:
        with pytest.raises(ValueError, match="a cache is on device 1"):
            fk.copy_pages([cache], one, one)
    finally:
        device[0] = 0
