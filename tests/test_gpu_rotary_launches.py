"""Turned writes of very many pages times heads: to both sides of where they go by rows, and at the largest launch. Values are those
of Rotary.rotate and of a plain write, bit for bit."""

import numpy as np
import pytest

import serving

pytestmark = pytest.mark.gpu
LIMIT = 0xffffff // 4  # workgroups of 512 for the pages, and as many for the queries: together under 2^32 threads


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


def same(a, b):
    import torch
    return torch.equal(a.contiguous().view(torch.int32), b.contiguous().view(torch.int32))


def page_workgroups(rows, sequences, kv_heads):
    assert rows > 16 * sequences and rows * kv_heads > 2048  # (fewer go by rows)
    return (rows // 64 + 2 * sequences) * kv_heads * 2


@pytest.mark.parametrize("sequences,by_pages", [(225, True), (226, False)])
@pytest.mark.parametrize("dims", [4, 2])
def test_pages_times_heads_around_the_limit(fk, gpu, sequences, by_pages, dims):
    import torch
    rows, kv_heads = 17 * sequences, 4096
    assert (page_workgroups(rows, sequences, kv_heads) <= LIMIT) == by_pages
    rng = np.random.default_rng(sequences)
    step = serving.Step([17] * sequences, [17 + int(p) for p in rng.integers(0, 60, sequences)])
    rotary, batch = fk.Rotary(dims, layout="pairs"), step.batch(fk, gpu)
    g = torch.Generator(device=gpu).manual_seed(dims)
    k, v = (torch.randn(rows, kv_heads, 4, device=gpu, generator=g) for _ in range(2))
    q = torch.randn(rows, 3, 4, device=gpu, generator=g)
    cache = fk.PagedCache(step.pages, kv_heads, 4, device=gpu)
    turned = cache.write(batch, k, v, rotary=rotary, queries=q)
    assert same(turned, rotary.rotate(batch, q))
    plain = fk.PagedCache(step.pages, kv_heads, 4, device=gpu)
    plain.write(batch, rotary.rotate(batch, k), v)
    read = [torch.empty_like(k) for _ in range(4)]
    cache.read(batch, *read[:2])
    plain.read(batch, *read[2:])
    assert torch.equal(read[0], read[2]) and torch.equal(read[1], read[3])


def test_the_largest_launch(fk, gpu):
    """Pages near the limit and queries past theirs, which go round: 8.27 million workgroups of 512."""
    import torch
    sequences, kv_heads, heads = 2000, 450, 65536
    rows = 17 * sequences
    assert LIMIT * 31 // 32 < page_workgroups(rows, sequences, kv_heads) <= LIMIT
    assert rows * (heads // 64) > 8 * LIMIT  # a wave has 64 heads of four values
    rng = np.random.default_rng(0)
    step = serving.Step([17] * sequences, [17 + int(p) for p in rng.integers(0, 60, sequences)])
    rotary, batch = fk.Rotary(2), step.batch(fk, gpu)
    g = torch.Generator(device=gpu).manual_seed(0)
    k, v = (torch.randn(rows, kv_heads, 4, device=gpu, generator=g) for _ in range(2))
    q = torch.randn(1, heads, 4, device=gpu, generator=g).expand(rows, heads, 4)
    out = torch.full((rows, heads, 4), float("nan"), device=gpu)  # 36 GB
    cache, plain = (fk.PagedCache(step.pages, kv_heads, 4, device=gpu) for _ in range(2))
    cache.write(batch, k, v, rotary=rotary, queries=q, out=out)
    for first in (0, 30000, heads - 1000):
        part = q[:1, first:first + 1000].contiguous().expand(rows, 1000, 4)
        assert same(out[:, first:first + 1000], rotary.rotate(batch, part))
    assert not any(bool(torch.isnan(out[r:r + 1000]).any()) for r in range(0, rows, 1000))
    plain.write(batch, rotary.rotate(batch, k), v)
    read = [torch.empty_like(k) for _ in range(4)]
    cache.read(batch, *read[:2])
    plain.read(batch, *read[2:])
    assert torch.equal(read[0], read[2]) and torch.equal(read[1], read[3])
