"""The paged cache's levels and scales: what is written comes back as the 8-bit values it stands for,
bit for bit (level * scale in f32), and nothing else changes."""

import numpy as np
import pytest

import serving

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


def rows_of(step, heads, dim, seed, scale=1.0):
    import torch
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(step.total(), heads, dim, generator=g) * scale
    return x * torch.where(torch.rand(heads, dim, generator=g) < 0.05, 9.0, 1.0)


def same(a, b):
    import torch
    return torch.equal(a.cpu().view(torch.int32), b.cpu().float().view(torch.int32))


def stored(fk, cache, step, heads, dim, device, fill=float("nan")):
    import torch
    keys, values = (torch.full((step.total(), heads, dim), fill, device=device) for _ in range(2))
    cache.read(step.batch(fk, device), keys, values)
    return keys, values


# rows of the sequences, their lengths; more than 2048 rows, and than 16 a sequence, take the page kernels, others the row kernels
STEPS = [([1], [1]), ([1, 1, 1], [64, 65, 130]), ([1, 0, 1, 0], [7, 0, 200, 3]), ([64], [64]), ([65, 3], [65, 130]),
         ([200, 0, 1, 130], [201, 5, 77, 130]), ([63], [127]), ([5, 6], [61, 64 + 3]),
         ([2050, 66, 0, 3], [2060, 200, 5, 3]), ([64 * 33], [64 * 33]), ([700, 1, 1400], [701, 64, 1463])]
HEADS = [(1, 4), (2, 64), (3, 36), (2, 128), (1, 132), (4, 72), (1, 256), (2, 192)]


@pytest.mark.parametrize("rows,lengths", STEPS)
@pytest.mark.parametrize("heads,dim", HEADS)
def test_written_tokens_come_back(fk, gpu, rows, lengths, heads, dim):
    import torch
    print(f"cache {rows} {lengths} {heads}x{dim}", flush=True)
    step = serving.Step(rows, lengths, seed=dim, padding=2)
    whole = step.whole()
    cache = fk.PagedCache(step.pages, heads, dim, device=gpu)
    old_k, old_v = rows_of(whole, heads, dim, 1), rows_of(whole, heads, dim, 2, 0.01)
    cache.write(whole.batch(fk, gpu), old_k.to(gpu), old_v.to(gpu))
    k, v = rows_of(step, heads, dim, 3), rows_of(step, heads, dim, 4, 100.0)
    cache.write(step.batch(fk, gpu), k.to(gpu), v.to(gpu))
    got_k, got_v = stored(fk, cache, step, heads, dim, gpu)
    n = int(step.starts[-1])
    assert same(got_k[:n], serving.quantized(k[:n])) and same(got_v[:n], serving.quantized(v[:n]))
    assert bool(torch.isnan(got_k[n:]).all()) and bool(torch.isnan(got_v[n:]).all())  # the padding's rows
    # every other token as before
    all_k, all_v = stored(fk, cache, whole, heads, dim, gpu)
    for want, new, got in ((old_k.clone(), k, all_k), (old_v.clone(), v, all_v)):
        for s, (r, length) in enumerate(zip(rows, lengths)):
            end = int(whole.starts[s + 1])
            want[end - r:end] = new[int(step.starts[s]):int(step.starts[s + 1])]
        assert same(got, serving.quantized(want))


def test_special_values(fk, gpu):
    """Zero rows, subnormal ones, the largest, NaN beside numbers, infinity (its level 0 times an
    infinite scale is NaN), ties."""
    import torch
    dim = 32
    x = torch.zeros(9, 1, dim)
    x[1, 0, 3] = -0.0
    x[2, 0, :4] = torch.tensor([1e-45, -3e-45, 2e-44, 0.0])
    x[3, 0, :3] = torch.tensor([3.4e38, -3.4e38, 1e30])
    x[4, 0, :3] = torch.tensor([float("nan"), 2.0, -1.0])
    x[5] = float("nan")
    x[6, 0, :2] = torch.tensor([float("inf"), 1.0])
    x[7, 0, :6] = torch.tensor([127.0, 0.5, 1.5, -2.5, 63.5, -126.5])
    x[8, 0] = torch.linspace(-1e-20, 1e-20, dim)
    for rows, lengths in (([9], [9]), ([1] * 9, [1] * 9), ([9 * 240], [9 * 240])):
        if rows[0] > 9:
            x = x.repeat(240, 1, 1)  # the page kernels
        step = serving.Step(rows, lengths)
        cache = fk.PagedCache(step.pages, 1, dim, device=gpu)
        cache.write(step.batch(fk, gpu), x.to(gpu), x.to(gpu))
        for got in stored(fk, cache, step, 1, dim, gpu):
            want = serving.quantized(x).float()
            nan = torch.isnan(want)
            assert torch.equal(torch.isnan(got.cpu()), nan) and bool(nan[6::9].all()) and not bool(nan[5::9].any())
            assert torch.equal(got.cpu()[~nan], want[~nan])


@pytest.mark.parametrize("rows,lengths", [([70], [70]), ([1, 1], [3, 70]), ([1100], [1111])])
def test_strides_and_unaligned_rows(fk, gpu, rows, lengths):
    """Keys and values as slices of one projection's rows, at an address of any float; one row for all."""
    import torch
    step = serving.Step(rows, lengths)
    heads, dim, n = 2, 36, sum(rows)
    flat = torch.randn(n * 151 + 7, generator=torch.Generator().manual_seed(5)).to(gpu)
    k = flat[1:].as_strided((n, heads, dim), (151, dim, 1))
    v = flat[1:].as_strided((n, heads, dim), (151, dim, 1), 1 + 75)
    cache = fk.PagedCache(step.pages, heads, dim, device=gpu)
    cache.write(step.batch(fk, gpu), k, v)
    room = torch.full((n * 200 + 3,), 7.0, device=gpu)
    got_k = room.as_strided((n, heads, dim), (200, dim, 1), 3)
    got_v = room.as_strided((n, heads, dim), (200, dim, 1), 3 + 80)
    cache.read(step.batch(fk, gpu), got_k, got_v)
    assert same(got_k.contiguous(), serving.quantized(k.cpu())) and same(got_v.contiguous(), serving.quantized(v.cpu()))
    assert int((room == 7.0).sum()) == room.numel() - 2 * n * heads * dim
    one = k[:1].expand(n, heads, dim)
    cache.write(step.batch(fk, gpu), one, one)
    got_k, got_v = stored(fk, cache, step, heads, dim, gpu)
    assert same(got_k, serving.quantized(one.cpu())) and same(got_v, got_k)


@pytest.mark.parametrize("rows,lengths", [([3, 2, 2], [2, 130, 5]), ([100, 70], [40, 200]), ([1200, 70], [1090, 200])])
def test_rows_without_a_place(fk, gpu, rows, lengths):
    """Rows before position 0, pages outside the cache and past the table: not written, read as 0."""
    import torch
    heads, dim = 2, 64
    step = serving.Step(rows, lengths, extra_columns=0)
    step.table[1, lengths[1] // 64 - 1] = step.pages  # one past the last page
    step.table[:, -1] = np.where(step.table[:, -1] < 0, -1, -7)
    x = rows_of(step, heads, dim, 9)
    cache = fk.PagedCache(step.pages, heads, dim, device=gpu)
    cache.write(step.batch(fk, gpu), x.to(gpu), -x.to(gpu))
    got_k, got_v = stored(fk, cache, step, heads, dim, gpu)
    want = serving.quantized(x)
    for s, (r, length) in enumerate(zip(rows, lengths)):
        for i in range(r):
            p = length - r + i
            held = 0 <= p and p // 64 < step.table.shape[1] and 0 <= step.table[s, p // 64] < step.pages
            if not held:
                want[int(step.starts[s]) + i] = 0
    assert same(got_k + 0.0, want + 0.0) and same(got_v + 0.0, 0.0 - want)


@pytest.mark.parametrize("rows,lengths", [([70, 1], [70, 200]), ([300, 1], [300, 200])])
def test_offsets_past_32_bits(fk, gpu, rows, lengths):
    import torch
    heads, dim = 8, 256
    step = serving.Step(rows, lengths, spare=0)
    step.pages = 17000  # 17000 pages of 8 x 33 KB: 4.5 GB
    step.table[step.table >= 0] += step.pages - 1 - step.table.max()
    x = rows_of(step, heads, dim, 1)
    cache = fk.PagedCache(step.pages, heads, dim, device=gpu)
    cache.write(step.batch(fk, gpu), x.to(gpu), -x.to(gpu))
    got_k, got_v = stored(fk, cache, step, heads, dim, gpu)
    assert same(got_k, serving.quantized(x)) and same(got_v, serving.quantized(-x))


def test_many_sequences(fk, gpu):
    """More sequences than a wave has lanes, many without rows."""
    rng = np.random.default_rng(3)
    for high, count in ((2, 4300), (40, 4300), (100, 300)):
        rows = [int(r) if rng.random() < 0.6 else 0 for r in rng.integers(0, high, count)]
        step = serving.Step(rows, [r + int(p) for r, p in zip(rows, rng.integers(0, 9, count))], padding=1)
        x = rows_of(step, 1, 32, 1)
        cache = fk.PagedCache(step.pages, 1, 32, device=gpu)
        cache.write(step.batch(fk, gpu), x.to(gpu), -x.to(gpu))
        got_k, got_v = stored(fk, cache, step, 1, 32, gpu)
        n = int(step.starts[-1])
        assert same(got_k[:n], serving.quantized(x[:n])) and same(got_v[:n], serving.quantized(-x[:n]))


def test_more_heads_than_a_launch_of_rows_takes(fk, gpu):
    """One token each of 16400 sequences, of 4096 heads: past 2^32 threads of a wave a head. Attention, which
    takes a workgroup a sequence and head, refuses them."""
    import torch
    heads, n = 4096, 16400
    cache = fk.PagedCache(1, heads, 4, device=gpu)
    pages = torch.full((n, 1), -1, dtype=torch.int32, device=gpu)
    pages[n - 2] = 0
    batch = fk.Batch(torch.arange(n + 1, dtype=torch.int32, device=gpu), torch.full((n,), 9, dtype=torch.int32, device=gpu), pages)
    keys = torch.randn(n, heads, 4, device=gpu)
    cache.write(batch, keys, -keys)
    want = serving.quantized(keys[n - 2].cpu())
    values, back = torch.full_like(keys, 3.0), torch.full_like(keys, 3.0)
    cache.read(batch, back, values)
    assert same(back[n - 2], want) and same(values[n - 2], -want + 0.0)
    back[n - 2] = values[n - 2] = 0
    assert not bool(back.any()) and not bool(values.any())
    with pytest.raises(fk.ShapeError, match="than a launch takes"):
        cache.attend(batch, keys)


def test_refusals(fk, gpu):
    import torch
    step = serving.Step([2], [2])
    batch = step.batch(fk, gpu)
    cache = fk.PagedCache(step.pages, 2, 64, device=gpu)
    good = torch.zeros(2, 2, 64, device=gpu)
    for bad in (good.cpu(), good.double(), good[:, :1], good.transpose(0, 2), good[..., ::2], good[0], good.transpose(0, 1)[:, ::2]):
        with pytest.raises(fk.ShapeError):
            cache.write(batch, bad, good)
        with pytest.raises(fk.ShapeError):
            cache.read(batch, good, bad)
    with pytest.raises(fk.ShapeError):
        cache.write(batch, good, good[:1])
    with pytest.raises(fk.ShapeError):
        cache.read(batch, good[:1].expand(2, 2, 64), good)
    starts, lengths, pages = batch.row_starts, batch.lengths, batch.pages
    for args in ((starts.long(), lengths, pages), (starts[:1], lengths, pages), (starts, lengths[:0], pages),
                 (starts, lengths, pages[0]), (starts, lengths, pages.cpu()), (starts, lengths, pages.repeat(1, 2)[:, ::2])):
        with pytest.raises(fk.ShapeError):
            fk.Batch(*args)
    for shape in ((4, 0, 64), (4, 2, 30), (4, 2, 512)):
        with pytest.raises(fk.ShapeError):
            fk.PagedCache(*shape, device=gpu)
    empty = fk.PagedCache(0, 2, 64, device=gpu)  # no pages: nothing is kept
    empty.write(batch, good + 1, good + 1)
    empty.read(batch, good, good)
    assert not bool(good.any())
