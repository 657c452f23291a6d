"""Forms of the serving kernels that other tests' sizes do not reach: the decode kernel's parts and their
join for every size of head, both sides of the routing between the two kernels, and sampling of more rows than one
batch of workgroups takes. The bounds are those of test_gpu_cache_attend.py and test_gpu_sample.py."""

import numpy as np
import pytest

import serving
import test_gpu_sample as sampling
from test_gpu_cache_attend import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


# heads of 4 are kept as 32, of 72 as 96, of 132 as 192
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 4), (3, 1, 32), (4, 2, 72), (6, 2, 96), (8, 2, 132), (8, 1, 192), (4, 2, 256)])
@pytest.mark.parametrize("rows,lengths", [([1, 3], [5000, 1500]), ([2, 0, 1], [1100, 7, 2049])])
@pytest.mark.parametrize("window", [0, 1200])
def test_parts_of_the_decode_kernel(fk, gpu, heads, kv_heads, dim, rows, lengths, window):
    """Tables of more than 16 pages and few tiles: parts, joined by a second launch; with a window some are empty."""
    import torch
    print(f"parts {heads}/{kv_heads}x{dim} {rows} {lengths} {window}", flush=True)
    case = Case(fk, gpu, rows, lengths, heads, kv_heads, dim, seed=dim, padding=1)
    got = case.run(window=window)
    case.check(got, window=window)
    assert torch.equal(got, case.run(window=window))


# pairs of a new token and a query head of one key head, a sequence: the decode kernel takes 96, or 64 of heads past 128
@pytest.mark.parametrize("pairs,dim", [(64, 192), (65, 192), (64, 256), (65, 256), (96, 64), (97, 64), (96, 128), (97, 128)])
def test_both_sides_of_the_routing(fk, gpu, pairs, dim):
    for rows, lengths in (([pairs], [1300]), ([pairs, pairs], [pairs, 200])):
        case = Case(fk, gpu, rows, lengths, 1, 1, dim, seed=pairs)
        case.check(case.run())


@pytest.mark.parametrize("vocab", [40, 700])
def test_more_rows_than_a_batch(fk, gpu, vocab):
    """4100 rows: three batches of at most 2048 that take the scratch one after the other, settings a row each."""
    rng = np.random.default_rng(vocab)
    rows = 4100
    sampling.check(fk, gpu, sampling.logits_of(rng, rows, vocab), rng.random(rows), temperature=rng.uniform(0.3, 1.5, rows),
                   top_k=rng.integers(0, 30, rows), top_p=rng.uniform(0.5, 1.0, rows))


@pytest.mark.parametrize("heads,kv_heads", [(40, 1), (34, 2), (300, 1)])
@pytest.mark.parametrize("rows,lengths", [([1], [90]), ([1, 2], [2000, 65]), ([5], [1300])])
def test_more_heads_of_a_key_head_than_a_tile_has_pairs(fk, gpu, heads, kv_heads, rows, lengths):
    """One token's heads lie in several tiles, of both kernels, whole and split."""
    case = Case(fk, gpu, rows, lengths, heads, kv_heads, 32, seed=heads)
    case.check(case.run())


@pytest.mark.parametrize("rows,lengths", [([2, 1], [70, 300]), ([20, 0, 150], [100, 9, 400]), ([1, 2], [2000, 1500])])
def test_rows_before_the_first_sequence(fk, gpu, rows, lengths):
    """row_starts may begin past 0: the rows before are no sequence's, in writes, reads and attention."""
    import torch
    case = Case(fk, gpu, rows, lengths, 4, 2, 64)
    want = case.run()
    n, before = int(case.step.starts[-1]), 7
    keys, values = (torch.randn(before + n, 2, 64, generator=torch.Generator().manual_seed(s)) for s in (1, 2))
    for s, (r, length) in enumerate(zip(rows, lengths)):  # the same keys and values as are there
        a, b, end = int(case.step.starts[s]), int(case.step.starts[s + 1]), int(case.whole.starts[s + 1])
        keys[before + a:before + b], values[before + a:before + b] = case.keys[end - r:end], case.values[end - r:end]
    case.step.starts = case.step.starts + before
    batch = case.step.batch(fk, gpu)
    case.cache.write(batch, keys.to(gpu), values.to(gpu))
    back_k, back_v = torch.full((before + n, 2, 64), 3.0, device=gpu), torch.full((before + n, 2, 64), 3.0, device=gpu)
    case.cache.read(batch, back_k, back_v)
    for x, back in ((keys, back_k), (values, back_v)):
        assert bool((back[:before] == 3.0).all()) and torch.equal(back[before:].cpu().double(), serving.quantized(x[before:]).float().double())
    query = torch.cat([torch.full((before, 4, 64), float("nan")), case.query[:n]])
    out = torch.full_like(query, 5.0, device=gpu)
    case.cache.attend(batch, query.to(gpu), out=out)
    assert bool((out[:before] == 5.0).all()) and torch.equal(out[before:].cpu(), want[:n])


@pytest.mark.parametrize("rows,lengths,columns", [([1, 2], [700, 200], 3), ([1], [3000], 20), ([150], [400], 3), ([2], [3000], 17)])
@pytest.mark.parametrize("window", [0, 130])
def test_tables_shorter_than_the_sequences(fk, gpu, rows, lengths, columns, window):
    """Positions past the table hold nothing: the last tokens see what it has, or with a window nothing."""
    case = Case(fk, gpu, rows, lengths, 4, 2, 64, seed=columns)
    case.step.table = np.ascontiguousarray(case.step.table[:, :columns])
    got = case.run(window=window)
    case.check(got, window=window)


def test_no_sequences(fk, gpu):
    """Rows, but no sequence that holds them: nothing is read or written."""
    import torch
    cache = fk.PagedCache(2, 2, 64, device=gpu)
    ints = dict(dtype=torch.int32, device=gpu)
    batch = fk.Batch(torch.zeros(1, **ints), torch.zeros(0, **ints), torch.zeros(0, 3, **ints))
    keys, out = torch.full((5, 2, 64), 2.0, device=gpu), torch.full((5, 4, 64), 3.0, device=gpu)
    cache.write(batch, keys, keys)
    cache.read(batch, keys, keys.clone())
    cache.attend(batch, out.clone(), out=out)
    assert bool((keys == 2.0).all()) and bool((out == 3.0).all())
    assert not bool(cache.attend(batch, out).any())
