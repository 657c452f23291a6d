"""Forms of the serving kernels that other tests' sizes do not reach: the decode kernel's parts and their
join for every size of head, both sides of the routing between the two kernels, and sampling of more rows than one
batch of workgroups takes. The bounds are those of test_gpu_cache_attend.py and test_gpu_sample.py."""

import numpy as np
import pytest

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
