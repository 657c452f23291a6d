"""Attention over value vectors that hold nothing, or next to nothing, beside others: they take no bits from
the others and no sum leaves its range. The bound is that of test_gpu_cache_attend.py, in which a value of zeros
counts as what it is, 0."""

import numpy as np
import pytest

import serving
from test_gpu_cache_attend import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


# the decode kernel, whole and split, and the one for many rows, whole and split
STEPS = [([1], [64]), ([3, 1], [200, 70]), ([2], [2600]), ([100], [200]), ([150], [2600])]


@pytest.mark.parametrize("rows,lengths", STEPS)
@pytest.mark.parametrize("size", [1e-3, 1e-5, 1e-6, 1e-7, 1e-9])
@pytest.mark.parametrize("nothing", ["one", "half", "nan"])
def test_value_vectors_of_zeros(fk, gpu, rows, lengths, size, nothing):
    """... or of NaN alone, which are kept as zeros."""
    import torch
    print(f"zero values {rows} {lengths} {size} {nothing}", flush=True)
    g = torch.Generator().manual_seed(5)
    n = sum(lengths)
    values = size * torch.randn(n, 2, 64, generator=g)
    if nothing == "half":
        values[torch.rand(n, 2, generator=g) < 0.5] = 0
    else:
        values[0] = values[7, 1] = values[-1] = 0 if nothing == "one" else float("nan")
    case = Case(fk, gpu, rows, lengths, 4, 2, 64, seed=3, values=values)
    case.check(case.run())


@pytest.mark.parametrize("rows", [1, 100])
@pytest.mark.parametrize("size", [1e-5, 1e-8])
def test_tokens_that_were_never_written(fk, gpu, rows, size):
    """A token of a fresh page is a key and a value of zeros: it weighs e^0, and adds nothing."""
    import torch
    g = torch.Generator().manual_seed(6)
    length = 150
    keys, values = 0.3 * torch.randn(length, 2, 64, generator=g), size * torch.randn(length, 2, 64, generator=g)
    keys[:20], values[:20] = 0, 0
    case = Case(fk, gpu, [rows], [length], 4, 2, 64, keys=keys, values=values)
    case.cache = fk.PagedCache(case.step.pages, 2, 64, device=gpu)
    step = serving.Step([length - 20], [length])
    step.table, step.pages = case.step.table, case.step.pages
    case.cache.write(step.batch(fk, gpu), keys[20:].to(gpu), values[20:].to(gpu))
    case.check(case.run())
