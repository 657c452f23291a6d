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


@pytest.mark.parametrize("rows,length,every", [(1, 900, 256), (100, 900, 256), (150, 2560, 64)])
@pytest.mark.parametrize("late", [1.0, 1e-30])
def test_next_to_nothing_at_rising_scores(fk, gpu, rows, length, every, late):
    """Values of 1e-36 whose scores rise by 18 (2^26 in weight) every `every` tokens, a page of each wave's: they
    raise the sum of the weights and leave weight times value small. Values of `late` size come last, at the
    highest score: the outputs are theirs.

    A weight alone is at most 2^100 and the row's largest over 2^99, so the total is over 2^99; a weight times its
    value's scale is off by half of f16's smallest step, 2^-25, times the level, 127. So 127 * 2^-25 / 2^99 < 2^-117 a
    key is added to the bound: of rows that see only values of 1e-36 nothing is left."""
    import torch
    print(f"rising {rows} {length} {late}", flush=True)
    g = torch.Generator().manual_seed(7)
    keys, values = torch.zeros(length, 1, 32), torch.randn(length, 1, 32, generator=g)
    keys[:, 0, 0] = 18.0 * (torch.arange(length) // every)
    values[:-64] *= 1e-36
    values[-64:] *= late
    case = Case(fk, gpu, [rows], [length], 2, 1, 32, keys=keys, values=values)
    case.query = torch.zeros_like(case.query)
    case.query[:, :, 0] = 1.0
    got = case.run(scale=1.0).double()
    want, weighed, largest = serving.attention(case.query, serving.quantized(keys), serving.quantized(values),
                                               range(length - rows, length), 1.0)
    most = float(keys.max())  # of |scale q k|
    bound = weighed * 2.0 ** -24 * (2 * most * (32 + 8) + 2 * length + 16) + length * (2.0 ** -34 * largest[..., None] + 2.0 ** -117)
    worst = float(((got - want).abs() / bound).max())
    print(f"  {worst:.3f} of the bound", flush=True)
    assert worst <= 1


@pytest.mark.parametrize("rows,length", [(1, 200), (100, 200)])
def test_the_largest_keys_and_scores(fk, gpu, rows, length):
    """Keys of 1e33 against queries of 1e-33, and scores of 1e7: at the ends of what fg_cache_attend documents,
    every sum is finite. (Where one key has all the weight, an output is that key's value to its weight's two
    pieces, 2^-22, and four roundings of 2^-24: under 2^-20 of it.)"""
    import torch
    g = torch.Generator().manual_seed(8)
    keys = 1e33 * torch.randn(length, 2, 256, generator=g).clamp(-1, 1)
    case = Case(fk, gpu, [rows], [length], 4, 2, 256, keys=keys)
    case.query = case.query * 1e-33
    case.check(case.run())
    for size in (1.0, 1e-25, 1e30):  # of the values
        keys = torch.zeros(length, 1, 64)
        keys[:, 0, 0] = torch.rand(length, generator=g) - 0.5
        keys[-rows - 3, 0, 0] = 1.0  # whose weight is all that counts
        values = size * torch.randn(length, 1, 64, generator=g)
        case = Case(fk, gpu, [rows], [length], 2, 1, 64, keys=keys, values=values)
        case.query[:, :, 0] = 1e7
        got, want = case.run(scale=1.0), serving.quantized(values)[-rows - 3, 0]
        assert bool(((got.double() - want).abs() <= 2.0 ** -20 * want.abs().max()).all())


@pytest.mark.parametrize("rows,lengths", [([1], [16]), ([2, 1], [16, 9]), ([200], [200])])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_the_pieces_of_weights_and_queries(fk, gpu, rows, lengths, dim):
    """Scores that f32 holds exactly, over at most 16 keys, so that the bound is close to what the pieces leave.

    Keys are whole numbers k of magnitude up to 127 with one of 127 (scale 1), queries j + i / 2^11 with whole j and i
    of up to 4 and 2^11 (14 bits: both pieces count), of which a 32nd are not 0: a score's products and sums are
    multiples of 2^-11 under 2^13, exact in f32. The scale 2^-9 is exact; times log2 e it is rounded (e = 2^-24), so t, at
    most T = 16 * 1.45 in magnitude, is off by 2 e T, the difference from the reference by 2 e (T + 10) more at most; the
    exponential adds 4 e. A weight's pieces leave 2^-22 = 4 e, its product with the value's scale e; sums of 16 over and
    under the division 16 e each, the division e. Together (4 T + 20 + 9 + 33 + 1) e W < 160 e W for the weighed sum
    W; as elsewhere 2^-34 a key of the largest is added. One f16 piece would leave 2^-12 = 4096 e."""
    import torch
    g = torch.Generator().manual_seed(dim)
    n = sum(lengths)
    keys = torch.randint(-127, 128, (n, 1, dim), generator=g).float()
    keys[:, 0, 0] = 127
    case = Case(fk, gpu, rows, lengths, 2, 1, dim, keys=keys)
    shape = case.query.shape
    query = torch.randint(-4, 5, shape, generator=g) + torch.randint(0, 2 ** 11, shape, generator=g) / 2 ** 11
    case.query = torch.where(torch.rand(shape, generator=g) < 1 / 32, query, torch.zeros(()))
    assert float((case.query.abs().flatten(0, 1) @ keys[:, 0].abs().T).max()) < 2 ** 13
    got = case.run(scale=2.0 ** -9, window=16).double()
    values = serving.quantized(case.values)
    for s, (r, length) in enumerate(zip(rows, lengths)):
        a, b = int(case.whole.starts[s]), int(case.step.starts[s])
        want, weighed, largest = serving.attention(case.query[b:b + r], keys[a:a + length], values[a:a + length],
                                                   range(length - r, length), 2.0 ** -9, 16)
        bound = 160 * 2.0 ** -24 * weighed + 16 * 2.0 ** -34 * largest[..., None]
        worst = float(((got[b:b + r] - want).abs() / bound).max())
        print(f"  sequence {s}: {worst:.3f} of the bound", flush=True)
        assert worst <= 1
