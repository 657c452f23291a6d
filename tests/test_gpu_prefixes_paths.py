"""Attention of sequences that share prefixes, where the shared pages are worked through apart: every case here says so by the
scratch that its call asks for. The tolerance is test_gpu_cache_attend.py's unless a test has its own."""

import numpy as np
import pytest

import serving
from test_gpu_prefixes import HEADS, Shared
from test_gpu_prefixes_limits import sizes_of_scratch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


def takes_shared(case, window=0):
    """The host's rule, and for no window what the call's scratch says of it."""
    group, rows = case.heads // case.kv_heads, case.step.total()
    padded = -(-case.dim // 32) * 32 if case.dim <= 128 else 192 if case.dim <= 192 else 256
    sequences = min(len(case.step.lengths), rows)
    columns = case.step.table.shape[1] if not window else min(case.step.table.shape[1], window // 64 + 2)
    room = sequences * columns * case.kv_heads * (128 * padded + 512) >= 224 * 2 ** 20
    shared = sequences > 1 and room and rows * group <= (96 if padded <= 128 else 64) * sequences
    if not window:
        sizes = sizes_of_scratch(case)
        assert (sizes[0] > sizes[1]) == shared, sizes
    return shared


@pytest.mark.parametrize("count,groups", [(1500, 500), (900, 300), (1020, 3), (3000, 40), (1024, 1), (1025, 1)])
def test_more_spans_than_the_plan_has_threads(fk, gpu, count, groups):
    """The plan lists 1024 spans at a time: tasks, joins and rows' records of the later ones lie behind the first ones', and past 1024
    sequences the arrays are read from memory. The last sequences and groups have rows, several tiles and shared pages."""
    rng = np.random.default_rng(count)
    starts = np.concatenate([[0], np.sort(rng.integers(0, count - 30, groups - 1)), [count - 3]]).tolist()
    pages = rng.integers(0, 4, groups).tolist()
    pages[-1] = 3
    lengths = [192 + int(p) for p in rng.integers(1, 150, count)]
    rows = [int(r) for r in rng.integers(0, 3, count)]
    for s, r in ((count - 1, 130), (count - 2, 7), (count - 5, 140), (count - 6, 1), (0, 60), (count // 2, 110)):
        rows[s] = r
    case = Shared(fk, gpu, rows, lengths, starts, pages, 2, 1, 32, padding=2)
    assert takes_shared(case)
    checked = set(range(30)) | set(range(count // 2 - 5, count // 2 + 5)) | set(range(count - 40, count)) | set(range(1020, min(1030, count)))
    got = case.run()
    case.check(got, skip=set(range(count)) - checked)
    import torch
    assert torch.equal(got, case.run())


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
def test_chunks_among_the_sequences_of_a_group(fk, gpu, heads, kv_heads, dim):
    """A sequence's large tiles joined to its group's parts; beside it enough single tokens that the rows are few on average."""
    rows, lengths = [40, 1, 1, 130, 1, 0, 1], [1360, 1290, 1400, 1600, 1300, 1290, 2600]
    rows, lengths = rows[:6] + [1] * 24 + rows[6:], lengths[:6] + [1300 + 5 * s for s in range(24)] + lengths[6:]
    case = Shared(fk, gpu, rows, lengths, [0, 30, 31], [20, 40], heads, kv_heads, dim, seed=dim, padding=3)
    assert takes_shared(case)
    case.check(case.run(), skip=set(range(8, 28)))


@pytest.mark.parametrize("window", [1, 64, 100, 1250, 1400])
@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 4, 128), (8, 2, 256), (6, 2, 96), (4, 2, 160)])
def test_windows_over_shared_pages(fk, gpu, heads, kv_heads, dim, window):
    rows, lengths = [30, 1, 1, 130, 2, 0, 1], [1360, 1290, 1400, 1600, 1300, 1290, 2600]
    case = Shared(fk, gpu, rows, lengths, [0, 6, 7], [20, 40], heads, kv_heads, dim, seed=dim, empty=6000)
    assert takes_shared(case, window)
    case.check(case.run(window=window), window=window)


@pytest.mark.parametrize("heads,kv_heads,dim", [(90, 1, 32), (96, 1, 64), (64, 1, 192), (48, 1, 36), (49, 1, 128)])
def test_many_query_heads_of_a_key_head(fk, gpu, heads, kv_heads, dim):
    for count in (2, 5):
        case = Shared(fk, gpu, [1] * count, [1290 + 3 * s for s in range(count)], [0, count], [20], heads, kv_heads, dim, seed=count)
        assert takes_shared(case)
        case.check(case.run())


@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (16, 4, 128), (4, 2, 160)])
def test_large_tiles_of_rows_without_a_position(fk, gpu, heads, kv_heads, dim):
    """More new rows than tokens, in large tiles: the first rows give 0, in a group and behind it."""
    import torch
    single, rows, length = 60, 203, 200
    case = Shared(fk, gpu, [1] * single + [1, 1], [1300] * single + [length, length], [0, single + 1], [3], heads, kv_heads, dim)
    assert takes_shared(case)
    step = case.step
    g = torch.Generator().manual_seed(1)
    step.rows, step.starts = [1] * single + [rows, rows], np.concatenate([np.arange(single + 1), [single + rows, single + 2 * rows]]).astype(np.int32)
    case.query = torch.randn(single + 2 * rows, heads, dim, generator=g)
    assert takes_shared(case)
    got = case.run()
    none = torch.zeros(single + 2 * rows, dtype=torch.bool)
    none[single:single + 3] = none[single + rows:single + rows + 3] = True
    assert not bool(got[none].any())
    # the oracle: the same without those rows
    step.rows, step.starts = [1] * single + [length, length], np.concatenate([np.arange(single + 1), [single + length, single + 2 * length]]).astype(np.int32)
    case.query = case.query[~none]
    case.check(got[~none], skip=set(range(3, single)))


@pytest.mark.parametrize("rows,lengths,pages", [([1] * 9, [64 + s for s in range(1, 10)], 1), ([1] * 40, [64 + s % 17 + 1 for s in range(40)], 1),
                                                ([1] * 5 + [120] + [1] * 30, [70] * 5 + [190] + [66] * 30, 1),
                                                ([2, 1, 3], [64, 9, 16], 1)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 32), (4, 2, 64), (6, 2, 96), (4, 2, 128), (2, 2, 160), (2, 1, 256)])
def test_the_pieces_of_weights_and_queries(fk, gpu, rows, lengths, pages, heads, kv_heads, dim):
    """Scores that f32 holds exactly, over few keys, so that the bound is close to what the two f16 pieces of the queries (split
    once, for the tiles of all heads) and of the weights leave: in small and large tiles of a group, and of a sequence.

    Keys are whole numbers of magnitude up to 127 with one of 127 (scale 1), queries j + i / 2^11 with whole j and i of up to 4
    and 2^11 (14 bits: both pieces count), of which a 32nd (an eighth for heads of 32) are not 0: a score's products and sums are multiples
    of 2^-11 under 2^13, exact in f32. The scale 2^-9 is exact; times log2 e it is rounded (e = 2^-24), so t, at most T = 16 * 1.45 in
    magnitude, is off by 2 e T, the difference from the reference by 2 e (T + 10) more at most; the exponential adds 4 e. A weight's
    pieces leave 2^-22 = 4 e, its product with the value's scale e; sums of n and of the joined parts, of which there are under 16 here
    (their factors are powers of two), n + 16 e each over and under the division, the division e. Together
    (4 T + 20 + 9 + 2 (n + 16) + 1) e W < (155 + 2 n) e W for the weighed sum W; n 2^-34 of the largest is added as elsewhere. One
    piece would leave 2^-12 = 4096 e of a query's values, and so of t."""
    import torch
    g = torch.Generator().manual_seed(dim + len(rows))
    n = sum(lengths)
    keys = torch.randint(-127, 128, (n, kv_heads, dim), generator=g).float()
    keys[:, :, 0] = 127
    case = Shared(fk, gpu, rows, lengths, [0, len(rows)], [pages], heads, kv_heads, dim, keys=keys)
    assert takes_shared(case)
    shape = case.query.shape
    query = torch.randint(-4, 5, shape, generator=g) + torch.randint(0, 2 ** 11, shape, generator=g) / 2 ** 11
    case.query = torch.where(torch.rand(shape, generator=g) < max(1 / 32, 4 / dim), query, torch.zeros(()))
    assert float((case.query.abs().flatten(0, 1).double() @ case.keys.abs().flatten(0, 1).double().T).max()) < 2 ** 13
    got = case.run(scale=2.0 ** -9).double()
    values = serving.quantized(case.values)
    for s, (r, length) in enumerate(zip(rows, lengths)):
        a, b = int(case.whole.starts[s]), int(case.step.starts[s])
        want, weighed, largest = serving.attention(case.query[b:b + r], case.keys[a:a + length], values[a:a + length],
                                                   range(length - r, length), 2.0 ** -9)
        bound = (155 + 2 * length) * 2.0 ** -24 * weighed + length * 2.0 ** -34 * largest[..., None]
        worst = float(((got[b:b + r] - want).abs() / bound).max())
        if s < 3 or worst > 0.5:
            print(f"  sequence {s}: {worst:.3f} of the bound", flush=True)
        assert worst <= 1
