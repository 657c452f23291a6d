"""Attention over the paged cache against 64 bits.

Tolerance of an output, with W the sum of |weight * value| over its row's keys, A the largest sum of
|scale * q * k| over its keys and e = 2^-24 (half a step of f32): a score's products are exact, their
f32 sum of D terms is off by at most D e A, the two f16 pieces of the query and the scales' products
by 2^-22 A and 4 e A, so t by (D + 8) e A; an exponential follows it and adds 4 e; the weights' pieces
2^-22 = 4 e; the sums over n keys n e each, above and below the division. Together
W e (2 A (D + 8) + 2 n + 16).

A weight times its value's scale is also no finer than f16's smallest step, 2^-24, in units where the row's
largest is at least 2^9: off by half of that, 2^-34 of the largest, a key. Times the levels, n 2^-34 of
the row's largest |weight * value| is added. (A row whose one heavy key has level 0 in a dimension shows
it: there W is next to nothing.)
"""

import numpy as np
import pytest

import serving

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


class Case:
    """A step whose cache holds random tokens; the oracle's keys and values are what the cache holds."""

    def __init__(self, fk, gpu, rows, lengths, heads, kv_heads, dim, seed=0, padding=0, keys=None, values=None):
        import torch
        self.fk, self.gpu, self.heads, self.kv_heads, self.dim = fk, gpu, heads, kv_heads, dim
        self.step = serving.Step(rows, lengths, seed=seed, padding=padding)
        self.whole = self.step.whole()
        g = torch.Generator().manual_seed(seed)
        n = self.whole.total()
        self.keys = torch.randn(n, kv_heads, dim, generator=g) + 0.5 if keys is None else keys
        self.values = torch.randn(n, kv_heads, dim, generator=g) if values is None else values
        self.query = torch.randn(self.step.total(), heads, dim, generator=g)
        self.cache = fk.PagedCache(self.step.pages, kv_heads, dim, device=gpu)
        self.cache.write(self.whole.batch(fk, gpu), self.keys.to(gpu), self.values.to(gpu))

    def run(self, **options):
        import torch
        out = torch.full((self.step.total(), self.heads, self.dim), 5.0, device=self.gpu)
        self.cache.attend(self.step.batch(self.fk, self.gpu), self.query.to(self.gpu), out=out, **options)
        return out.cpu()

    def check(self, got, scale=None, window=0, skip=()):
        import torch
        scale = self.dim ** -0.5 if scale is None else scale
        k, v = serving.quantized(self.keys), serving.quantized(self.values)
        group = self.heads // self.kv_heads
        for s, (rows, length) in enumerate(zip(self.step.rows, self.step.lengths)):
            if rows == 0 or s in skip:
                continue
            a, b = int(self.whole.starts[s]), int(self.step.starts[s])
            ks, vs, q = k[a:a + length], v[a:a + length], self.query[b:b + rows]
            absent = torch.zeros(length, dtype=torch.bool)
            for p in range(0, length, 64):
                column = p // 64
                if column >= self.step.table.shape[1] or not 0 <= self.step.table[s, column] < self.step.pages:
                    absent[p:p + 64] = True
            positions = np.arange(length - rows, length)
            want, weighed, largest = serving.attention(q, ks, vs, positions, scale, window, absent)
            most = torch.zeros(rows, self.heads)
            for h in range(self.heads):
                most[:, h] = (q[:, h].double().abs() @ ks[:, h // group].abs().T).amax(1).float() * abs(scale)
            bound = weighed * 2.0 ** -24 * (2 * most[..., None].double() * (self.dim + 8) + 2 * length + 16)
            bound = bound + length * 2.0 ** -34 * largest[..., None] + 1e-37
            error = (got[b:b + rows].double() - want).abs()
            worst = float((error / bound).max())
            print(f"  sequence {s}: {rows} rows of {length}, error {float(error.max()):.2e}, {worst:.3f} of the bound", flush=True)
            assert worst <= 1, (s, rows, length)
        assert bool((got[int(self.step.starts[-1]):] == 5.0).all())  # the padding's rows


# one token a sequence; few; chunks (each with lengths around a page's and a tile's ends)
STEPS = [([1], [1]), ([1, 1, 1, 1], [64, 65, 2, 700]), ([2, 0, 5], [63, 9, 300]), ([9], [9]), ([70, 1], [70, 129]),
         ([33, 0, 128, 1], [161, 0, 128, 1]), ([130], [450])]
HEADS = [(1, 1, 32), (14, 2, 64), (4, 4, 72), (16, 4, 128), (5, 5, 36), (6, 2, 96), (8, 1, 128), (4, 2, 160), (2, 1, 256), (3, 3, 4)]


@pytest.mark.parametrize("rows,lengths", STEPS)
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
def test_against_64_bits(fk, gpu, rows, lengths, heads, kv_heads, dim):
    print(f"attend {rows} {lengths} {heads}/{kv_heads}x{dim}", flush=True)
    case = Case(fk, gpu, rows, lengths, heads, kv_heads, dim, seed=len(rows) + dim, padding=3)
    case.check(case.run())


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 100, 5000])
@pytest.mark.parametrize("rows,lengths", [([1, 1], [300, 40]), ([150], [400]), ([4, 3], [70, 200]), ([130, 1], [1500, 2100])])
def test_windows(fk, gpu, rows, lengths, window):
    case = Case(fk, gpu, rows, lengths, 4, 2, 64, seed=window)
    case.check(case.run(window=window), window=window)


@pytest.mark.parametrize("rows,length", [(3, 2), (6, 70), (130, 70), (40, 3000)])
@pytest.mark.parametrize("window", [2 ** 31 - 64, 2 ** 31 - 1, 2 ** 31, 2 ** 63])
def test_windows_longer_than_any_sequence(fk, gpu, rows, length, window):
    """... see what no window sees, rows before position 0 among them."""
    import torch
    case = Case(fk, gpu, [length], [length], 4, 2, 64)
    case.step.rows, case.step.starts = [rows], np.array([0, rows], np.int32)
    case.query = torch.randn(rows, 4, 64, generator=torch.Generator().manual_seed(1))
    assert torch.equal(case.run(window=window), case.run())


@pytest.mark.parametrize("rows,lengths,heads,kv_heads,dim", [
    ([1], [5000], 14, 2, 64), ([1, 1, 1], [9000, 1, 3001], 4, 1, 128), ([3], [4097], 8, 4, 128), ([40, 1], [2500, 1400], 4, 2, 64),
    ([400, 1], [2500, 1400], 4, 2, 64), ([150], [2600], 8, 2, 128), ([300], [2000], 3, 3, 72), ([120], [3000], 2, 1, 192)])
def test_long_caches_split_over_workgroups(fk, gpu, rows, lengths, heads, kv_heads, dim):
    case = Case(fk, gpu, rows, lengths, heads, kv_heads, dim)
    got = case.run()
    case.check(got)
    import torch
    assert torch.equal(got, case.run())  # nothing in the result depends on timing


@pytest.mark.parametrize("rows,lengths", [([1, 2], [3, 130]), ([100, 40], [60, 400])])
def test_rows_that_see_nothing(fk, gpu, rows, lengths):
    """Pages outside the cache hold no keys; rows before position 0, or all of whose pages are such, give 0."""
    case = Case(fk, gpu, rows, lengths, 4, 2, 64)
    case.step.table[0, :] = -1                   # no page at all
    case.step.table[1, 0] = case.step.pages + 5  # the first
    got = case.run()
    case.check(got)
    assert not bool(got[:rows[0]].any())
    # a table of no columns
    case.step.table = case.step.table[:, :0]
    got = case.run()
    assert not bool(got[:sum(rows)].any())


@pytest.mark.parametrize("rows", [1, 3, 150])
def test_a_cache_of_no_pages(fk, gpu, rows):
    """Nothing to see; the loads of a page that is not there stay inside the cache's memory, of every head."""
    import torch
    cache = fk.PagedCache(0, 8, 256, device=gpu)
    step = serving.Step([rows], [rows], padding=1)
    step.table[:] = -1
    query = torch.randn(step.total(), 16, 256, generator=torch.Generator().manual_seed(0)).to(gpu)
    out = torch.full_like(query, 5.0)
    cache.attend(step.batch(fk, gpu), query, out=out)
    assert not bool(out[:rows].any()) and bool((out[rows:] == 5.0).all())


def test_rows_past_their_sequence_length(fk, gpu):
    """More new rows than tokens: the first rows have no position."""
    import torch
    for rows, length in ((3, 2), (130, 70)):
        case = Case(fk, gpu, [length], [length], 4, 2, 64)
        step = case.step
        step.rows, step.starts = [rows], np.array([0, rows], np.int32)
        case.query = torch.randn(rows, 4, 64, generator=torch.Generator().manual_seed(1))
        got = case.run()
        assert not bool(got[:rows - length].any())
        step.rows, step.starts = [length], np.array([0, length], np.int32)
        case.query = case.query[rows - length:]
        case.check(got[rows - length:])


@pytest.mark.parametrize("rows,length", [(1, 100), (6, 100), (90, 100)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), 3e38, 1e30])
def test_what_is_masked_changes_nothing(fk, gpu, rows, length, bad):
    """Tokens behind a row's position, in its own page, hold anything: the row is as without them."""
    import torch
    case = Case(fk, gpu, [rows], [length], 8, 2, 64)
    want = case.run()
    full = serving.Step([60], [length + 60])
    full.table[:, :2], full.pages = case.step.table[:, :2], max(case.step.pages, full.pages)
    ids = [i for i in range(case.step.pages) if i not in case.step.table[0]]
    full.table[0, 2] = ids[0]
    later = torch.randn(60, 2, 64)
    later[:, 0, 0] = bad
    later[::3] = bad
    case.cache.write(full.batch(fk, gpu), later.to(gpu), later.to(gpu))
    assert torch.equal(case.run(), want)


@pytest.mark.parametrize("rows,length", [(1, 80), (7, 200), (100, 200)])
def test_values_of_very_different_sizes(fk, gpu, rows, length):
    """A value far larger than the others that hardly weighs anything leaves them their bits; tiny
    and huge values throughout."""
    import torch
    g = torch.Generator().manual_seed(3)
    keys = torch.randn(length, 1, 64, generator=g)
    for size in (1e25, 1e-25, 1e-30, 1e36):
        values = torch.randn(length, 1, 64, generator=g)
        values[5] *= size
        away = keys.clone()
        away[5] = -20.0
        case = Case(fk, gpu, [rows], [length], 4, 1, 64, keys=away, values=values)
        case.query = case.query.abs() + 0.2  # key 5 weighs e^-100 and less
        case.check(case.run())
        # 1e36 * 127 levels sum past f32's range: that is the values' own overflow
        case = Case(fk, gpu, [rows], [length], 4, 1, 64, keys=keys, values=values * 0 + torch.randn(length, 1, 64, generator=g) * min(size, 1e30))
        case.check(case.run())


@pytest.mark.parametrize("rows", [1, 5, 80])
def test_queries_and_scores_of_every_size(fk, gpu, rows):
    import torch
    for size, scale in ((1e-30, 1e30), (1e30, 1e-30), (30.0, None), (0.0, None), (1.0, -1.0), (1.0, 0.0)):
        case = Case(fk, gpu, [rows], [150], 4, 2, 32)
        case.query = case.query * size
        case.check(case.run(scale=scale), scale=scale)


@pytest.mark.parametrize("rows", [2, 80])
def test_nan_and_infinity_stay_in_their_rows(fk, gpu, rows):
    """A query of NaN, a key or value of infinity: the rows that see it are NaN, the others exact."""
    import torch
    case = Case(fk, gpu, [rows], [100], 4, 2, 64)
    clean = case.run()
    query = case.query.clone()
    case.query[rows - 1, 1] = float("nan")
    got = case.run()
    assert bool(torch.isnan(got[rows - 1, 1]).all())
    got[rows - 1, 1] = clean[rows - 1, 1]
    assert torch.equal(got, clean)
    case.query = query
    tokens = torch.randn(1, 2, 64)
    tokens[0, 1, 3] = float("inf")  # the second key head's last token
    case.step.rows, case.step.starts = [1], np.array([0, 1], np.int32)
    case.cache.write(case.step.batch(fk, gpu), tokens.to(gpu), tokens.to(gpu))
    case.step.rows, case.step.starts = [rows], np.array([0, rows], np.int32)
    got = case.run()
    assert bool(torch.isnan(got[rows - 1, 2:]).all()) and not bool(torch.isnan(got[rows - 1, :2]).any())
    assert torch.equal(got[:rows - 1], clean[:rows - 1])


def test_strides_and_unaligned_rows(fk, gpu):
    import torch
    for rows in ([1, 1], [90, 3], [200, 3]):
        case = Case(fk, gpu, rows, [max(rows[0], 95), 100], 4, 2, 36)
        n, width = case.step.total(), 4 * 36
        flat = torch.full((n * 301 + 1,), 9.0, device=gpu)
        query = flat.as_strided((n, 4, 36), (301, 36, 1), 1)
        query.copy_(case.query)
        out = flat.as_strided((n, 4, 36), (301, 36, 1), 1 + width + 2)
        case.cache.attend(case.step.batch(fk, gpu), query, out=out)
        case.check(out.cpu())
        assert torch.equal(query.cpu(), case.query) and int((flat == 9.0).sum()) == flat.numel() - 2 * n * width


def test_sequences_that_share_pages(fk, gpu):
    """Two sequences over one prompt's pages, their own tokens in pages of their own."""
    import torch
    case = Case(fk, gpu, [5, 5], [133, 133], 4, 2, 64)
    case.step.table[1, :2] = case.step.table[0, :2]
    a, b = int(case.whole.starts[0]), int(case.whole.starts[1])
    case.keys[b:b + 128], case.values[b:b + 128] = case.keys[a:a + 128], case.values[a:a + 128]
    case.check(case.run())


@pytest.mark.parametrize("rows,lengths", [([1, 1], [2500, 40]), ([9], [70]), ([150, 3], [2500, 300]), ([300], [300])])
def test_outputs_over_the_queries(fk, gpu, rows, lengths):
    """`out` may be `queries`: a row's are read before its outputs are written."""
    case = Case(fk, gpu, rows, lengths, 8, 2, 64, padding=2)
    want = case.run()
    both = case.query.to(gpu)
    case.cache.attend(case.step.batch(fk, gpu), both, out=both)
    import torch
    n = int(case.step.starts[-1])
    assert torch.equal(both.cpu()[:n], want[:n]) and torch.equal(both.cpu()[n:], case.query[n:])


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_a_page_named_twice(fk, gpu, rows):
    """... by one sequence is seen twice."""
    case = Case(fk, gpu, [rows], [300], 4, 2, 64)
    case.step.table[0, 0] = case.step.table[0, 2]
    case.keys[:64], case.values[:64] = case.keys[128:192], case.values[128:192]
    case.check(case.run())


def test_many_sequences(fk, gpu):
    rng = np.random.default_rng(1)
    for high in (2, 9):
        rows = [int(r) for r in rng.integers(0, high, 150)]
        case = Case(fk, gpu, rows, [r + int(p) for r, p in zip(rows, rng.integers(0, 90, 150))], 2, 1, 32, padding=2)
        case.check(case.run())


def test_more_sequences_than_64_bits_of_lanes(fk, gpu):
    import torch
    rows = [1 if s % 7 else 0 for s in range(5000)]
    case = Case(fk, gpu, rows, [1 + s % 3 for s in range(5000)], 1, 1, 32)
    got = case.run()
    # one, two or three keys: the last rows checked whole, the others for being there
    assert bool(torch.isfinite(got).all())
    keep = set(range(4900, 5000))
    case.check(got, skip=set(range(5000)) - keep)


def test_offsets_past_32_bits(fk, gpu):
    import torch
    case = Case(fk, gpu, [1, 40], [200, 130], 16, 8, 256)
    pages = 17000  # 4.5 GB
    case.step.table[case.step.table >= 0] += pages - case.step.pages
    case.step.pages = case.whole.pages = pages
    case.whole.table = case.step.table
    case.cache = fk.PagedCache(pages, 8, 256, device=gpu)
    case.cache.write(case.whole.batch(fk, gpu), case.keys.to(gpu), case.values.to(gpu))
    case.check(case.run())


def test_refusals(fk, gpu):
    import torch
    case = Case(fk, gpu, [2], [2], 4, 2, 64)
    batch, good = case.step.batch(fk, gpu), case.query.to(gpu)
    for bad in (good.cpu(), good.double(), good[:, :3], good[..., :32], good[0], good.transpose(0, 1)):
        with pytest.raises(fk.ShapeError):
            case.cache.attend(batch, bad)
    for bad in (good.double(), good[:1], good[:, :2], good[:1].expand(2, 4, 64)):
        with pytest.raises(fk.ShapeError):
            case.cache.attend(batch, good, out=bad)
    with pytest.raises(fk.ShapeError):
        case.cache.attend(batch, good, window=-1)
    for scale in (float("nan"), float("inf"), 3e38, -3e38):
        with pytest.raises(ValueError):
            case.cache.attend(batch, good, scale=scale)
    assert case.cache.attend(batch, good[:0]).shape == (0, 4, 64)
