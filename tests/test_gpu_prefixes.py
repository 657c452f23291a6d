"""Attention of sequences that share prefixes against 64 bits, with the bound of test_gpu_cache_attend.py: the
order of additions differs, their number does not.

Shared pages are worked through apart where what the sequences may see of their tables together, all of them or a window,
has room for 224 MiB; the tables here are widened with columns of no page for that, or with sequences of no tokens."""

import numpy as np
import pytest

import serving
from test_gpu_cache_attend import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


class Shared(Case):
    """A step of groups of sequences: group g's first starts[g + 1] - starts[g] sequences begin with pages[g] pages of the
    group's first sequence."""

    def __init__(self, fk, gpu, rows, lengths, starts, pages, heads, kv_heads, dim, wide=True, empty=0, padding=0, **options):
        rows, lengths = list(rows) + [0] * empty, list(lengths) + [0] * empty
        super().__init__(fk, gpu, rows, lengths, heads, kv_heads, dim, padding=max(padding, empty), **options)
        if wide:
            page = kv_heads * (128 * (-(-dim // 32) * 32) + 512)  # bytes, at least
            columns = -(-2 ** 28 // (page * min(len(rows), sum(rows))))
            more = np.full((len(rows), max(0, columns - self.step.table.shape[1])), -1, np.int32)
            self.step.table = np.concatenate([self.step.table, more], 1)
            self.whole.table = self.step.table
        self.groups = (list(starts), list(pages))
        for g, n in enumerate(pages):
            for s in range(starts[g] + 1, starts[g + 1]):
                a, b = int(self.whole.starts[starts[g]]), int(self.whole.starts[s])
                m = min(64 * n, lengths[s], lengths[starts[g]])
                self.step.table[s, :n] = self.step.table[starts[g], :n]
                self.keys[b:b + m], self.values[b:b + m] = self.keys[a:a + m], self.values[a:a + m]

    def run(self, **options):
        import torch
        starts, pages = (torch.tensor(x, dtype=torch.int32, device=self.gpu) for x in self.groups)
        return super().run(prefixes=self.fk.Prefixes(starts, pages), **options)


# rows and lengths of the sequences, the groups' starts, the pages they share: one token each, several, chunks among
# them, groups without rows or without pages, sequences before, between and behind the groups
STEPS = [([1] * 5, [130, 140, 129, 200, 128 + 64], [0, 5], [2]),
         ([1] * 70, [1300 + 7 * s for s in range(70)], [0, 70], [20]),
         ([1, 2, 1, 1, 3, 1], [1400, 1500, 90, 2300, 2310, 7], [1, 2, 2, 3, 5], [17, 3, 1, 30]),
         ([40, 1, 1, 130, 1, 0, 1], [1360, 1290, 1400, 1600, 1300, 1290, 2600], [0, 6, 7], [20, 40]),
         ([0, 0, 1], [1300, 1300, 1300], [0, 2, 3], [20, 20]),
         ([1, 1, 1, 1], [2000, 2010, 300, 2600], [0, 2, 4], [31, 0]),
         ([9] * 8, [1100 + 64 * s for s in range(8)], [0, 8], [17])]
HEADS = [(14, 2, 64), (16, 4, 128), (4, 4, 72), (5, 5, 36), (8, 1, 128), (6, 2, 96), (4, 2, 160), (2, 1, 256), (3, 1, 4)]


@pytest.mark.parametrize("step", range(len(STEPS)))
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
def test_against_64_bits(fk, gpu, step, heads, kv_heads, dim):
    print(f"prefixes {step} {heads}/{kv_heads}x{dim}", flush=True)
    case = Shared(fk, gpu, *STEPS[step], heads, kv_heads, dim, seed=dim, padding=3)
    got = case.run()
    case.check(got)
    import torch
    assert torch.equal(got, case.run())  # nothing in the result depends on timing


@pytest.mark.parametrize("step", range(len(STEPS)))
def test_narrow_tables(fk, gpu, step):
    """... where each sequence reads its table by itself."""
    case = Shared(fk, gpu, *STEPS[step], 4, 2, 64, wide=False, seed=step, padding=1)
    case.check(case.run())


@pytest.mark.parametrize("rows,pages", [([102], 4), ([102], 5), ([250, 250], 7), ([250, 3], 9), ([120] * 4, 8), ([120] * 4, 9), ([78] * 13, 16)])
@pytest.mark.parametrize("window", [0, 200])
@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (16, 4, 128), (8, 2, 256), (5, 5, 36)])
def test_chunks_over_short_tables(fk, gpu, rows, pages, window, heads, kv_heads, dim):
    """Tables of 4 to 16 pages, to both sides of where a chunk's tiles are split."""
    print(f"chunks {rows} {pages} pages {heads}/{kv_heads}x{dim} window {window}", flush=True)
    lengths = [64 * pages - 17 * s for s in range(len(rows))]
    case = Shared(fk, gpu, rows, lengths, [0, len(rows)], [1], heads, kv_heads, dim, wide=False, seed=pages)
    case.check(case.run(window=window), window=window)


@pytest.mark.parametrize("window", [1, 63, 64, 100, 1250, 1400, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("step", [0, 1, 2, 3])
@pytest.mark.parametrize("empty", [0, 8000])  # (as many windows of two pages of 17 KiB are more than that)
def test_windows(fk, gpu, step, window, empty):
    case = Shared(fk, gpu, *STEPS[step], 4, 2, 64, seed=window % 1000, padding=1, empty=empty)
    case.check(case.run(window=window), window=window)


@pytest.mark.parametrize("heads,kv_heads,dim", [(16, 4, 128), (14, 2, 64), (1, 1, 32), (34, 1, 32), (300, 1, 32)])
def test_many_pairs_of_a_group(fk, gpu, heads, kv_heads, dim):
    """Tiles whose pairs begin in the middle of a token's heads, groups around the sizes where the kernels change."""
    for count in (2, 6, 7, 12, 13, 14, 24, 25, 33):
        case = Shared(fk, gpu, [1] * count, [1200 + 3 * s for s in range(count)], [0, count], [18], heads, kv_heads, dim, seed=count)
        case.check(case.run(), skip=set(range(2, count - 2)))


@pytest.mark.parametrize("rows", [[3, 70, 1, 200], [3, 70, 1, 100], [1, 5, 1, 2]])
def test_prefixes_longer_than_a_sequence(fk, gpu, rows):
    """Tokens inside the shared pages see what lies up to them, whether the step wrote them or not."""
    for heads, kv_heads in ((4, 2), (2, 2)):
        for empty in (0, 2000):
            case = Shared(fk, gpu, rows, [1300, 1250, 640, 1290], [0, 4], [20], heads, kv_heads, 64, empty=empty)
            case.check(case.run())
            case.check(case.run(window=500), window=500)


def test_sequences_of_no_tokens_and_one(fk, gpu):
    """... in groups and between them, beside long ones."""
    import torch
    case = Shared(fk, gpu, [1, 0, 1, 1, 0, 1, 1], [1300, 0, 1, 1310, 0, 1, 1290], [0, 2, 5], [20, 0], 4, 2, 64)
    case.check(case.run())
    case.step.lengths[3] = 0  # a new row of a sequence without tokens has no position
    got = case.run()
    assert not bool(got[2].any())
    case.check(got, skip={3})
    empty = case.cache.attend(fk.Batch(*(torch.zeros(s, dtype=torch.int32, device=gpu) for s in (1, 0, (0, 30)))), case.query.to(gpu)[:0],
                              prefixes=fk.Prefixes(*(torch.zeros(s, dtype=torch.int32, device=gpu) for s in (1, 0))))
    assert empty.shape == (0, 4, 64)


def test_arrays_of_any_values(fk, gpu):
    """Groups past the sequences, of negative or too many pages, are taken as far as they reach."""
    import torch
    rows, lengths = [1, 1, 1, 2], [1300, 1310, 1320, 1400]
    for starts, pages in (([0, 9], [2000]), ([-3, 2, 99], [20, 20]), ([0, 4], [-5]), ([0, 2, 2 ** 31 - 1], [20, 2 ** 31 - 1]), ([3, 3, 3], [5, 6]),
                          ([0], [])):
        case = Shared(fk, gpu, rows, lengths, [0, 4], [20], 4, 2, 64)
        if pages and max(pages) > 20:  # every table the same
            case.step.table[:] = case.step.table[0]
            case.step.lengths = case.whole.rows = case.whole.lengths = lengths = [1300] * 4
            case = Shared(fk, gpu, rows, [1300] * 4, [0, 4], [21], 4, 2, 64)
        case.groups = (starts, pages)
        case.check(case.run())


def test_starts_that_fall_reach_no_memory_outside(fk, gpu):
    """Rows of a batch that breaks its rules hold anything; rows that no sequence holds, and the rest of memory, stay."""
    import torch
    case = Shared(fk, gpu, [1] * 6, [1300 + s for s in range(6)], [0, 6], [20], 4, 2, 64, padding=2)
    case.step.starts = np.array([0, 5, 2, 6, 1, 3, 6], np.int32)
    case.groups = ([4, 0, 6, 2], [20, 3, 20])
    got = case.run()
    assert bool((got[6:] == 5.0).all())


def test_pages_that_are_not_there(fk, gpu):
    case = Shared(fk, gpu, [1, 1, 5], [1400, 1300, 1350], [0, 3], [18], 4, 2, 64)
    case.step.table[:, 3] = -1                 # a shared page
    case.step.table[1, 19] = case.step.pages   # one of a sequence's own
    case.step.table[2, :] = -1
    case.groups = ([0, 2, 3], [18, 18])
    got = case.run()
    case.check(got)
    assert not bool(got[2:7].any())


def test_few_rows_past_their_sequence_length(fk, gpu):
    import torch
    case = Shared(fk, gpu, [1, 1, 1], [1300, 1300, 80], [0, 2], [20], 2, 2, 64)
    step = case.step
    step.rows, step.starts = [1, 1, 90], np.array([0, 1, 2, 92], np.int32)  # the last: 90 rows, 80 tokens
    case.query = torch.randn(92, 2, 64, generator=torch.Generator().manual_seed(1))
    got = case.run()
    assert not bool(got[2:12].any())
    step.rows, step.starts = [1, 1, 80], np.array([0, 1, 2, 82], np.int32)
    case.query = torch.cat([case.query[:2], case.query[12:]])
    case.check(torch.cat([got[:2], got[12:]]))


def test_rows_past_their_sequence_length(fk, gpu):
    """More new rows than tokens: the first rows have no position and give 0."""
    import torch
    case = Shared(fk, gpu, [1, 1], [1300, 1300], [0, 2], [20], 4, 2, 64)
    step = case.step
    step.rows, step.starts, step.lengths = [1, 1303], np.array([0, 1, 1304], np.int32), [1300, 1300]
    case.query = torch.randn(1304, 4, 64, generator=torch.Generator().manual_seed(1))
    got = case.run()
    assert not bool(got[1:4].any())
    step.rows, step.starts = [1, 1300], np.array([0, 1, 1301], np.int32)
    case.query = torch.cat([case.query[:1], case.query[4:]])
    case.check(torch.cat([got[:1], got[4:]]), skip={0})


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), 3e38, 1e30])
def test_what_is_masked_changes_nothing(fk, gpu, bad):
    """Tokens behind a row's position, in the shared pages and in its own, hold anything."""
    import torch
    case = Shared(fk, gpu, [1] * 9, [1300 + s for s in range(9)], [0, 9], [20], 8, 2, 64)
    short = Shared(fk, gpu, [1] * 9, [1300 + s for s in range(9)], [0, 9], [20], 8, 2, 64)
    want = case.run()
    later = torch.full((1, 2, 64), bad).to(gpu)
    for s in range(9):
        p = 1300 + s  # the token behind the sequence's last
        page = torch.from_numpy(case.step.table[s:s + 1]).to(gpu)
        one = fk.Batch(torch.tensor([0, 1], dtype=torch.int32, device=gpu), torch.tensor([p + 1], dtype=torch.int32, device=gpu), page)
        case.cache.write(one, later, later)
    assert torch.equal(case.run(), want)
    # rows inside the shared pages: the first sequence's last prefix tokens are bad, sequences that end before do not see them
    short.step.lengths = [1270] * 9
    want = short.run()
    one = fk.Batch(torch.tensor([0, 10], dtype=torch.int32, device=gpu), torch.tensor([1280], dtype=torch.int32, device=gpu),
                   torch.from_numpy(short.step.table[:1]).to(gpu))
    short.cache.write(one, later.expand(10, 2, 64), later.expand(10, 2, 64))
    assert torch.equal(short.run(), want)


@pytest.mark.parametrize("size,scale", [(1e-30, 1e30), (1e30, 1e-30), (30.0, None), (0.0, None), (1.0, -1.0)])
def test_queries_and_scores_of_every_size(fk, gpu, size, scale):
    case = Shared(fk, gpu, [1] * 30, [1300 + s for s in range(30)], [0, 30], [20], 4, 2, 32)
    case.query = case.query * size
    case.check(case.run(scale=scale), scale=scale, skip=set(range(3, 27)))


def test_values_of_very_different_sizes(fk, gpu):
    """... in the shared pages beside those of the sequences' own, and the other way round."""
    import torch
    g = torch.Generator().manual_seed(3)
    lengths = [1290] * 6
    n = sum(lengths)
    for shared, own in ((1e25, 1.0), (1.0, 1e25), (1e-25, 1.0), (1.0, 1e-25)):
        values = torch.randn(n, 1, 64, generator=g).view(6, 1290, 1, 64)
        values[:, :1280] *= shared
        values[:, 1280:] *= own
        case = Shared(fk, gpu, [1] * 6, lengths, [0, 6], [20], 4, 1, 64, values=values.reshape(n, 1, 64))
        case.check(case.run())


def test_nan_stays_in_its_rows(fk, gpu):
    import torch
    case = Shared(fk, gpu, [1] * 40, [1300 + s for s in range(40)], [0, 40], [20], 4, 2, 64)
    clean = case.run()
    case.query[7, 1] = float("nan")
    got = case.run()
    assert bool(torch.isnan(got[7, 1]).all())
    got[7, 1] = clean[7, 1]
    assert torch.equal(got, clean)


def test_strides_and_outputs_over_the_queries(fk, gpu):
    import torch
    for count in (3, 60):
        case = Shared(fk, gpu, [1] * count, [1300 + s for s in range(count)], [0, count], [20], 4, 2, 36, padding=2)
        want = case.run()
        starts, pages = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in case.groups)
        prefixes, batch, n, width = fk.Prefixes(starts, pages), case.step.batch(fk, gpu), count + 2, 4 * 36
        flat = torch.full((n * 301 + 1,), 9.0, device=gpu)
        query = flat.as_strided((n, 4, 36), (301, 36, 1), 1)
        query.copy_(case.query)
        out = flat.as_strided((n, 4, 36), (301, 36, 1), 1 + width + 2)
        out[count:] = 5.0
        case.cache.attend(batch, query, out=out, prefixes=prefixes)
        assert torch.equal(out.cpu(), want) and torch.equal(query.cpu(), case.query)
        assert int((flat == 9.0).sum()) == flat.numel() - 2 * n * width
        case.cache.attend(batch, query, out=query, prefixes=prefixes)
        assert torch.equal(query.cpu()[:count], want[:count]) and torch.equal(query.cpu()[count:], case.query[count:])


def test_many_sequences_and_groups(fk, gpu):
    rng = np.random.default_rng(1)
    for count, groups in ((300, 90), (700, 3), (520, 520)):
        starts = np.concatenate([[0], np.sort(rng.integers(0, count, groups - 1)), [count - 5]]).tolist()
        pages = rng.integers(0, 20, groups).tolist()
        lengths = [1281 + int(p) for p in rng.integers(0, 90, count)]
        rows = [int(r) for r in rng.integers(0, 3, count)]
        case = Shared(fk, gpu, rows, lengths, starts, pages, 2, 1, 32, padding=2)
        case.check(case.run(), skip=set(range(40, count - 40)))


def test_offsets_past_32_bits(fk, gpu):
    case = Shared(fk, gpu, [1] * 20, [1300 + s for s in range(20)], [0, 20], [20], 16, 8, 256)
    pages = 17000  # 4.5 GB
    case.step.table[case.step.table >= 0] += pages - case.step.pages
    case.step.pages = case.whole.pages = pages
    case.whole.table = case.step.table
    case.cache = fk.PagedCache(pages, 8, 256, device=gpu)
    case.cache.write(case.whole.batch(fk, gpu), case.keys.to(gpu), case.values.to(gpu))
    case.check(case.run(), skip=set(range(2, 18)))


def test_a_captured_call_replays_with_other_groups(fk, gpu):
    """Replays with other queries, lengths, pages and groups, eager calls and synchronizations between them; scratch of the
    program and of the library."""
    import torch
    from fusor_kernels import serving as module
    for own_scratch in (True, False):
        with pytest.MonkeyPatch.context() as patch:
            if not own_scratch:
                patch.setattr(module, "_scratch", lambda size, device: None)
            case = Shared(fk, gpu, [1] * 40, [1300 + 9 * s for s in range(40)], [0, 25, 40], [20, 15], 8, 2, 64, padding=1)
            batch = case.step.batch(fk, gpu)
            query, out = case.query.to(gpu), torch.zeros(41, 8, 64, device=gpu)
            starts, pages = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in case.groups)
            prefixes = fk.Prefixes(starts, pages)
            case.cache.attend(batch, query, out=out, prefixes=prefixes)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                case.cache.attend(batch, query, out=out, prefixes=prefixes)
            for replay in range(5):
                query.copy_(torch.randn(query.shape, generator=torch.Generator().manual_seed(replay)))
                batch.lengths.copy_(torch.tensor([n - 3 * replay for n in case.step.lengths], dtype=torch.int32))
                pages.copy_(torch.tensor([20 - replay, 15 - 2 * replay], dtype=torch.int32))
                starts.copy_(torch.tensor([0, 25 - replay if replay < 3 else 25, 40 - replay], dtype=torch.int32))
                if replay in (1, 2):  # sequences that change their group share less
                    pages[1] = 0
                out.fill_(float("nan"))
                graph.replay()
                torch.cuda.synchronize()
                got = out.clone()
                want = case.cache.attend(batch, query, out=torch.full_like(out, float("nan")), prefixes=prefixes)
                assert torch.equal(got[:40], want[:40]) and not bool(torch.isnan(got[:40]).any()) and bool(torch.isnan(got[40:]).all())
                plain = case.cache.attend(batch, query)
                assert float((plain[:40] - got[:40]).abs().max()) < 1e-5
            del graph
            torch.cuda.synchronize()


def test_streams_and_threads_at_once(fk, gpu):
    import threading

    import torch
    cases = [Shared(fk, gpu, *STEPS[i], 4, 2, 64, seed=i) for i in (1, 2, 3, 6)]
    work = []
    for case in cases:
        starts, pages = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in case.groups)
        query = case.query.to(gpu)
        work.append((case, case.step.batch(fk, gpu), fk.Prefixes(starts, pages), query, torch.zeros_like(query), case.run()))
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    errors = []

    def go(i):
        try:
            case, batch, prefixes, query, out, _ = work[i]
            for _ in range(8):
                case.cache.attend(batch, query, out=out, prefixes=prefixes, stream=streams[i])
            streams[i].synchronize()
        except Exception as error:  # shown by the main thread
            errors.append(error)

    threads = [threading.Thread(target=go, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for case, _, _, _, out, want in work:
        n = int(case.step.starts[-1])
        assert torch.equal(out.cpu()[:n], want[:n])


def test_refusals(fk, gpu):
    import ctypes

    import torch
    from fusor_kernels import _lib
    case = Shared(fk, gpu, [1, 1], [1300, 1310], [0, 2], [20], 4, 2, 64)
    starts, pages = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in case.groups)
    for s, p in ((starts[:1], pages), (starts.long(), pages), (starts, pages.cpu()), (starts, pages.view(1, 1)), (starts.cpu(), pages.cpu())):
        with pytest.raises(fk.ShapeError):
            fk.Prefixes(s, p)
    prefixes, batch, query = fk.Prefixes(starts, pages), case.step.batch(fk, gpu), case.query.to(gpu)
    for bad in (query.double(), query[0], query[:, :3], query[..., :32]):
        with pytest.raises(fk.ShapeError):
            case.cache.attend(batch, bad, prefixes=prefixes)
    with pytest.raises(ValueError):
        case.cache.attend(batch, query, scale=float("nan"), prefixes=prefixes)
    lib, fg, ffi = _lib.lib(), batch._ffi(2), prefixes._ffi()
    out = torch.zeros_like(query)

    def call(prefixes, scratch, size):
        return lib.fg_cache_attend_shared(case.cache.handle, ctypes.byref(fg), prefixes, query.data_ptr(), 256, 4, 0.125, 0, out.data_ptr(), 256,
                                          scratch, size, None)

    assert call(None, None, 0) == _lib.FG_ERR_ARG and "null prefixes" in lib.fg_last_error().decode()
    assert call(ctypes.byref(_lib.FgPrefixes(65537, starts.data_ptr(), pages.data_ptr())), None, 0) == _lib.FG_ERR_SHAPE
    assert call(ctypes.byref(_lib.FgPrefixes(1, None, pages.data_ptr())), None, 0) == _lib.FG_ERR_ARG
    assert call(ctypes.byref(_lib.FgPrefixes(1, starts.data_ptr(), None)), None, 0) == _lib.FG_ERR_ARG
    size = lib.fg_cache_attend_shared_scratch(case.cache.handle, ctypes.byref(fg), ctypes.byref(ffi), 4)
    assert size > 0
    memory = torch.zeros(size + 16, dtype=torch.uint8, device=gpu)
    assert call(ctypes.byref(ffi), memory.data_ptr(), size - 1) == _lib.FG_ERR_SHAPE and "scratch" in lib.fg_last_error().decode()
    assert call(ctypes.byref(ffi), memory.data_ptr() + 4, size) == _lib.FG_ERR_SHAPE
    torch.cuda.synchronize()
    assert call(ctypes.byref(ffi), memory.data_ptr(), size) == _lib.FG_OK
    torch.cuda.synchronize()
    case.check(out.cpu())
    assert torch.equal(out.cpu(), case.run())
