"""Attention of sequences that share prefixes: batches that break their rules, and what the calls reach of memory."""

import ctypes

import pytest

from test_gpu_prefixes import Shared

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


def test_starts_that_fall_read_no_memory_behind_the_scratch(fk, gpu):
    """2000 sequences that all name row 0 have more tasks than 1000 rows have room for, and behind them a long one whose parts
    would lie past the scratch's end, by 134 MiB. What lies there is NaN here, in the same allocation, and the scratch 0."""
    import torch
    from fusor_kernels import _lib
    lib = _lib.lib()
    sequences, rows, columns, heads = 4003, 1000, 600, 64
    cache = fk.PagedCache(1, heads, 4, device=gpu)
    starts = torch.tensor([s % 2 for s in range(4001)] + [0, 5, 5], dtype=torch.int32, device=gpu)
    lengths = torch.ones(sequences, dtype=torch.int32, device=gpu)
    lengths[4001] = 64 * columns
    batch = fk.Batch(starts, lengths, torch.full((sequences, columns), -1, dtype=torch.int32, device=gpu))
    prefixes = fk.Prefixes(torch.zeros(2, dtype=torch.int32, device=gpu), torch.ones(1, dtype=torch.int32, device=gpu))
    query, out = torch.ones(rows, heads, 4, device=gpu), torch.zeros(rows, heads, 4, device=gpu)
    fg, ffi = batch._ffi(rows), prefixes._ffi()
    size = lib.fg_cache_attend_shared_scratch(cache.handle, ctypes.byref(fg), ctypes.byref(ffi), heads)
    assert size % 4 == 0 and size > lib.fg_cache_attend_scratch(cache.handle, ctypes.byref(fg), heads)
    memory = torch.full((size // 4 + (160 << 18),), float("nan"), device=gpu)
    memory[:size // 4] = 0.0
    _lib.check(lib.fg_cache_attend_shared(cache.handle, ctypes.byref(fg), ctypes.byref(ffi), query.data_ptr(), heads * 4, heads, 0.5, 0,
                                          out.data_ptr(), heads * 4, memory.data_ptr(), size, None))
    torch.cuda.synchronize()
    assert not bool(torch.isnan(out).any()) and not bool(out[5:].any())
    assert bool(torch.isnan(memory[size // 4:]).all())


def sizes_of_scratch(case):
    """... of a case's call, and of the one over each sequence's own table."""
    import torch
    from fusor_kernels import _lib
    fg = case.step.batch(case.fk, case.gpu)._ffi(case.step.total())
    prefixes = case.fk.Prefixes(*(torch.tensor(x, dtype=torch.int32, device=case.gpu) for x in case.groups))
    lib, ffi = _lib.lib(), prefixes._ffi()
    return (lib.fg_cache_attend_shared_scratch(case.cache.handle, ctypes.byref(fg), ctypes.byref(ffi), case.heads),
            lib.fg_cache_attend_scratch(case.cache.handle, ctypes.byref(fg), case.heads))


def test_arrays_with_room_for_more_groups(fk, gpu):
    """... than the batch has sequences, all but one of them empty, work a prefix through once as arrays of one group do."""
    import torch
    case = Shared(fk, gpu, [1] * 9, [1300 + 9 * s for s in range(9)], [0, 9], [20], 8, 2, 64)
    shared, by_itself = sizes_of_scratch(case)
    assert shared > by_itself
    want = case.run()
    case.check(want)
    for room in (8, 9, 40):
        case.groups = ([0] + [9] * room, [20] + [0] * (room - 1))
        assert sizes_of_scratch(case)[0] > by_itself
        assert torch.equal(case.run(), want)
