"""Attention of sequences that share prefixes: batches that break their rules, and what the calls reach of memory."""

import ctypes

import pytest

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
