"""CPU checks of the pages' book-keeping (Pages) and of the copies that are refused before any device work."""

import ctypes

import numpy as np
import pytest

import fusor_kernels as fk
from fusor_kernels import _lib


def test_pages_are_taken_shared_and_freed():
    pages = fk.Pages(10)
    a = pages.take(3)
    assert a == [0, 1, 2] and pages.free_pages == 7
    b, (sources, targets) = pages.fork(a, 2 * 64 + 5)  # two whole pages and a part
    assert b[:2] == a[:2] and sources == [2] and targets == [b[2]] == [3]
    assert [pages.users(p) for p in range(5)] == [2, 2, 1, 1, 0]
    c, copies = pages.fork(a, 128)  # whole pages only; a's third is not part of it
    assert c == a[:2] and copies == ([], []) and pages.users(2) == 1
    d, copies = pages.fork(a, 0)
    assert d == [] and copies == ([], [])
    pages.free(a)
    assert [pages.users(p) for p in range(5)] == [2, 2, 0, 1, 0] and pages.free_pages == 7
    pages.free(b), pages.free(c)
    assert pages.free_pages == 10 and not any(pages.users(p) for p in range(10))


def test_what_is_refused():
    pages = fk.Pages(4)
    a = pages.take(3)
    for bad in (5, -1):
        with pytest.raises(fk.Error):
            pages.take(bad)
    b, _ = pages.fork(a, 64 * 2 + 1)  # the last free page
    with pytest.raises(fk.Error, match="none is free"):
        pages.fork(a, 64 * 2 + 1)
    assert [pages.users(p) for p in range(4)] == [2, 2, 1, 1]  # nothing was shared by the refused fork
    for bad in ([0, 0], [7], [-1]):
        with pytest.raises(fk.ShapeError):
            pages.free(bad)
    with pytest.raises(fk.ShapeError):
        pages.fork(a, 64 * 3 + 1)
    pages.free(b), pages.free(a)
    with pytest.raises(fk.ShapeError):
        pages.free([0])


@pytest.mark.parametrize("seed", range(20))
def test_compaction(seed):
    """What every sequence holds is the same after the moves, in the lowest pages, and no page is moved onto one that is
    held or moved itself."""
    rng = np.random.default_rng(seed)
    count = int(rng.integers(1, 80))
    pages, sequences = fk.Pages(count), []
    content = {}
    for step in range(60):
        if rng.random() < 0.5 and pages.free_pages:
            got = pages.take(int(rng.integers(1, min(4, pages.free_pages) + 1)))
            for p in got:
                content[p] = (step, p)
            sequences.append(got)
        elif sequences and rng.random() < 0.5:
            source = sequences[int(rng.integers(len(sequences)))]
            if pages.free_pages:
                child, (old, new) = pages.fork(source, int(rng.integers(0, 64 * len(source) + 1)))
                for s, t in zip(old, new):
                    content[t] = content[s]
                sequences.append(child)
        elif sequences:
            pages.free(sequences.pop(int(rng.integers(len(sequences)))))
    held = [[content[p] for p in s] for s in sequences]
    used = count - pages.free_pages
    moves = pages.compact()
    sources, targets = list(moves), list(moves.values())
    assert len(set(targets)) == len(targets) and not set(targets) & set(sources)
    assert all(p >= used for p in sources) and all(p < used for p in targets)
    for s, t in moves.items():
        content[t] = content[s]
    sequences = [[moves.get(p, p) for p in s] for s in sequences]
    assert [[content[p] for p in s] for s in sequences] == held
    in_use = {p for s in sequences for p in s}
    assert in_use == set(range(used)) and pages.free_pages == count - used
    assert all(pages.users(p) == sum(p in s for s in sequences) for p in range(count))
    assert pages.compact() == {} and sorted(pages.take(count - used)) == list(range(used, count))


@pytest.mark.parametrize("kind", ["tuple", "array", "tensor", "iterator"])
def test_pages_of_any_kind_of_sequence(kind):
    """A row of a step's page table, for one: its ids, no sums with them, and none freed twice."""
    import torch
    of = {"tuple": tuple, "array": lambda p: np.array(p, np.int32), "tensor": lambda p: torch.tensor(p, dtype=torch.int32), "iterator": iter}[kind]
    pages = fk.Pages(10)
    a = pages.take(3)
    b, copies = pages.fork(of(a + [-1, -1]), 2 * 64 + 5)  # (a table's columns behind the sequence's)
    assert b == [0, 1, 3] and copies == ([2], [3]) and all(type(p) is int for p in b + copies[0])
    assert [pages.users(p) for p in range(5)] == [2, 2, 1, 1, 0] and pages.free_pages == 6
    with pytest.raises(fk.ShapeError):
        pages.free(of([1, 1]))
    pages.free(of(b))
    assert [pages.users(p) for p in range(5)] == [1, 1, 1, 0, 0]
    for bad in ([0.5], [None]):
        with pytest.raises(TypeError):
            pages.free(bad)
    pages.free(of(a))
    assert pages.free_pages == 10 and not any(pages.users(p) for p in range(10)) and sorted(pages.take(10)) == list(range(10))


class Cache:
    """What copy_pages looks at of a cache before any device work."""

    def __init__(self, pages, device="cuda:0"):
        import torch
        self.pages, self.device = pages, torch.device(device)


@pytest.mark.parametrize("sources,targets", [([1, 2], [3, 3]), ([1, 2], [2, 4]), ([1, 3], [3, 3]), ([1], [8]), ([-1], [2]), ([0, 9], [1, 2])])
def test_lists_that_are_refused(sources, targets):
    with pytest.raises(fk.ShapeError):
        fk.copy_pages([Cache(8), Cache(9)], sources, targets)


def test_ids_of_lists_are_whole_numbers():
    """... also where they come as tensors, which compare but do not hash alike."""
    import torch
    two = [torch.tensor(3), torch.tensor(3)]
    with pytest.raises(fk.ShapeError, match="named twice"):
        fk.copy_pages([Cache(8)], [1, 2], two)
    with pytest.raises(TypeError):
        fk.copy_pages([Cache(8)], [1, 2], [3.2, 3.7])


def test_copies_that_are_refused():
    import torch
    assert fk.copy_pages([], [1], [2]) is None
    with pytest.raises(fk.ShapeError, match="one device"):
        fk.copy_pages([Cache(8), Cache(8, "cuda:1")], [1], [2])
    with pytest.raises(fk.ShapeError):
        fk.copy_pages([Cache(8)], torch.tensor([1], dtype=torch.int32), [2])
    with pytest.raises(fk.ShapeError):
        fk.copy_pages([Cache(8)], torch.tensor([1], dtype=torch.int32), torch.tensor([2], dtype=torch.int32))
    copy = _lib.lib().fg_cache_copy
    some, caches = ctypes.c_void_p(256), (ctypes.c_void_p * 1)(None)
    assert copy(caches, 0, None, None, 5, None) == copy(caches, 1, None, None, 0, None) == _lib.FG_OK
    assert copy(None, 1, some, some, 1, None) == copy(caches, 1, None, some, 1, None) == copy(caches, 1, some, None, 1, None) == _lib.FG_ERR_ARG
    for count, pages in ((65537, 1), (1, (1 << 24) + 1)):
        assert copy(caches, count, some, some, pages, None) == _lib.FG_ERR_SHAPE
