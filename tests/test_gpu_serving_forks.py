"""Rotary positions, forks, attention over shared prefixes, copies and compactions as a program uses them together: answers
drawn from one prompt, and a step captured in a graph. Every stage is checked against 64 bits on the inputs that it got."""

import numpy as np
import pytest

import serving

pytestmark = pytest.mark.gpu

HEADS, KV_HEADS, DIM = 8, 2, 64
COLUMNS = 4000  # tables so wide that four sequences' take the shared pages apart


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


class Program:
    """Two layers' caches, their pages, and sequences as lists of pages; `stored` is what each layer's cache holds of them."""

    def __init__(self, fk, gpu, pages):
        self.fk, self.gpu = fk, gpu
        self.pages = fk.Pages(pages)
        self.caches = [fk.PagedCache(pages, KV_HEADS, DIM, device=gpu) for _ in range(2)]
        self.rotary = fk.Rotary(DIM, base=1e6, stretch=4.0, trained=512, device=gpu)
        import torch
        self.g = torch.Generator().manual_seed(0)

    class Sequence:
        def __init__(self):
            self.pages, self.length, self.stored = [], 0, [([], []), ([], [])]

    def batch(self, sequences, counts):
        import torch
        for s, n in zip(sequences, counts):
            s.length += n
            s.pages += self.pages.take(-(-s.length // 64) - len(s.pages))
        table = np.full((len(sequences), COLUMNS), -1, np.int32)
        for i, s in enumerate(sequences):
            table[i, :len(s.pages)] = s.pages
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        return starts, self.fk.Batch(torch.from_numpy(starts).to(self.gpu),
                                     torch.tensor([s.length for s in sequences], dtype=torch.int32, device=self.gpu),
                                     torch.from_numpy(table).to(self.gpu))

    def prefixes(self, groups):
        """Runs of sequences, each with as many pages as all of it begin with."""
        import torch
        starts, counts = [0], []
        for run in groups:
            n = 0
            while all(n < len(s.pages) and s.pages[n] == run[0].pages[n] for s in run) and len(run) > 1:
                n += 1
            starts.append(starts[-1] + len(run))
            counts.append(n)
        return self.fk.Prefixes(*(torch.tensor(x, dtype=torch.int32, device=self.gpu) for x in (starts, counts))), counts

    def step(self, groups, counts):
        import torch
        sequences = [s for run in groups for s in run]
        starts, batch = self.batch(sequences, counts)
        prefixes, shared = self.prefixes(groups)
        n = int(starts[-1])
        positions = np.concatenate([np.arange(s.length - c, s.length) for s, c in zip(sequences, counts)])
        for layer, cache in enumerate(self.caches):
            qkv = torch.randn(n, HEADS + 2 * KV_HEADS, DIM, generator=self.g).to(self.gpu)
            q, k, v = qkv.split([HEADS, KV_HEADS, KV_HEADS], 1)  # slices of one projection's rows
            keys = self.rotary.rotate(batch, k)
            turned = cache.write(batch, k, v, rotary=self.rotary, queries=q, out=torch.zeros(n, HEADS, DIM, device=self.gpu))
            check_turned(self.rotary, q.cpu(), positions, turned.cpu())
            check_turned(self.rotary, k.cpu(), positions, keys.cpu())
            out = cache.attend(batch, turned, prefixes=prefixes)
            for i, s in enumerate(sequences):
                a, b = starts[i], starts[i + 1]
                kept = s.stored[layer]
                kept[0].append(serving.quantized(keys[a:b].cpu()))
                kept[1].append(serving.quantized(v[a:b].cpu()))
                want, weighed, _ = serving.attention(turned[a:b], torch.cat(kept[0]), torch.cat(kept[1]), np.arange(s.length - (b - a), s.length), DIM ** -0.5)
                # the scores here are under 40: the bound of test_gpu_cache_attend.py
                assert bool(((out[a:b].cpu().double() - want).abs() <= weighed * 2.0 ** -24 * (2 * 40 * (DIM + 8) + 2 * s.length + 16) + 1e-9).all())
        return shared

    def fork(self, parent, count):
        """`count` more sequences that go on from `parent`, their partial pages copied in every layer by one call."""
        sources, targets, children = [], [], []
        for _ in range(count):
            child = self.Sequence()
            child.pages, copies = self.pages.fork(parent.pages, parent.length)
            sources += copies[0]
            targets += copies[1]
            child.length = parent.length
            child.stored = [([*k], [*v]) for k, v in parent.stored]
            children.append(child)
        self.fk.copy_pages(self.caches, sources, targets)
        return children

    def free(self, sequence):
        self.pages.free(sequence.pages)

    def compact(self, sequences):
        moves = self.pages.compact()
        self.fk.copy_pages(self.caches, list(moves), list(moves.values()))
        for s in sequences:
            s.pages = [moves.get(p, p) for p in s.pages]
        return moves


def check_turned(rotary, x, positions, got):
    from test_gpu_rotary import check
    check(rotary, x, positions, got)


def test_answers_from_one_prompt(fk, gpu):
    program = Program(fk, gpu, 90)
    prompt, other = program.Sequence(), program.Sequence()
    program.step([[prompt], [other]], [600, 70])
    answers = [prompt, *program.fork(prompt, 3)]  # 9 whole pages shared, the tenth copied
    for _ in range(3):
        shared = program.step([answers, [other]], [1] * 5)
        assert shared[0] == 9
    # each goes on for a page or more; one of them is forked in its turn
    program.step([answers, [other]], [70, 1, 65, 130, 1])
    branch = program.fork(answers[3], 2)
    late = program.step([[answers[3], *branch], answers[:3], [other]], [1] * 7)
    assert late[0] > 9 and late[1] == 9
    # some end; what is left moves to the lowest pages
    for s in (answers[0], answers[2], branch[0]):
        program.free(s)
    rest = [answers[1], answers[3], branch[1], other]
    used = program.pages.count - program.pages.free_pages
    moves = program.compact(rest)
    assert moves and max(max(s.pages) for s in rest) == used - 1
    for _ in range(2):
        program.step([[answers[3], branch[1]], [answers[1]], [other]], [1, 2, 1, 1])
    for s in rest:
        program.free(s)
    assert program.pages.free_pages == 90


def test_a_captured_step_replays(fk, gpu):
    """Turned write, attention over shared pages and the copy of a page in one graph, replayed with other inputs and
    lengths; eager steps between the replays, on another cache. Every replay is the eager step bit for bit."""
    import torch
    n = 24
    step = serving.Step([1] * n, [1290 + s for s in range(n)], extra_columns=1000, padding=1)
    g = torch.Generator().manual_seed(0)
    caches = [fk.PagedCache(step.pages + 2, KV_HEADS, DIM, device=gpu) for _ in range(2)]
    whole = step.whole()
    x = torch.randn(whole.total(), KV_HEADS, DIM, generator=g).to(gpu)
    for cache in caches:
        cache.write(whole.batch(fk, gpu), x, -x)  # (to pages of each sequence's own)
    step.table[:, :20] = step.table[0, :20]
    torch.cuda.synchronize()
    batch, rotary = step.batch(fk, gpu), fk.Rotary(DIM, layout="pairs", device=gpu)
    prefixes = fk.Prefixes(torch.tensor([0, n], dtype=torch.int32, device=gpu), torch.tensor([20], dtype=torch.int32, device=gpu))
    q, k, v = (torch.randn(n + 1, h, DIM, generator=g).to(gpu) for h in (HEADS, KV_HEADS, KV_HEADS))
    turned, out = torch.zeros_like(q), torch.zeros_like(q)
    sources, targets = (torch.tensor([p], dtype=torch.int32, device=gpu) for p in (int(step.table[3, 20]), step.pages))

    def run(cache):
        cache.write(batch, k, v, rotary=rotary, queries=q, out=turned)
        cache.attend(batch, turned, out=out, prefixes=prefixes)
        fk.copy_pages([cache], sources, targets)

    copied = fk.Batch(torch.tensor([0, 64], dtype=torch.int32, device=gpu), torch.tensor([64], dtype=torch.int32, device=gpu), targets.view(1, 1))
    for cache in caches:
        run(cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(caches[0])
    for replay in range(5):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        batch.lengths.copy_(torch.tensor([m - 2 * replay for m in step.lengths], dtype=torch.int32))
        turned.zero_(), out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = [turned.clone(), out.clone()] + [torch.zeros(64, KV_HEADS, DIM, device=gpu) for _ in range(2)]
        caches[0].read(copied, *got[2:])
        turned.zero_(), out.fill_(float("nan"))
        run(caches[1])
        want = [turned.clone(), out.clone()] + [torch.zeros(64, KV_HEADS, DIM, device=gpu) for _ in range(2)]
        caches[1].read(copied, *want[2:])
        for a, b in zip(got, want):
            assert torch.equal(a[:n], b[:n]) and not bool(torch.isnan(a[:n]).any())
        assert bool(torch.isnan(got[1][n:]).all())
    del graph
    torch.cuda.synchronize()
