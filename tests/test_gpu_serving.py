"""The serving operators as a program uses them: steps of several sequences through cache, attention and
sampling, captured in HIP graphs, on several streams and threads at once, with the program's scratch
or the library's."""

import ctypes
import threading

import numpy as np
import pytest

import serving

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


def check_tokens(logits, random, settings, tokens, chances):
    logits, random, tokens, chances = (t.cpu().numpy() for t in (logits, random, tokens, chances))
    settings = {k: v.cpu().numpy() for k, v in settings.items()}
    for r in range(len(tokens)):
        token, chance = serving.draw(logits[r], random[r], **{k: v[r] for k, v in settings.items()})
        assert tokens[r] == token and abs(chances[r] - chance) <= 2.0 ** -23 * chance + 2.0 ** -40


def test_sequences_from_prompts_to_tokens(fk, gpu):
    """Two layers' caches over one page table: prompts of several lengths read together, one in two
    chunks, then decode steps in which a sequence ends and another takes its pages. Every stage is
    checked against 64 bits on the inputs that it got."""
    import torch
    g = torch.Generator().manual_seed(11)
    heads, kv_heads, dim, hidden, vocab = 4, 2, 64, 256, 1000
    pages, columns = 24, 5
    width = (heads + 2 * kv_heads) * dim
    embed = torch.randn(vocab, hidden, generator=g).to(gpu)

    def table(rows, cols):
        return fk.Table(fk.Tensor.encode(fk.DType.Q8b32, [rows, cols], (torch.randn(rows * cols, generator=g) / cols ** 0.5).numpy()))

    layers = [(table(width, hidden), table(hidden, heads * dim), fk.PagedCache(pages, kv_heads, dim, device=gpu)) for _ in range(2)]
    head = table(vocab, hidden)
    free = list(range(pages))
    stored = {}  # (layer, sequence): the keys and values written so far, as the cache holds them

    class Sequence:
        def __init__(self, name, prompt):
            self.name, self.waiting, self.length, self.pages = name, list(prompt), 0, []

    def step(sequences, counts):
        ids, lengths, rows = [], [], []
        for s, n in zip(sequences, counts):
            ids += s.waiting[:n]
            del s.waiting[:n]
            s.length += n
            while len(s.pages) * 64 < s.length:
                s.pages.append(free.pop())
            lengths.append(s.length)
            rows.append(n)
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        paged = np.full((len(sequences), columns), -1, np.int32)
        for i, s in enumerate(sequences):
            paged[i, :len(s.pages)] = s.pages
        batch = fk.Batch(torch.from_numpy(starts).to(gpu), torch.tensor(lengths, dtype=torch.int32, device=gpu), torch.from_numpy(paged).to(gpu))
        n = len(ids)
        x = embed[torch.tensor(ids, device=gpu)]
        for index, (qkv_table, out_table, cache) in enumerate(layers):
            qkv = fk.matmul(qkv_table.matrix(), fk.Input(f32=x.reshape(-1)), range(0, width)).view(n, -1, dim)
            q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)  # slices of one projection's rows
            cache.write(batch, k, v)
            o = cache.attend(batch, q)
            for i, s in enumerate(sequences):
                a, b = starts[i], starts[i + 1]
                kept = stored.setdefault((index, s.name), ([], []))
                kept[0].append(serving.quantized(k[a:b].cpu()))
                kept[1].append(serving.quantized(v[a:b].cpu()))
                want, weighed, _ = serving.attention(q[a:b], torch.cat(kept[0]), torch.cat(kept[1]), np.arange(s.length - (b - a), s.length), dim ** -0.5)
                # the scores here are under 40 and the sums of at most 260 keys: the bound of test_gpu_cache_attend.py
                assert bool(((o[a:b].cpu().double() - want).abs() <= weighed * 2.0 ** -24 * (2 * 40 * (dim + 8) + 2 * 260 + 16) + 1e-9).all())
            x = x + fk.matmul(out_table.matrix(), fk.Input(f32=o.reshape(-1)), range(0, hidden))
            x = x / x.square().mean(-1, keepdim=True).sqrt()
        last = x[torch.from_numpy(starts[1:] - 1).to(gpu).long()]
        logits = 3 * fk.matmul(head.matrix(), fk.Input(f32=last.reshape(-1).contiguous()), range(0, vocab))
        random = torch.rand(len(sequences), generator=g).to(gpu)
        settings = {"temperature": torch.linspace(0.5, 1.2, len(sequences), device=gpu), "top_k": torch.full((len(sequences),), 40, dtype=torch.int32, device=gpu),
                    "top_p": torch.full((len(sequences),), 0.9, device=gpu)}
        tokens, chances = fk.sample(logits, random, **settings)
        check_tokens(logits, random, settings, tokens, chances)
        for s, token in zip(sequences, tokens.tolist()):
            if not s.waiting:
                s.waiting = [token]
        return tokens

    rng = np.random.default_rng(0)
    a, b, c = (Sequence(name, rng.integers(0, vocab, n)) for name, n in (("a", 200), ("b", 1), ("c", 63)))
    step([a, b, c], [130, 1, 63])  # a in two chunks
    step([a, b, c], [70, 1, 1])
    for _ in range(3):
        step([a, b, c], [1, 1, 1])
    free.extend(b.pages)  # b ends; d takes its pages
    d = Sequence("d", rng.integers(0, vocab, 90))
    step([a, c, d], [1, 1, 90])
    for _ in range(2):
        step([a, c, d], [1, 1, 1])


class Step:
    """A step's static buffers, as a program that replays graphs keeps them."""

    def __init__(self, fk, gpu, rows, lengths, heads=8, kv_heads=2, dim=64, vocab=2000, seed=0):
        import torch
        self.fk, self.gpu = fk, gpu
        self.step = serving.Step(rows, lengths, seed=seed, padding=1)
        g = torch.Generator().manual_seed(seed)
        n = self.step.total()
        self.batch = self.step.batch(fk, gpu)
        self.k, self.v, self.q = (torch.randn(n, h, dim, generator=g).to(gpu) for h in (kv_heads, kv_heads, heads))
        self.out = torch.zeros_like(self.q)
        self.logits = (2 * torch.randn(len(rows), vocab, generator=g)).to(gpu)
        self.random = torch.rand(len(rows), generator=g).to(gpu)
        self.top_p = torch.full((len(rows),), 0.8, device=gpu)
        self.tokens = torch.zeros(len(rows), dtype=torch.int32, device=gpu)
        self.chances = torch.zeros(len(rows), device=gpu)

    def new_cache(self, kv_heads=2, dim=64):
        import torch
        cache = self.fk.PagedCache(self.step.pages, kv_heads, dim, device=self.gpu)
        whole = self.step.whole()
        g = torch.Generator().manual_seed(99)
        x = torch.randn(whole.total(), kv_heads, dim, generator=g).to(self.gpu)
        cache.write(whole.batch(self.fk, self.gpu), x, -x)
        return cache

    def run(self, cache, stream=None):
        cache.write(self.batch, self.k, self.v, stream=stream)
        cache.attend(self.batch, self.q, out=self.out, stream=stream)
        self.fk.sample(self.logits, self.random, top_p=self.top_p, tokens=self.tokens, chances=self.chances, stream=stream)

    def results(self):
        return self.out.cpu(), self.tokens.cpu(), self.chances.cpu()


def equal(a, b):
    import torch
    return all(torch.equal(x, y) for x, y in zip(a, b))


# few rows over long caches (split over workgroups), many rows, single tokens of many sequences
SHAPES = [([1, 1], [2500, 1700], 151936), ([150, 1, 40], [400, 2200, 40], 500), ([1] * 70, [40 + s for s in range(70)], 3000)]


@pytest.mark.parametrize("rows,lengths,vocab", SHAPES)
@pytest.mark.parametrize("own_scratch", [True, False])
def test_a_captured_step_replays_with_new_sequences(fk, gpu, rows, lengths, vocab, own_scratch, monkeypatch):
    """A graph of one step, replayed with other inputs, lengths and pages in its buffers; eager steps and
    synchronizations between the replays. Every replay is the eager step bit for bit. Without the program's
    scratch the library's belongs to the graph."""
    import torch
    from fusor_kernels import serving as module
    print(f"graph {rows} {lengths} {own_scratch}", flush=True)
    if not own_scratch:
        monkeypatch.setattr(module, "_scratch", lambda size, device: None)
    s = Step(fk, gpu, rows, lengths, vocab=vocab)
    cache, twin = s.new_cache(), s.new_cache()
    s.run(cache)  # once before the capture: kernels loaded, pools warm
    s.run(twin)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run(cache)
    other = Step(fk, gpu, [3, 1], [70, 900], seed=5)
    other_cache = other.new_cache()
    for replay in range(5):
        g = torch.Generator().manual_seed(replay)
        for t in (s.k, s.v, s.q, s.logits):
            t.copy_(torch.randn(t.shape, generator=g))
        s.random.copy_(torch.rand(s.random.shape, generator=g))
        # other lengths: every sequence loses `replay` tokens (but not its new ones); pages in another order
        s.batch.lengths.copy_(torch.tensor([max(r, n - replay) for r, n in zip(rows, lengths)], dtype=torch.int32))
        s.batch.pages.copy_(torch.from_numpy(np.where(s.step.table < 0, -1, (s.step.table + replay) % s.step.pages)))
        s.out.fill_(float("nan")), s.tokens.fill_(-9), s.chances.fill_(-9)
        graph.replay()
        torch.cuda.synchronize()
        got = s.results()
        s.out.fill_(float("nan")), s.tokens.fill_(-9), s.chances.fill_(-9)
        s.run(twin)
        want = s.results()
        n = int(s.step.starts[-1])
        assert torch.equal(got[0][:n], want[0][:n]) and not bool(torch.isnan(got[0][:n]).any()), replay
        assert bool(torch.isnan(got[0][n:]).all()) and equal(got[1:], want[1:]), replay
        other.run(other_cache)
        torch.cuda.synchronize()
    del graph
    torch.cuda.synchronize()
    s.run(twin)  # frees what the graph's scratch was
    assert equal([t[:n] for t in s.results()[:1]], [want[0][:n]])


def test_streams_and_threads_at_once(fk, gpu):
    """Steps on streams of their own from threads of their own, all on one cache (pages apart): each as alone."""
    import torch
    steps = [Step(fk, gpu, *shape[:2], vocab=shape[2], seed=i) for i, shape in enumerate(SHAPES)]
    steps.append(Step(fk, gpu, [1, 5, 9], [900, 70, 800], vocab=151936, seed=7))
    total = sum(s.step.pages for s in steps)
    base = 0
    for s in steps:  # pages of one large cache, apart
        table = np.where(s.step.table < 0, -1, s.step.table + base).astype(np.int32)
        s.batch = fk.Batch(s.batch.row_starts, s.batch.lengths, torch.from_numpy(table).to(gpu))
        base += s.step.pages
    cache = fk.PagedCache(total, 2, 64, device=gpu)
    alone = []
    for s in steps:
        s.run(cache)
        torch.cuda.synchronize()
        alone.append(s.results())
        s.out.zero_(), s.tokens.zero_(), s.chances.zero_()
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            for _ in range(6):
                steps[i].run(cache, stream=streams[i])
            streams[i].synchronize()
        except Exception as error:  # shown by the main thread
            errors.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(steps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for s, want in zip(steps, alone):
        assert equal(s.results(), want)


def test_outputs_made_here_belong_to_the_given_stream(fk, gpu):
    """attend and sample that make their own outputs, on a stream that is not the current one."""
    import torch
    s = Step(fk, gpu, [1, 1], [2500, 1700])
    cache = s.new_cache()
    s.run(cache)
    torch.cuda.synchronize()
    want = s.results()
    side = torch.cuda.Stream()
    for _ in range(3):
        out = cache.attend(s.batch, s.q, stream=side)
        tokens, chances = fk.sample(s.logits, s.random, top_p=s.top_p, stream=side)
        side.synchronize()
        assert equal((out.cpu(), tokens.cpu(), chances.cpu()), want)


def test_scratch_of_the_program(fk, gpu):
    """Through the C ABI: scratch that is too small, or not aligned, is refused; none and enough agree."""
    import torch
    from fusor_kernels import _lib
    lib = _lib.lib()
    s = Step(fk, gpu, [1, 1], [2500, 1700], vocab=151936)
    cache = s.new_cache()
    s.run(cache)
    torch.cuda.synchronize()
    want = s.results()
    batch = s.batch._ffi(s.q.shape[0])
    size = lib.fg_cache_attend_scratch(cache.handle, ctypes.byref(batch), 8)
    room = lib.fg_sample_scratch(2, 151936)
    assert size > 0 and room > 0
    memory = torch.zeros(max(size, room) + 16, dtype=torch.uint8, device=gpu)

    def attend(scratch, bytes_):
        return lib.fg_cache_attend(cache.handle, ctypes.byref(batch), _lib.ptr(s.q), s.q.stride(0), 8, 0.125, 0, _lib.ptr(s.out),
                                   s.out.stride(0), scratch, bytes_, _lib.stream_handle())

    settings = _lib.FgSampling(_lib.ptr(s.random), None, None, _lib.ptr(s.top_p), None)

    def draw(scratch, bytes_):
        return lib.fg_sample(_lib.ptr(s.logits), 2, 151936, s.logits.stride(0), ctypes.byref(settings), _lib.ptr(s.tokens),
                             _lib.ptr(s.chances), scratch, bytes_, _lib.stream_handle())

    at = memory.data_ptr()
    for call, bytes_ in ((attend, size), (draw, room)):
        assert call(ctypes.c_void_p(at), bytes_ - 1) == _lib.FG_ERR_SHAPE and "scratch" in lib.fg_last_error().decode()
        assert call(ctypes.c_void_p(at + 4), bytes_) == _lib.FG_ERR_SHAPE
    for scratch in (None, ctypes.c_void_p(at)):
        s.out.zero_(), s.tokens.zero_(), s.chances.zero_()
        assert attend(scratch, size) == _lib.FG_OK and draw(scratch, room) == _lib.FG_OK
        assert equal(s.results(), want)


def test_a_cache_on_another_device_is_refused(fk, gpu, monkeypatch):
    """The Python calls make the cache's device current; the C calls refuse another one. (A handle that
    says it is on device 1 stands for that: nothing is launched.)"""
    from fusor_kernels import _lib
    s = Step(fk, gpu, [1], [70])
    cache = s.new_cache()
    device = ctypes.cast(cache.handle, ctypes.POINTER(ctypes.c_int))  # the handle's first field
    assert device[0] == 0
    device[0] = 1
    try:
        with pytest.raises(ValueError, match="the cache is on device 1"):
            cache.attend(s.batch, s.q, out=s.out)
        with pytest.raises(ValueError, match="the cache is on device 1"):
            cache.write(s.batch, s.k, s.v)
    finally:
        device[0] = 0
