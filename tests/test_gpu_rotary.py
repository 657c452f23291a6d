"""Rotary positions against 80-bit angles, and keys turned on their way into the cache.

Tolerance of a turned value a c - b s, e = 2^-24 (half a step of f32): c and s are rounded once (e of each) and carry the
angle's error, position * 2^-65 turns for the step's rounding and what 64 bits round, 2^-50 in all; the products e each, the
sum e of itself: 3 e (|a c| + |b s|), and (|a| + |b|) (position 2^-62 + 2^-50). Products under f32's normal range are
off by half its smallest step, 2^-150, each."""

import numpy as np
import pytest

import serving

pytestmark = pytest.mark.gpu
TWO_PI = np.longdouble("6.28318530717958647692528676655900577")


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


def positions_of(step):
    return np.concatenate([np.arange(n - r, n) for r, n in zip(step.rows, step.lengths)] + [np.zeros(0, int)]).astype(np.int64)


def check(rotary, x, positions, got):
    """[rows, heads, dim] f32 before and after, on the host."""
    x, got = x.double().numpy(), got.double().numpy()
    n = rotary.dims // 2
    first = np.arange(n) if rotary.layout == "halves" else np.arange(0, 2 * n, 2)
    second = first + n if rotary.layout == "halves" else first + 1
    angle = positions.astype(np.longdouble)[:, None] * np.array(rotary.frequencies, np.longdouble)
    angle = np.fmod(angle, TWO_PI)
    m = rotary.magnitude
    c, s = (m * np.cos(angle)).astype(np.float64)[:, None], (m * np.sin(angle)).astype(np.float64)[:, None]
    placed = positions >= 0
    a, b = x[..., first], x[..., second]
    slack = (np.abs(a) + np.abs(b)) * abs(m) * (np.maximum(positions, 0)[:, None, None] * 2.0 ** -62 + 2.0 ** -50) + 2.0 ** -148
    bound = 3 * 2.0 ** -24 * (np.abs(a * c) + np.abs(b * s)) + slack
    assert (np.abs(got[..., first] - (a * c - b * s)) <= bound)[placed].all()
    bound = 3 * 2.0 ** -24 * (np.abs(b * c) + np.abs(a * s)) + slack
    assert (np.abs(got[..., second] - (b * c + a * s)) <= bound)[placed].all()
    assert np.array_equal(got[placed][..., rotary.dims:], x[placed][..., rotary.dims:])
    assert not got[~placed].any()


STEPS = [([1], [1]), ([1, 1, 1], [64, 65, 2000]), ([1, 0, 1, 0], [7, 0, 200, 3]), ([70, 1], [70, 129]), ([33, 0, 128, 1], [161, 0, 128, 1]),
         ([700, 1, 1400], [701, 64, 1463]), ([3, 40], [2, 30])]
# heads, head_dim, values turned; whole quads of pairs and others
HEADS = [(14, 64, 64), (1, 4, 2), (5, 36, 36), (16, 72, 72), (3, 128, 128), (16, 128, 32), (2, 128, 40), (7, 96, 18), (3, 80, 78), (2, 256, 256),
         (1, 256, 2), (2, 256, 254), (70, 32, 32)]


@pytest.mark.parametrize("rows,lengths", STEPS)
@pytest.mark.parametrize("heads,dim,dims", HEADS)
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_rotate(fk, gpu, rows, lengths, heads, dim, dims, layout):
    import torch
    print(f"rotate {rows} {lengths} {heads}x{dim} {dims} {layout}", flush=True)
    rotary = fk.Rotary(dims, base=1e6, layout=layout)
    step = serving.Step(rows, lengths, padding=2)
    n = step.total() - 2
    x = torch.randn(n + 2, heads, dim, generator=torch.Generator().manual_seed(dims))
    batch, on = step.batch(fk, gpu), x.to(gpu)
    out = torch.full_like(on, 5.0)
    assert rotary.rotate(batch, on, out=out) is out and torch.equal(on.cpu(), x)
    check(rotary, x[:n], positions_of(step), out.cpu()[:n])
    assert bool((out[n:] == 5.0).all())
    made = rotary.rotate(batch, on)
    assert torch.equal(made[:n], out[:n]) and not bool(made[n:].any())
    rotary.rotate(batch, on, out=on)  # in place
    assert torch.equal(on[:n], out[:n]) and torch.equal(on[n:].cpu(), x[n:])


@pytest.mark.parametrize("where", [10 ** 6, 2 ** 24 + 7, 2 ** 31 - 2])
def test_far_positions(fk, gpu, where):
    import torch
    step = serving.Step([5], [40])
    step.lengths = [where + 1]
    batch = fk.Batch(torch.tensor([0, 5], dtype=torch.int32, device=gpu), torch.tensor([where + 1], dtype=torch.int32, device=gpu),
                     torch.zeros(1, 0, dtype=torch.int32, device=gpu))
    x = torch.randn(5, 3, 64, generator=torch.Generator().manual_seed(1))
    for options in ({"base": 1e4}, {"base": 5e5, "stretch": 8.0, "trained": 8192}, {"frequencies": np.linspace(-3.0, 3.0, 32)},
                    {"magnitude": 1.25}, {"stretch": 4.0, "magnitude": -0.5}):
        rotary = fk.Rotary(64, **options)
        check(rotary, x, positions_of(step), rotary.rotate(batch, x.to(gpu)).cpu())


def test_special_values(fk, gpu):
    """Infinities and NaN stay in their pairs, subnormal values keep their bits at position 0."""
    import torch
    rotary = fk.Rotary(32, layout="halves")
    x = torch.randn(3, 2, 32, generator=torch.Generator().manual_seed(2))
    x[1, 1, 3], x[2, 0, 20] = float("inf"), float("nan")
    x[0, 0, :4] = torch.tensor([1e-45, -3e-45, 2e-44, -0.0])
    step = serving.Step([3], [3])
    got = rotary.rotate(step.batch(fk, gpu), x.to(gpu)).cpu()
    assert torch.equal(got[0], x[0])
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[1, 1, [3, 19]] = bad[2, 0, [4, 20]] = True
    assert not bool(torch.isfinite(got[bad]).any()) and bool(torch.isfinite(got[~bad]).all())


def same(a, b):
    import torch
    return torch.equal(a.cpu().view(torch.int32), b.cpu().float().view(torch.int32))


@pytest.mark.parametrize("rows,lengths", STEPS + [([2050, 66, 0, 3], [2060, 200, 5, 3]), ([64 * 33], [64 * 33]), ([2100, 9], [2100, 1000])])
@pytest.mark.parametrize("heads,kv_heads,dim,dims", [(14, 2, 64, 64), (4, 1, 36, 36), (16, 4, 128, 64), (2, 2, 72, 18), (3, 1, 132, 132), (4, 2, 256, 250)])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
def test_turned_keys_in_the_cache(fk, gpu, rows, lengths, heads, kv_heads, dim, dims, layout):
    """Keys and queries as Rotary.rotate turns them, values as they are, bit for bit; nothing else in the cache changes."""
    import torch
    print(f"keep {rows} {lengths} {heads}/{kv_heads}x{dim} {dims} {layout}", flush=True)
    step = serving.Step(rows, lengths, seed=dim, padding=2)
    g = torch.Generator().manual_seed(dims)
    q, k, v = (torch.randn(step.total(), h, dim, generator=g).to(gpu) for h in (heads, kv_heads, kv_heads))
    rotary = fk.Rotary(dims, layout=layout)
    cache, plain = (fk.PagedCache(step.pages, kv_heads, dim, device=gpu) for _ in range(2))
    whole, batch = step.whole(), step.batch(fk, gpu)
    old = torch.randn(whole.total(), kv_heads, dim, generator=g).to(gpu)
    for c in (cache, plain):
        c.write(whole.batch(fk, gpu), old, -old)
    out = torch.full_like(q, 5.0)
    assert cache.write(batch, k, v, rotary=rotary, queries=q, out=out) is out
    n = int(step.starts[-1])
    turned_q, turned_k = rotary.rotate(batch, q), rotary.rotate(batch, k)
    assert same(out[:n], turned_q[:n]) and bool((out[n:] == 5.0).all())
    plain.write(batch, turned_k, v)
    every = [torch.full_like(old, float("nan")) for _ in range(4)]
    cache.read(whole.batch(fk, gpu), *every[:2])
    plain.read(whole.batch(fk, gpu), *every[2:])
    assert same(every[0], every[2]) and same(every[1], every[3])
    # keys alone; and queries in place
    again = fk.PagedCache(step.pages, kv_heads, dim, device=gpu)
    again.write(whole.batch(fk, gpu), old, -old)
    assert again.write(batch, k, v, rotary=rotary) is None
    again.read(whole.batch(fk, gpu), *every[2:])
    assert same(every[0], every[2]) and same(every[1], every[3])
    cache.write(batch, k, v, rotary=rotary, queries=q, out=q)
    assert same(q[:n], out[:n])


@pytest.mark.parametrize("rows,lengths", [([1, 1], [3, 70]), ([70], [70]), ([1100], [1111])])
@pytest.mark.parametrize("dims,layout", [(32, "halves"), (36, "pairs"), (30, "halves")])
def test_strides_and_unaligned_rows(fk, gpu, rows, lengths, dims, layout):
    """Slices of one projection's rows at an address of any float, one row for all, turned in place in the projection."""
    import torch
    step = serving.Step(rows, lengths)
    heads, kv_heads, dim, n = 4, 2, 36, sum(rows)
    width = (heads + 2 * kv_heads) * dim
    flat = torch.randn(n * (width + 7) + 1, generator=torch.Generator().manual_seed(5)).to(gpu)
    q, k, v = (flat.as_strided((n, h, dim), (width + 7, dim, 1), 1 + at * dim) for h, at in ((heads, 0), (kv_heads, heads), (kv_heads, heads + kv_heads)))
    before = flat.clone()
    rotary, batch = fk.Rotary(dims, layout=layout), step.batch(fk, gpu)
    want_q, want_k = rotary.rotate(batch, q.contiguous()), rotary.rotate(batch, k.contiguous())
    cache = fk.PagedCache(step.pages, kv_heads, dim, device=gpu)
    cache.write(batch, k, v, rotary=rotary, queries=q, out=q)
    got_k, got_v = torch.zeros_like(want_k), torch.zeros_like(want_k)
    cache.read(batch, got_k, got_v)
    assert same(q.contiguous(), want_q) and same(got_k, serving.quantized(want_k.cpu())) and same(got_v, serving.quantized(v.cpu()))
    q.copy_(before.as_strided(q.shape, q.stride(), 1))
    assert torch.equal(flat, before)  # nothing beside the queries changed
    one = q[:1].expand(n, heads, dim)
    check(rotary, one.cpu(), positions_of(step), rotary.rotate(batch, one).cpu())


def test_many_sequences_and_offsets_past_32_bits(fk, gpu):
    import torch
    rng = np.random.default_rng(3)
    rows = [int(r) if rng.random() < 0.6 else 0 for r in rng.integers(0, 9, 4300)]
    step = serving.Step(rows, [r + int(p) for r, p in zip(rows, rng.integers(0, 9, 4300))], padding=1)
    rotary = fk.Rotary(32)
    x = torch.randn(step.total(), 1, 32)
    n = int(step.starts[-1])
    check(rotary, x[:n], positions_of(step), rotary.rotate(step.batch(fk, gpu), x.to(gpu)).cpu()[:n])
    # the last of 70000 rows lies 4.4e9 values on
    count, stride = 70000, 64000
    step = serving.Step([count], [count])
    flat = torch.zeros(count * stride, device=gpu)  # 18 GB
    rows = flat.as_strided((count, 2, 64), (stride, 64, 1))
    rows.copy_(torch.randn(count, 2, 64))
    x = rows.cpu()
    out = fk.Rotary(64, layout="pairs").rotate(step.batch(fk, gpu), rows, out=rows)
    rotary = fk.Rotary(64, layout="pairs")
    check(rotary, x[-500:], np.arange(count - 500, count), out[-500:].cpu())


def test_replays_with_other_positions(fk, gpu):
    """A captured call reads the batch as it is at the replay."""
    import torch
    for rows, lengths in (([1, 1, 1], [64, 65, 130]), ([1100, 7], [1300, 200])):
        step = serving.Step(rows, lengths)
        g = torch.Generator().manual_seed(0)
        q, k, v = (torch.randn(step.total(), h, 64, generator=g).to(gpu) for h in (4, 2, 2))
        rotary, batch = fk.Rotary(64), step.batch(fk, gpu)
        cache, twin = (fk.PagedCache(step.pages, 2, 64, device=gpu) for _ in range(2))
        out, alone = torch.zeros_like(q), torch.zeros_like(q)
        cache.write(batch, k, v, rotary=rotary, queries=q, out=out)
        rotary.rotate(batch, q, out=alone)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.write(batch, k, v, rotary=rotary, queries=q, out=out)
            rotary.rotate(batch, q, out=alone)
        for replay in range(5):
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=g))
            batch.lengths.copy_(torch.tensor([max(r, n - replay) for r, n in zip(rows, lengths)], dtype=torch.int32))
            out.zero_(), alone.zero_()
            graph.replay()
            torch.cuda.synchronize()
            want = twin.write(batch, k, v, rotary=rotary, queries=q)
            reads = [torch.zeros_like(k) for _ in range(4)]
            cache.read(batch, *reads[:2])
            twin.read(batch, *reads[2:])
            assert torch.equal(out, want) and torch.equal(alone, want)
            assert torch.equal(reads[0], reads[2]) and torch.equal(reads[1], reads[3])
        del graph


def test_streams(fk, gpu):
    """Outputs made here belong to the given stream."""
    import torch
    step = serving.Step([1, 40], [64, 65])
    x = torch.randn(step.total(), 4, 64).to(gpu)
    rotary, batch = fk.Rotary(64), step.batch(fk, gpu)
    cache = fk.PagedCache(step.pages, 4, 64, device=gpu)
    want = rotary.rotate(batch, x).cpu()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        a = rotary.rotate(batch, x, stream=side)
        b = cache.write(batch, x, x, rotary=rotary, queries=x, stream=side)
        side.synchronize()
        assert torch.equal(a.cpu(), want) and torch.equal(b.cpu(), want)


def test_refusals(fk, gpu):
    import ctypes

    import torch
    from fusor_kernels import _lib
    step = serving.Step([2], [2])
    batch = step.batch(fk, gpu)
    rotary, cache = fk.Rotary(64), fk.PagedCache(step.pages, 2, 64, device=gpu)
    good = torch.zeros(2, 2, 64, device=gpu)
    for bad in (good.cpu(), good.double(), good[0], good.transpose(0, 2), good[..., ::2], torch.zeros(2, 2, 32, device=gpu),
                torch.zeros(2, 2, 66, device=gpu), torch.zeros(2, 2, 260, device=gpu), good[:, :0]):
        with pytest.raises(fk.ShapeError):
            rotary.rotate(batch, bad)
    for bad in (good.cpu(), good.double(), good[:1], good[:, :1], good[:1].expand(2, 2, 64)):
        with pytest.raises(fk.ShapeError):
            rotary.rotate(batch, good, out=bad)
        with pytest.raises(fk.ShapeError):
            cache.write(batch, good, good, rotary=rotary, queries=good, out=bad)
    for bad in (good[:1], good[..., :32], good[0], good.double(), good.cpu()):
        with pytest.raises(fk.ShapeError):
            cache.write(batch, good, good, rotary=rotary, queries=bad)
    with pytest.raises(fk.ShapeError):
        cache.write(batch, good, good, queries=good)
    with pytest.raises(fk.ShapeError):
        cache.write(batch, good, good, rotary=rotary, out=good)
    with pytest.raises(fk.ShapeError):
        cache.write(batch, good, good, rotary=fk.Rotary(66))
    wide = torch.zeros(2, 400, device=gpu)
    x, out = wide.as_strided((2, 2, 64), (200, 64, 1)), wide.as_strided((2, 2, 64), (300, 64, 1))
    with pytest.raises(fk.ShapeError, match="stride"):
        rotary.rotate(batch, x, out=out)  # over the rows with another stride
    device = ctypes.cast(rotary.handle, ctypes.POINTER(ctypes.c_int))  # the handle's first field
    assert device[0] == 0
    device[0] = 1
    try:
        for call in (lambda: rotary.rotate(batch, good), lambda: cache.write(batch, good, good, rotary=rotary)):
            with pytest.raises(ValueError, match="the rotary positions are on device 1"):
                call()
    finally:
        device[0] = 0
    none = _lib.FgBatch(1, 2, 1, None, None, None)
    assert _lib.lib().fg_rotary_rotate(rotary.handle, ctypes.byref(none), good.data_ptr(), 128, 2, 64, good.data_ptr(), 128, None) == _lib.FG_ERR_ARG
    assert rotary.rotate(batch, good[:0]).shape == (0, 2, 64)
