"""Sampling against its definition in 64 bits: tokens equal, chances to f32's rounding (2^-23: one
rounding of a quotient, and weights of 2^-45 of the largest)."""

import numpy as np
import pytest

import serving

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fk(gpu):
    import fusor_kernels
    return fusor_kernels


def run(fk, gpu, logits, random, **settings):
    import torch
    on = {k: torch.as_tensor(np.asarray(v, np.int32 if k == "top_k" else np.float32)).to(gpu) for k, v in settings.items()}
    tokens, chances = fk.sample(torch.as_tensor(logits).to(gpu), torch.as_tensor(np.asarray(random, np.float32)).to(gpu), **on)
    return tokens.cpu().numpy(), chances.cpu().numpy()


def check(fk, gpu, logits, random, **settings):
    tokens, chances = run(fk, gpu, logits, random, **settings)
    for row in range(len(logits)):
        options = {k: np.asarray(v, np.int32 if k == "top_k" else np.float32)[row] for k, v in settings.items()}
        token, chance = serving.draw(logits[row], np.float32(random[row]), **options)
        assert tokens[row] == token, (row, tokens[row], token, options, random[row])
        assert abs(chances[row] - chance) <= 2.0 ** -23 * chance + 2.0 ** -40, (row, options)
    return tokens, chances


def logits_of(rng, rows, vocab, spread=2.0):
    x = (spread * rng.standard_normal((rows, vocab))).astype(np.float32)
    for r in range(rows):
        likely = rng.integers(0, vocab, 12)
        x[r, likely] += rng.uniform(2, 9, 12).astype(np.float32)
    return x


VOCABS = [1, 2, 3, 63, 64, 257, 1000, 4095, 4097, 32003, 151936]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("kind", ["plain", "top_k", "top_p", "min_p", "all", "greedy"])
def test_draws(fk, gpu, vocab, kind):
    print(f"sample {vocab} {kind}", flush=True)
    rng = np.random.default_rng(vocab + len(kind))
    rows = 12 if vocab < 100000 else 6
    logits, random = logits_of(rng, rows, vocab), rng.random(rows)
    settings = {}
    if kind != "plain":
        settings["temperature"] = np.exp(rng.uniform(np.log(0.2), np.log(3.0), rows))
    if kind in ("top_k", "all"):
        settings["top_k"] = np.exp(rng.uniform(0, np.log(vocab + 2), rows)).astype(np.int32)
    if kind in ("top_p", "all"):
        settings["top_p"] = rng.uniform(0.02, 1.0, rows)
    if kind in ("min_p", "all"):
        settings["min_p"] = np.exp(rng.uniform(np.log(1e-4), 0, rows))
    if kind == "greedy":
        settings["temperature"] = np.array([0.0, -1.0] * (rows // 2))
    check(fk, gpu, logits, random, **settings)


@pytest.mark.parametrize("rows", [1, 3, 100, 700])
def test_rows(fk, gpu, rows):
    rng = np.random.default_rng(rows)
    logits = logits_of(rng, rows, 5003)
    check(fk, gpu, logits, rng.random(rows), temperature=rng.uniform(0.3, 1.5, rows), top_k=rng.integers(0, 80, rows),
          top_p=rng.uniform(0.5, 1.0, rows), min_p=rng.uniform(0, 0.1, rows))


def test_batches_past_the_cache(fk, gpu):
    """More rows than one batch of the kernels takes (192 MiB of logits), with settings a row each."""
    rng = np.random.default_rng(5)
    rows, vocab = 30, 2100007
    base = rng.standard_normal(vocab).astype(np.float32)
    logits = np.stack([np.roll(base, 1001 * r) for r in range(rows)])
    check(fk, gpu, logits, rng.random(rows), temperature=np.where(np.arange(rows) % 5 == 0, 0.0, 0.4),
          top_k=np.where(np.arange(rows) % 2, 50, 0), top_p=np.where(np.arange(rows) % 3, 0.9, 1.0))


@pytest.mark.parametrize("vocab", [10, 1000, 40000])
def test_ties(fk, gpu, vocab):
    """Equal logits: the lowest indices are kept; every random number's token."""
    rng = np.random.default_rng(vocab)
    rows = 40
    random = np.linspace(0, 1, rows, endpoint=False)
    equal = np.zeros((rows, vocab), np.float32)
    for k in (0, 1, 7, vocab - 1):
        check(fk, gpu, equal, random, top_k=np.full(rows, k))
    for p in (0.5, 0.25, 0.1):
        check(fk, gpu, equal, random, top_p=np.full(rows, p))
    few = rng.integers(0, 3, (rows, vocab)).astype(np.float32)
    few[:, ::5] = -0.0
    check(fk, gpu, few, random, top_k=rng.integers(1, vocab, rows), top_p=rng.uniform(0.1, 1, rows))
    check(fk, gpu, few, random, min_p=np.exp(rng.uniform(-3, 0, rows)))


@pytest.mark.parametrize("vocab", [5, 63, 64, 65, 127, 128, 129, 130, 6000])
@pytest.mark.parametrize("tied", [False, True])
def test_short_lists(fk, gpu, vocab, tied):
    """Lists of up to 64, up to 128 and more tokens, cut by one limit or several, in one place or apart."""
    rng = np.random.default_rng(vocab)
    rows = 60
    logits = (2 * rng.standard_normal((rows, vocab))).astype(np.float32)
    if tied:
        logits = np.round(logits * 2) / 2
    top_k = rng.integers(1, min(vocab, 140) + 1, rows)
    top_k[::7] = 0
    top_p = np.where(np.arange(rows) % 3 == 0, 1.0, rng.uniform(0.05, 0.999, rows))
    min_p = np.where(np.arange(rows) % 4 == 0, np.exp(rng.uniform(-6, 0, rows)), 0.0)
    check(fk, gpu, logits, rng.random(rows), temperature=np.exp(rng.uniform(-1, 1, rows)), top_k=top_k, top_p=top_p, min_p=min_p)
    check(fk, gpu, logits, np.linspace(0, 1, rows, endpoint=False), top_k=top_k)


def test_zeros_of_both_signs_are_equal(fk, gpu):
    logits = np.full((2, 300), -1.0, np.float32)
    logits[0, 100], logits[0, 200] = -0.0, 0.0
    logits[1, 100], logits[1, 200] = 0.0, -0.0
    tokens, _ = check(fk, gpu, logits, [0.5, 0.5], top_k=[1, 1])
    assert list(tokens) == [100, 100]
    check(fk, gpu, logits, [0.2, 0.7], top_k=[2, 2])


def test_special_logits(fk, gpu):
    inf, nan = np.inf, np.nan
    rng = np.random.default_rng(0)
    rows = [np.full(500, -inf), np.full(500, nan), np.where(np.arange(500) == 77, 1.0, -inf), rng.standard_normal(500),
            np.where(np.arange(500) % 100 == 3, inf, 0.0), rng.standard_normal(500) * 1e30, rng.standard_normal(500) * 1e-30,
            np.where(np.arange(500) == 9, 3.4e38, -3.4e38)]
    rows[3][::3] = nan
    rows[3][1::3] = -inf
    logits = np.stack(rows).astype(np.float32)
    n = len(rows)
    for random in (0.0, 0.4, 0.99999994):
        check(fk, gpu, logits, np.full(n, random))
        check(fk, gpu, logits, np.full(n, random), top_k=np.full(n, 3), top_p=np.full(n, 0.8), min_p=np.full(n, 0.01))
    tokens, chances = run(fk, gpu, logits, np.full(n, 0.5))
    assert list(tokens[:2]) == [-1, -1] and list(chances[:2]) == [0, 0]


def test_settings_at_their_ends(fk, gpu):
    rng = np.random.default_rng(2)
    logits = logits_of(rng, 1, 3000).repeat(10, 0)
    random, greedy = rng.random(10), np.argmax(logits[0])
    nan = np.nan
    assert all(run(fk, gpu, logits, random, temperature=[0, -0.0, -5, nan] + [1e-30] * 6)[0] == greedy)
    assert all(run(fk, gpu, logits, random, top_p=[0, -1, 1e-30] + [0.0] * 7)[0] == greedy)
    assert all(run(fk, gpu, logits, random, min_p=[1.0, 2.0, np.inf] + [1.0] * 7)[0] == greedy)
    free = check(fk, gpu, logits, random)[0]
    assert all(run(fk, gpu, logits, random, top_p=[1, 2, nan] + [1.0] * 7)[0] == free)
    assert all(run(fk, gpu, logits, random, min_p=[0, -1, nan] + [0.0] * 7)[0] == free)
    assert all(run(fk, gpu, logits, random, top_k=[0, -1, 3000, 3001, 2 ** 31 - 1] + [0] * 5)[0] == free)
    check(fk, gpu, logits, random, temperature=[1e30, np.inf, 1e-38, 100, 0.01] * 2)
    # random numbers at the ends, and outside
    first = run(fk, gpu, logits, [0.0, -1.0, nan] + [0.0] * 7)[0]
    assert all(first == first[0])
    last = run(fk, gpu, logits, [0.99999994, 1.0, 7.0] + [1.0] * 7, top_k=np.full(10, 5))[0]
    assert all(last == max(np.argsort(-logits[0], kind="stable")[:5]))


@pytest.mark.parametrize("spread", [0.0, 1e-4, 0.02, 40.0])
def test_dense_and_wide_rows(fk, gpu, spread):
    """Logits so close that a cut's bin holds more tokens than the list (they are found in the row
    again), or so wide that hardly any has company."""
    rng = np.random.default_rng(7)
    logits = (spread * rng.standard_normal((6, 60000))).astype(np.float32)
    check(fk, gpu, logits, rng.random(6), top_k=[0, 100, 30000, 59999, 4000, 0], top_p=[0.5, 1.0, 0.9, 0.3, 0.01, 0.999])
    check(fk, gpu, logits, rng.random(6), top_k=[20000] * 6, min_p=[0.5, 0.9, 0.999, 1e-3, 0, 1.0])


def test_strides_outputs_and_repeats(fk, gpu):
    import torch
    rng = np.random.default_rng(1)
    wide = torch.from_numpy(logits_of(rng, 9, 5000)).to(gpu)
    logits = wide[:, 1:4002]  # rows of a wider head, at an address of any float
    random = torch.rand(9, device=gpu)
    tokens, chances = torch.full((9,), -7, dtype=torch.int32, device=gpu), torch.zeros(9, device=gpu)
    back = fk.sample(logits, random, tokens=tokens, chances=chances)
    assert back[0] is tokens and back[1] is chances
    again = fk.sample(logits.contiguous(), random)
    assert torch.equal(tokens, again[0]) and torch.equal(chances, again[1])
    check(fk, gpu, logits.cpu().numpy(), random.cpu().numpy())
    one = fk.sample(logits[:1].expand(9, 4001), random)  # one row, nine random numbers
    for r in range(9):
        assert int(one[0][r]) == serving.draw(logits[0].cpu().numpy(), random[r].item())[0]


def test_refusals(fk, gpu):
    import torch
    logits, random = torch.zeros(3, 10, device=gpu), torch.zeros(3, device=gpu)
    for bad in (logits.cpu(), logits.half(), logits[0], logits.T, logits[:, ::2]):
        with pytest.raises(fk.ShapeError):
            fk.sample(bad, random)
    for bad in (random.cpu(), random.double(), random[:2], torch.zeros(6, device=gpu)[::2], torch.zeros(3, 1, device=gpu)):
        with pytest.raises(fk.ShapeError):
            fk.sample(logits, bad)
        with pytest.raises(fk.ShapeError):
            fk.sample(logits, random, top_p=bad)
    with pytest.raises(fk.ShapeError):
        fk.sample(logits, random, top_k=random)
    with pytest.raises(fk.ShapeError):
        fk.sample(logits, random, tokens=random)
    with pytest.raises(fk.ShapeError):
        fk.sample(logits[:, :0], random)
    tokens, chances = fk.sample(logits[:0], random[:0])
    assert tokens.shape == (0,) and chances.shape == (0,)
