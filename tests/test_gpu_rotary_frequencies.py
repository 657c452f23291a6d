"""Rotary positions of whole turns a token: frequencies up to the largest that is taken, near and far, against angles from
whole numbers.

The reference's turns, position * frequency * 2^256 / (2 pi), are exact to 2^-200; their fraction is rounded to 64 bits once,
its cosine and sine to 64. The tolerance is test_gpu_rotary.py's: 3 e (|a c| + |b s|), and (|a| + |b|) (position 2^-62 +
2^-50), of which the angle takes position 2^-65 * 2 pi for the step's half bit and 2^-50 for what 64 bits round."""

import numpy as np
import pytest

import serving
from test_gpu_rotary import positions_of
from test_rotary_phase import TURN_BITS, TWO_PI

pytestmark = pytest.mark.gpu

FREQUENCIES = [1023.9, 777.7, 1024.0, -1023.9, 1000.0 / 3, 2 * np.pi, 100.0, 6.3]


@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("length", [40, 2 ** 20, 2 ** 31 - 1])
def test_whole_turns_a_token(gpu, layout, length):
    import torch
    import fusor_kernels as fk
    rows, dims = 33, 2 * len(FREQUENCIES)
    rotary = fk.Rotary(dims, layout=layout, frequencies=FREQUENCIES)
    step = serving.Step([rows], [rows])
    step.lengths = [length]
    batch = fk.Batch(torch.tensor([0, rows], dtype=torch.int32, device=gpu), torch.tensor([length], dtype=torch.int32, device=gpu),
                     torch.zeros(1, 0, dtype=torch.int32, device=gpu))
    x = torch.randn(rows, 3, dims + 4, generator=torch.Generator().manual_seed(length % 1000))
    got, x = rotary.rotate(batch, x.to(gpu)).cpu().double().numpy(), x.double().numpy()
    positions = positions_of(step)
    angle = np.zeros((rows, len(FREQUENCIES)), np.longdouble)
    for r, p in enumerate(positions):
        for i, f in enumerate(FREQUENCIES):
            n, d = float(f).as_integer_ratio()
            fraction = int(p) * n * TURN_BITS // d % 2 ** 256 >> 192
            angle[r, i] = np.longdouble(fraction) / np.longdouble(2.0 ** 64) * TWO_PI
    c, s = np.cos(angle).astype(np.float64)[:, None], np.sin(angle).astype(np.float64)[:, None]
    n = len(FREQUENCIES)
    first = np.arange(n) if layout == "halves" else np.arange(0, 2 * n, 2)
    second = first + n if layout == "halves" else first + 1
    a, b = x[..., first], x[..., second]
    slack = (np.abs(a) + np.abs(b)) * (positions[:, None, None] * 2.0 ** -62 + 2.0 ** -50) + 2.0 ** -148
    for dims_of, want, sizes in ((first, a * c - b * s, np.abs(a * c) + np.abs(b * s)), (second, b * c + a * s, np.abs(b * c) + np.abs(a * s))):
        error, bound = np.abs(got[..., dims_of] - want), 3 * 2.0 ** -24 * sizes + slack
        print(f"  {layout} {length}: {float((error / bound).max()):.3f} of the bound", flush=True)
        assert (error <= bound).all()
    assert np.array_equal(got[..., dims:], x[..., dims:])
