"""Plain 64-bit forms of the serving operators and what their tests share."""

import numpy as np
import torch

PAGE = 64


def quantized(x):
    """Keys or values [..., dim] on their 8-bit grid, in 64 bits: one scale a head, f32 arithmetic by
    definition (a 64-bit quotient of f32 numbers rounded to 32 is the f32 quotient)."""
    x = x.double()
    finite = torch.where(torch.isnan(x), torch.zeros_like(x), x)
    scale = (finite.abs().amax(-1, keepdim=True) / 127).float().double()
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    level = (x / scale).float().double().round().clamp(-127, 127) + 0.0  # whole numbers: no -0
    return torch.where(torch.isnan(level), torch.zeros_like(level), level) * scale


class Step:
    """A step's sequences on the host: new rows and lengths, pages drawn without repeats."""

    def __init__(self, rows, lengths, seed=0, spare=3, extra_columns=1, padding=0):
        rng = np.random.default_rng(seed)
        self.rows, self.lengths, self.padding = list(rows), list(lengths), padding
        counts = [-(-n // PAGE) for n in self.lengths]
        self.pages = sum(counts) + spare
        ids = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((len(self.rows), max(counts, default=0) + extra_columns), -1, np.int32)
        at = 0
        for s, n in enumerate(counts):
            self.table[s, :n] = ids[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32)

    def total(self):
        return int(self.starts[-1]) + self.padding

    def batch(self, fk, device):
        return fk.Batch(torch.from_numpy(self.starts).to(device), torch.tensor(self.lengths, dtype=torch.int32, device=device),
                        torch.from_numpy(self.table).to(device))

    def whole(self):
        """The same sequences with every token new."""
        step = Step([0], [0])
        step.rows, step.lengths, step.padding, step.pages, step.table = self.lengths, self.lengths, 0, self.pages, self.table
        step.starts = np.concatenate([[0], np.cumsum(step.rows)]).astype(np.int32)
        return step


def attention(query, keys, values, positions, scale, window=0, absent=None):
    """One sequence in 64 bits: query [rows, heads, dim] at `positions`, keys and values [tokens,
    kv_heads, dim] as the cache holds them; tokens where `absent` hold nothing. Returns the outputs, the
    sums of |weight * value| and each row's and head's largest |weight * value|."""
    query, keys, values = query.double().cpu(), keys.double().cpu(), values.double().cpu()
    rows, heads, dim = query.shape
    group = heads // keys.shape[1]
    out = torch.zeros(rows, heads, dim, dtype=torch.float64)
    weighed, largest = out.clone(), torch.zeros(rows, heads, dtype=torch.float64)
    at = torch.arange(keys.shape[0])
    for r in range(rows):
        p = int(positions[r])
        seen = at <= p
        if window:
            seen &= at > p - window
        if absent is not None:
            seen &= ~absent
        if not bool(seen.any()):
            continue
        k, v = keys[seen], values[seen]
        for h in range(heads):
            s = (k[:, h // group] * query[r, h]).sum(-1) * scale
            w = torch.exp(s - s.max())
            x = w[:, None] / w.sum() * v[:, h // group]
            out[r, h], weighed[r, h], largest[r, h] = x.sum(0), x.abs().sum(0), x.abs().max()
    return out, weighed, largest


def draw(logits, random, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row's token and chance, by the definition in 64 bits."""
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, x) + 0.0
    if x.max() == -np.inf:
        return -1, 0.0
    order = np.argsort(-x, kind="stable")
    if not temperature > 0:
        return int(order[0]), 1.0
    with np.errstate(invalid="ignore", over="ignore"):
        z = np.where(x == x.max(), 0.0, (x - x.max()) / np.float64(temperature))
    w = np.where(x == -np.inf, 0.0, np.exp(z))
    kept = order if top_k <= 0 else order[:top_k]
    if top_p < 1:
        running = np.cumsum(w[kept])
        kept = kept[:max(1, int((running < top_p * running[-1]).sum()) + 1)]
    if min_p > 0:
        first = kept[:1]
        kept = kept[w[kept] >= min_p]
        kept = kept if len(kept) else first
    kept = np.sort(kept)
    running = np.cumsum(w[kept])
    i = min(int((running <= np.float64(random) * running[-1]).sum()), len(kept) - 1)
    return int(kept[i]), float(w[kept[i]] / running[-1])
