"""The block cache, its attention and its eviction in 64-bit numpy, and the device's tensors in the entries' types."""
import numpy as np
import torch

BLOCK = 16
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_STEP = {t: torch.finfo(d).eps / 2 for t, d in TYPES.items()}


def typed(x, t):
    """x rounded to the type: (its bytes as the device holds them, its values in 64 bits)."""
    y = torch.from_numpy(np.ascontiguousarray(x, np.float64)).to(TYPES[t])
    return y.view(torch.uint8).numpy(), y.double().numpy()


def values_of(raw, t, shape):
    """The device's bytes as 64-bit values."""
    return torch.from_numpy(np.ascontiguousarray(raw, np.uint8).reshape(-1)).view(TYPES[t]).double().numpy().reshape(shape)


def scale_of(amax):
    """The smallest 2^e, e >= -100, with amax <= 127 * 2^e, for an array."""
    m, e = np.frexp(amax)
    return np.ldexp(1.0, np.maximum(e - 7 + (m > 127 / 128), -100))


class Page:
    """One (sequence, layer, key/value head): codes [tokens][dim] and a scale per block, in the sequence's order."""

    def __init__(self, capacity, dim):
        self.codes = [np.zeros((capacity, dim)) for _ in "kv"]
        self.scales = [np.zeros(capacity // BLOCK) for _ in "kv"]

    def append(self, at, k, v):
        for codes, scales, x in zip(self.codes, self.scales, (k, v)):
            for blk in range(at // BLOCK, (at + len(x) - 1) // BLOCK + 1):
                lo, hi = max(at, blk * BLOCK), min(at + len(x), (blk + 1) * BLOCK)
                rows = x[lo - at:hi - at]
                if not (np.abs(rows) <= 127 * 2.0 ** 120).all():
                    scales[blk] = np.nan
                    continue
                s = scale_of(np.abs(rows).max())
                if lo > blk * BLOCK and not s > scales[blk]:
                    s = scales[blk]
                elif lo > blk * BLOCK:
                    held = slice(blk * BLOCK, lo)
                    codes[held] = np.rint(codes[held] * (scales[blk] / s))
                if np.isnan(s):
                    continue
                scales[blk] = s
                codes[lo:hi] = np.rint(rows / s)

    def values(self, n):
        return [c[:n] * np.repeat(s, BLOCK)[:n, None] for c, s in zip(self.codes, self.scales)]

    def reorder(self, order):
        """Blocks by former index; the rest stays behind them."""
        nb = len(self.scales[0])
        order = list(order) + [i for i in range(nb) if i not in set(order)]
        for i in range(2):
            self.codes[i] = self.codes[i].reshape(nb, BLOCK, -1)[order].reshape(nb * BLOCK, -1)
            self.scales[i] = self.scales[i][order]


def attention(page, q, at, scale):
    """q [rows of one query head: n][dim] over tokens [0, at + i]: out [n][dim], block weights, S, the largest sum of
    |q k| scale log2(e), which the scores' rounding goes by, and the same with the largest |q| for each."""
    n, dim = q.shape
    k, v = page.values(at + n)
    out, s_max, q_max = np.zeros((n, dim)), 0.0, 0.0
    weights = np.zeros(len(page.scales[0]))
    for i in range(n):
        t = at + i + 1
        s = k[:t] @ q[i] * scale
        with np.errstate(all="ignore"):
            p = np.exp(s - s.max())
            p /= p.sum()
        out[i] = p @ v[:t]
        weights += np.add.reduceat(np.pad(p, (0, len(weights) * BLOCK - t)), np.arange(0, len(weights) * BLOCK, BLOCK))
        s_max = max(s_max, np.nanmax(np.abs(k[:t]) @ np.abs(q[i])) * abs(scale) * np.log2(np.e))
        q_max = max(q_max, np.abs(q[i]).max() * np.nanmax(np.abs(k[:t]).sum(1)) * abs(scale) * np.log2(np.e))
    return out, weights, s_max, q_max


def relative_bound(s_max, tokens):
    """What a softmax weight of the device may be off, relatively.  A score's byte sums are exact; their two halves,
    the sum, the two scales and the difference to the maximum round six times by 2^-24 of at most S (in log2, so
    times ln 2 in the weight); exp2 and the factors that join tiles, waves and splits are good for 16 * 2^-24; and
    a sum of T weights takes T / 64 + 24 additions along one path."""
    return (np.log(2) * 6 * s_max + tokens / 64 + 40) * 2.0 ** -24


def prompt_bound(s_max, q_max, tokens, t):
    """The same where a call has more than 16 rows and no weights, and (half floats' rounding of a weight).  Products
    of half floats and codes are exact in FP32; a score is a sum of 128 in an order of the instruction's (127
    roundings by 2^-24 of S at most) times scales (3); a query's half floats leave 2^-24 of its largest value.  Sums
    over T tokens round T + 64 times at most.  A weight is one half float, 2^-12 of it, or for FP32 two, 2^-22."""
    rel = (np.log(2) * (130 * s_max + q_max) + tokens + 64) * 2.0 ** -24
    return rel, 2.0 ** -22 if t == "f32" else 2.0 ** -12


def evict(weights, held, keep, sinks, recent):
    """Former indices of the blocks that stay."""
    if held <= keep:
        return list(range(held))
    w = np.where(weights[:held] > 0, weights[:held], 0)
    middle = sorted(range(sinks, held - recent), key=lambda i: (-w[i], i))[:keep - sinks - recent]
    return sorted(list(range(sinks)) + middle + list(range(held - recent, held)))
