"""The paged cache in 64-bit numpy: rotated appends, trees, attention, kept paths; and a cache on the device fed the same."""
import numpy as np

import block_ref as R

PAGE = 64
NONE = -2


def random_tree(rng, n, count=None, deep=0.5):
    """Parents of `count` of n tokens: the token before, with probability `deep`, or any earlier one or the root."""
    count = n if count is None else count
    return [-1 if i == 0 else (i - 1 if rng.random() < deep else int(rng.integers(-1, i))) for i in range(count)] + \
        [NONE] * (n - count)


def chain(n):
    return list(range(-1, n - 1))


def places(parents):
    """Of each token: what it sees of the call [n][n], its depth, whether it is one."""
    n = len(parents)
    seen, depth = np.zeros((n, n), bool), np.zeros(n, int)
    for i, p in enumerate(parents):
        if p == NONE:
            continue
        if p >= 0:
            seen[i] = seen[p]
            depth[i] = depth[p] + 1
        seen[i, i] = True
    return seen, depth, np.array([p != NONE for p in parents], bool)


class Rotation:
    """The device's rotation: cos and sin computed in 64 bits and kept as FP32; a c - b s and b c + a s, the sine's product
    rounded to FP32 and then a fused multiply-add, then one rounding to the type."""

    def __init__(self, rotary_dim, positions=4096, theta=10000.0, halves=True):
        self.dim, self.positions, self.theta, self.halves = rotary_dim, positions, theta, halves
        f = theta ** (-np.arange(rotary_dim // 2) / (rotary_dim // 2))
        angle = np.arange(positions)[:, None] * f
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)

    def table(self, skv, ctx):
        return skv.RotaryTable(ctx, self.dim, self.positions, self.theta)

    def turn(self, x, at, t):
        """x [n][heads][dim], values of type t in 64 bits, by positions at [n]."""
        half = self.dim // 2
        i, j = (np.arange(half), half + np.arange(half)) if self.halves else (2 * np.arange(half), 2 * np.arange(half) + 1)
        c, s = (v[at][:, None].astype(np.float64) for v in (self.cos, self.sin))
        a, b = x[..., i], x[..., j]
        y = x.copy()
        single = lambda v: v.astype(np.float32).astype(np.float64)
        with np.errstate(all="ignore"):
            y[..., i] = R.typed(single(a * c - single(b * s)), t)[1]
            y[..., j] = R.typed(single(b * c + single(a * s)), t)[1]
        return y


def attention(q, k, v, seen, scale):
    """q [rows][dim] over k, v [tokens][dim]; seen [rows][tokens]: out, sums of weight times |v|, and the largest sum of
    |q k| scale log2(e) of a row."""
    k, v = (np.where(seen.any(0)[:, None], x, 0.0) for x in (k, v))
    s = np.where(seen, q @ k.T * scale, -np.inf)
    p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    size = (np.abs(q) @ np.abs(k).T * seen).max() * abs(scale) * np.log2(np.e)
    return p @ v, p @ np.abs(v), size


def bound(t, rows, dim, want, weighted, size, tokens, v_max):
    """What an output may be off.  Products of the types' values are exact in FP32; a score is a sum of `dim` of them in
    an order of the instruction's, at most dim roundings, the scale and the difference to the reference value three
    more, by 2^-23 (an instruction may cut instead of rounding) of at most `size`, times ln 2 in a weight; exp2 and the
    factors that join waves and splits are good for 16 * 2^-24, and sums over the tokens round once a token at most.
    A weight is one value of the type, or two for bfloat16 and at most 16 rows; float16's smallest steps, half of
    2^-24, count against a largest weight of 2^11 at least.  A weight and the sum of weights are off alike."""
    rel = np.log(2) * (dim + 3) * size * 2.0 ** -23 + (tokens + 16) * 2.0 ** -24 + 2.0 ** -20
    step = R.HALF_STEP[t]
    if t == "bf16" and rows <= 16:
        step = step * step
    off = (2 * rel + step) * weighted + (2.0 ** -36 * tokens * v_max if t == "f16" else 0.0)
    return off + R.HALF_STEP[t] * (np.abs(want) + off) + (2.0 ** -25 if t == "f16" else 2.0 ** -133)


class Rig:
    """A cache on the device and its rows in numpy."""

    def __init__(self, skv, ctx, t, heads, kv_heads, dim, batch=1, pages=None, layers=1, capacity=512, rotation=None, seed=0):
        self.skv, self.ctx, self.t, self.dt = skv, ctx, t, getattr(skv, t.upper())
        self.heads, self.kv, self.dim, self.batch, self.layers = heads, kv_heads, dim, batch, layers
        self.entries = (capacity + PAGE - 1) // PAGE
        pages = batch * self.entries if pages is None else pages
        self.cache = skv.PagedCache(ctx, layers, pages, batch, heads, kv_heads, dim, capacity, self.dt)
        self.rng = np.random.default_rng(seed)
        self.rotation = rotation
        self.table = None if rotation is None else rotation.table(skv, ctx)
        self.halves = True if rotation is None else rotation.halves
        # K and V [layer][page][token][head][channel]
        self.store = [np.zeros((layers, pages, PAGE, kv_heads, dim)) for _ in "kv"]
        self.pages = np.full((batch, self.entries), -1)

    def map_all(self, order=None):
        order = self.rng.permutation(self.store[0].shape[1])[:self.batch * self.entries] if order is None else order
        for b in range(self.batch):
            self.map(b, order[b * self.entries:(b + 1) * self.entries])

    def map(self, b, pages, first=0):
        self.pages[b, first:first + len(pages)] = pages
        self.cache.map(b, [int(p) for p in pages], first)

    def random(self, *shape, spread=1.0):
        return R.typed(self.rng.standard_normal(shape) * spread, self.t)

    def slots(self, b, tokens):
        tokens = np.asarray(tokens, int)
        return self.pages[b][tokens // PAGE], tokens % PAGE

    def rows(self, layer, b, tokens):
        page, at = self.slots(b, tokens)
        return [s[layer, page, at] for s in self.store]

    def note(self, at, k, v, parents=None, layer=0, seq0=0):
        """Rows k, v [batch][n][kv][dim] of a call into the numpy pages."""
        n = k.shape[1]
        for b, p in enumerate(at):
            if p < 0:
                continue
            _, depth, live = places(chain(n) if parents is None else parents[b])
            kk = k[b] if self.rotation is None else self.rotation.turn(k[b], np.where(live, p + depth, 0), self.t)
            page, place = self.slots(seq0 + b, p + np.arange(n)[live])
            self.store[0][layer, page, place] = kk[live]
            self.store[1][layer, page, place] = v[b][live]

    def append(self, at, n, parents=None, layer=0, seq0=0, k=None, v=None):
        (kr, k), (vr, v) = (self.random(len(at), n, self.kv, self.dim) if x is None else R.typed(x, self.t) for x in (k, v))
        self.skv.swiftkv_paged_append(self.ctx, self.ctx.to_device(kr), self.ctx.to_device(vr), self.cache, layer,
                                      list(at), n=n, table=self.table, halves=self.halves,
                                      parents=None if parents is None else sum(parents, []), seq0=seq0)
        self.ctx.synchronize()
        self.note(at, k, v, parents, layer, seq0)

    def values(self, at, n, layer0=0, layers=1, seq0=0):
        shape = (layers, len(at), n, self.kv, self.dim)
        size = 2 * int(np.prod(shape))
        bufs = [self.ctx.to_device(np.full(size, 0xff, np.uint8)) for _ in "kv"]
        self.skv.swiftkv_paged_values(self.ctx, self.cache, layer0, list(at), *bufs, n=n, layers=layers, seq0=seq0)
        self.ctx.synchronize()
        return [R.values_of(b.download(np.uint8, (size,)), self.t, shape) for b in bufs]

    def check_values(self, upto=None):
        """Every token that has a page, in every layer, bit for bit."""
        for b in range(self.batch):
            held = PAGE * int((self.pages[b] >= 0).argmin() if (self.pages[b] < 0).any() else self.entries)
            if held == 0:
                continue
            got = self.values([0], held, 0, self.layers, seq0=b)
            for layer in range(self.layers):
                for name, g, w in zip("kv", got, self.rows(layer, b, np.arange(held))):
                    np.testing.assert_array_equal(g[layer, 0], w, err_msg=f"{name} of sequence {b}, layer {layer}")

    def attend(self, at, n, parents=None, append=True, layer=0, seq0=0, scale=0.0, q=None, k=None, v=None, spread=1.0):
        """One call; its queries and outputs [batch][n][heads][dim]."""
        qr, q = self.random(len(at), n, self.heads, self.dim, spread=spread) if q is None else R.typed(q, self.t)
        dk = dv = None
        if append:
            (kr, k), (vr, v) = (self.random(len(at), n, self.kv, self.dim) if x is None else R.typed(x, self.t) for x in (k, v))
            dk, dv = self.ctx.to_device(kr), self.ctx.to_device(vr)
        out = self.ctx.to_device(np.full(qr.size, 0xff, np.uint8))
        self.skv.swiftkv_paged_attention(self.ctx, self.ctx.to_device(qr), dk, dv, self.cache, layer, list(at), out, n=n,
                                         table=self.table, halves=self.halves, scale=scale, seq0=seq0,
                                         parents=None if parents is None else sum(parents, []))
        self.ctx.synchronize()
        if append:
            self.note(at, k, v, parents, layer, seq0)
        return q, R.values_of(out.download(np.uint8, (qr.size,)), self.t, q.shape)

    def check_attention(self, at, n, parents=None, layer=0, seq0=0, scale=0.0, **how):
        q, out = self.attend(at, n, parents, layer=layer, seq0=seq0, scale=scale, **how)
        self.compare(q, out, at, parents, layer, seq0, scale)
        return out

    def compare(self, q, out, at, parents=None, layer=0, seq0=0, scale=0.0, call=None):
        """call: the tokens of the call that gave `out`, where q and out are some of its rows."""
        n, group = q.shape[1], self.heads // self.kv
        scale = scale or float(np.float32(1) / np.sqrt(np.float32(self.dim)))
        worst = 0.0
        for b, p in enumerate(at):
            own, depth, live = places(chain(n) if parents is None else parents[b])
            if p < 0 or not live.any():
                assert (out[b] == 0).all(), f"sequence {b}"
                continue
            assert (out[b][~live] == 0).all(), f"rows without a token of sequence {b}"
            tokens = p + int(live.sum())
            keys, values = self.rows(layer, seq0 + b, np.arange(tokens))
            turned = q[b] if self.rotation is None else self.rotation.turn(q[b], np.where(live, p + depth, 0), self.t)
            seen = np.concatenate([np.ones((int(live.sum()), p), bool), own[live][:, live]], 1)
            for h in range(self.heads):
                kh, vh = keys[:, h // group], values[:, h // group]
                want, weighted, size = attention(turned[live][:, h], kh, vh, seen, scale)
                off = bound(self.t, group * (call or n), self.dim, want, weighted, size, tokens, np.abs(vh).max())
                err = np.abs(out[b][live][:, h] - want)
                assert (err <= off).all(), f"sequence {b} head {h}: {(err / off).max():.3g} of the bound"
                worst = max(worst, (err / off).max())
        return worst

    def keep(self, at, accepted, layer0=0, layers=None, seq0=0):
        layers = self.layers if layers is None else layers
        m = len(accepted[0])
        left = self.skv.swiftkv_paged_keep(self.ctx, self.cache, layer0, layers, list(at), sum(accepted, []), m, seq0=seq0)
        self.ctx.synchronize()
        for b, (p, path) in enumerate(zip(at, accepted)):
            path = [a for a in path if a >= 0]
            if p < 0:
                assert left[b] == p
                continue
            assert left[b] == p + len(path)
            source, target = self.slots(seq0 + b, p + np.array(path, int)), self.slots(seq0 + b, p + np.arange(len(path)))
            for s in self.store:
                for layer in range(layer0, layer0 + layers):
                    s[layer][target] = s[layer][source].copy()
        return left
