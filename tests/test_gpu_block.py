"""The block cache on the GPU against its definition in 64 bits: codes and values, attention, weights, eviction, and
what the entries refuse."""
import numpy as np
import pytest

import block_ref as R

pytestmark = pytest.mark.gpu


class Rig:
    """A cache on the device and its pages in numpy, fed the same rows."""

    def __init__(self, skv, ctx, t, batch, heads, kv_heads, dim, capacity, layers=1):
        self.skv, self.ctx, self.t, self.dt = skv, ctx, t, getattr(skv, t.upper())
        self.batch, self.heads, self.kv, self.dim, self.layers = batch, heads, kv_heads, dim, layers
        self.cache = skv.BlockCache(ctx, layers, batch, heads, kv_heads, dim, capacity)
        cap = self.cache.blocks * R.BLOCK
        self.pages = {(l, b, h): R.Page(cap, dim) for l in range(layers) for b in range(batch) for h in range(kv_heads)}

    def rows(self, rng, batch, n, heads, spread=1.0):
        x = rng.standard_normal((batch, n, heads, self.dim))
        x *= np.where(rng.random((heads, self.dim)) < 1 / 32, spread, 1.0)
        return R.typed(x, self.t)

    def note(self, at, k, v, layer=0, seq0=0):
        """k, v [batch][n][kv][dim] into the numpy pages."""
        for b, p in enumerate(at):
            if p >= 0:
                for h in range(self.kv):
                    self.pages[layer, seq0 + b, h].append(p, k[b, :, h], v[b, :, h])

    def append(self, rng, at, n, spread=1.0, layer=0, seq0=0):
        (kr, k), (vr, v) = (self.rows(rng, len(at), n, self.kv, spread) for _ in "kv")
        dk, dv = self.ctx.to_device(kr), self.ctx.to_device(vr)
        self.skv.swiftkv_block_append(self.ctx, dk, dv, self.cache, layer, at, n=n, dtype=self.dt, seq0=seq0)
        self.ctx.synchronize()
        self.note(at, k, v, layer, seq0)

    def check_values(self, at, n, layer=0, seq0=0):
        """Every value of tokens [at, at + n), exactly: a code times a power of two is a value of each type unless it
        leaves float16's range, which these inputs do not."""
        count = len(at) * n * self.kv * self.dim
        size = 4 if self.t == "f32" else 2
        dk, dv = self.ctx.alloc(count * size), self.ctx.alloc(count * size)
        self.skv.swiftkv_block_values(self.ctx, self.cache, layer, at, dk, dv, n=n, dtype=self.dt, seq0=seq0)
        self.ctx.synchronize()
        for i, buf in enumerate((dk, dv)):
            got = R.values_of(buf.download(np.uint8, (count * size,)), self.t, (len(at), n, self.kv, self.dim))
            for b, p in enumerate(at):
                for h in range(self.kv):
                    want = self.pages[layer, seq0 + b, h].values(p + n)[i][p:]
                    np.testing.assert_array_equal(got[b, :, h], want, err_msg=f"{'kv'[i]} sequence {b} head {h}")

    def check_attention(self, rng, at, n, append=True, weights=False, scale=None, layer=0, seq0=0, spread=1.0):
        qr, q = self.rows(rng, len(at), n, self.heads)
        dq = self.ctx.to_device(qr)
        dk = dv = None
        if append:
            (kr, k), (vr, v) = (self.rows(rng, len(at), n, self.kv, spread) for _ in "kv")
            dk, dv = self.ctx.to_device(kr), self.ctx.to_device(vr)
            self.note(at, k, v, layer, seq0)
        dout = self.ctx.to_device(np.full(qr.size, 0xff, np.uint8))
        before = rng.random((len(at), self.kv, self.cache.blocks)).astype(np.float32)
        dw = self.ctx.to_device(before) if weights else None
        self.skv.swiftkv_block_attention(self.ctx, dq, dk, dv, self.cache, layer, at, dout, n=n, dtype=self.dt,
                                         scale=scale or 0.0, weights=dw, seq0=seq0)
        self.ctx.synchronize()
        out = R.values_of(dout.download(np.uint8, (qr.size,)), self.t, q.shape)
        self.compare(q, at, n, out, before, dw.download(np.float32, before.shape) if weights else None, scale, layer,
                     seq0)
        return out

    def compare(self, q, at, n, out, before, after, scale=None, layer=0, seq0=0):
        scale = self.dim ** -0.5 if scale is None else scale
        group = self.heads // self.kv
        for b, p in enumerate(at):
            if p < 0:
                assert (out[b] == 0).all()
                if after is not None:
                    np.testing.assert_array_equal(after[b], before[b])
                continue
            for h in range(self.kv):
                page = self.pages[layer, seq0 + b, h]
                v_max = np.abs(page.values(p + n)[1]).max()
                each, off = np.zeros(self.cache.blocks), 0.0
                for g in range(group):
                    want, w, s, s_q = R.attention(page, q[b, :, h * group + g], p, scale)
                    rel, step = R.relative_bound(s, p + n), 0.0
                    if group * n > 16 and after is None:
                        rel, step = R.prompt_bound(s, s_q, p + n, self.t)
                    bound = (2 * rel + step) * v_max + R.HALF_STEP[self.t] * np.abs(want) * (1 + 2 * rel) + 2.0 ** -24 * (self.t == "f16")
                    err = np.abs(out[b, :, h * group + g] - want)
                    assert (err <= bound).all(), f"sequence {b} head {h * group + g}: {(err / bound).max():.3g} of the bound"
                    each += w
                    # the block's and the row's log-sums round by 2^-24 of at most S + log2(tokens), twice each
                    off = max(off, 2 * rel + 4 * (s + 20) * 2.0 ** -24)
                if after is not None:
                    err = np.abs(after[b, h] - (before[b, h] + each))
                    bound = off * each + (group * n + 2) * 2.0 ** -24 * (before[b, h] + each) * (each > 0)
                    assert (err <= bound).all(), f"weights of sequence {b} head {h}: {(err - bound).max():.3g}"


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("spread", [1.0, 20.0])
def test_append_and_values(skv, ctx, t, dim, spread):
    """Rows one at a time and many at once, tail blocks that keep their scale and that need a larger one."""
    rng = np.random.default_rng(dim + int(spread))
    rig = Rig(skv, ctx, t, 3, 2, 2, dim, 200)
    at = [0, 0, 0]
    for n in (1, 1, 15, 16, 3, 33, 1, 64, 2):
        rig.append(rng, at, n, spread)
        rig.check_values(at, n)
        at = [p + n for p in at]
        rng = np.random.default_rng(at[0])
    rig.check_values([0, 0, 0], at[0])


def test_append_ragged_skipped_and_restarted(skv, ctx):
    rng = np.random.default_rng(7)
    rig = Rig(skv, ctx, "f32", 5, 3, 3, 64, 64)
    rig.append(rng, [0], 40, seq0=1)
    rig.append(rng, [0], 17, seq0=3)
    rig.append(rng, [0, 40, -1, 17, 0], 9)
    for seq, p, n in ((0, 0, 9), (1, 0, 49), (3, 0, 26), (4, 0, 9), (2, 0, 64)):
        rig.check_values([p], n, seq0=seq)
    rig.append(rng, [0], 5, seq0=1, spread=20.0)      # anew: the old scale of block 0 is gone
    rig.check_values([0], 5, seq0=1)
    rig.check_values([16], 33, seq0=1)


def test_scale_limits(skv, ctx):
    """127 * 2^e exactly, just above it, zeros, denormals and the largest value, whose code would stand for 2^128:
    such rows poison their block."""
    rig = Rig(skv, ctx, "f32", 6, 1, 1, 64, 64)
    x = np.zeros((6, 1, 1, 64))
    up = np.nextafter(np.float32(127), np.float32(200))
    x[0, 0, 0, 3], x[1, 0, 0, 3], x[2, 0, 0, 5] = 127.0, -float(up), 1e-40
    x[3, 0, 0, 0], x[4, 0, 0, 63], x[4, 0, 0, 1] = np.finfo(np.float32).max, 127.0 * 2.0 ** -100, 63.0 * 2.0 ** -100
    raw, k = R.typed(x, "f32")
    dk = ctx.to_device(raw)
    skv.swiftkv_block_append(ctx, dk, dk, rig.cache, 0, [0] * 6, dtype=skv.F32)
    rig.note([0] * 6, k, k)
    rig.check_values([0] * 6, 1)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 128), (8, 2, 128), (8, 1, 64), (5, 1, 128), (6, 2, 64)])
@pytest.mark.parametrize("at,n", [([0], 1), ([1, 0, 15], 1), ([16, 63, 64], 1), ([127, 300], 2), ([255, 3], 5),
                                  ([0, 40], 33)])
def test_attention(skv, ctx, t, heads, kv_heads, dim, at, n):
    rng = np.random.default_rng(heads * 1000 + n + len(at))
    rig = Rig(skv, ctx, t, len(at), heads, kv_heads, dim, max(at) + n)
    for b, p in enumerate(at):
        if p:
            rig.append(rng, [0], p, spread=5.0, seq0=b)
    rig.check_attention(rng, at, n, weights=n <= 8)


@pytest.mark.parametrize("split,n", [(256, 3), (512, 3), (256, 5), (256, 37), (512, 70)])
def test_forced_splits(skv, ctx, split, n):
    """Splits of a few tiles, some sequences with one split, some with many, one absent."""
    rng = np.random.default_rng(split)
    at = [1023, 200, -1, 777]
    rig = Rig(skv, ctx, "f32", 4, 8, 2, 64, 1100)
    for b, p in enumerate(at):
        if p > 0:
            rig.append(rng, [0], p, seq0=b)
    ctx.set_split_tokens(split)
    try:
        rig.check_attention(rng, at, n, weights=n <= 8)
    finally:
        ctx.set_split_tokens(0)


@pytest.mark.parametrize("n", [1, 4, 70])
def test_long_context(skv, ctx, n):
    rng = np.random.default_rng(n)
    rig = Rig(skv, ctx, "bf16", 1, 4, 1, 128, 20100)
    rig.append(rng, [0], 20011)
    rig.check_attention(rng, [20011], n, weights=n <= 8)
    if n == 1:
        rig.check_attention(rng, [20011], n, append=False, scale=0.5)     # a peaked softmax, nothing appended


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 3, 64), (8, 1, 128), (10, 2, 128)])
@pytest.mark.parametrize("at,n", [(0, 130), (100, 17), (64, 64), (8300, 20), (5, 300)])
def test_prompt_chunks(skv, ctx, t, heads, kv_heads, dim, at, n):
    """Chunks that end inside a row tile, a workgroup's rows and a block; more than 64 tiles; heavy channels."""
    rng = np.random.default_rng(at + n)
    rig = Rig(skv, ctx, t, 1, heads, kv_heads, dim, at + n)
    if at:
        rig.append(rng, [0], at, spread=20.0)
    rig.check_attention(rng, [at], n, spread=20.0)


@pytest.mark.parametrize("n", [1, 40])
def test_scales(skv, ctx, n):
    """A negative scale, and one that leaves all weights the same."""
    rng = np.random.default_rng(16)
    rig = Rig(skv, ctx, "f32", 1, 4, 2, 64, 256)
    rig.append(rng, [0], 100)
    rig.check_attention(rng, [100], n, scale=-0.3)
    rig.check_attention(rng, [100], n, append=False, scale=1e-30)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("steps", [3, 5])
def test_rising_scores_in_a_chunk(skv, ctx, t, dim, steps):
    """Scores that rise 2^steps-fold in 256 tokens, below and above what moves a row's reference value, over V blocks
    whose scales differ by 2^12."""
    rng = np.random.default_rng(17)
    tokens, n, heads, kv_heads = 1160, 40, 4, 2
    rig = Rig(skv, ctx, t, 1, heads, kv_heads, dim, 1216)
    along = rng.standard_normal(dim)
    along /= np.linalg.norm(along)
    rise = steps * np.log(2.0) / 256 * np.arange(tokens + n)
    k = rise[None, :, None, None] * along + 0.05 * rng.standard_normal((1, tokens + n, kv_heads, dim))
    v = rng.standard_normal(k.shape) * np.where(np.arange(tokens + n) // 16 % 3 == 0, 1.0, 2.0 ** -12)[None, :, None, None]
    q = dim ** 0.5 * along + 0.05 * rng.standard_normal((1, n, heads, dim))
    (_, k), (_, v), (qr, q) = (R.typed(x, t) for x in (k, v, q))
    for first, count in ((0, tokens), (tokens, n)):
        part = slice(first, first + count)
        dk, dv = (ctx.to_device(R.typed(x[:, part], t)[0]) for x in (k, v))
        skv.swiftkv_block_append(ctx, dk, dv, rig.cache, 0, [first], n=count, dtype=rig.dt)
        rig.note([first], k[:, part], v[:, part])
        ctx.synchronize()
    dq, dout = ctx.to_device(qr), ctx.alloc(qr.size)
    skv.swiftkv_block_attention(ctx, dq, None, None, rig.cache, 0, [tokens], dout, n=n, dtype=rig.dt)
    ctx.synchronize()
    rig.compare(q, [tokens], n, R.values_of(dout.download(np.uint8, (qr.size,)), t, q.shape), None, None)


def test_not_a_number_in_a_chunk(skv, ctx):
    """Within a chunk: a poisoned block reaches the queries that see it and no others."""
    rng = np.random.default_rng(15)
    rig = Rig(skv, ctx, "f32", 2, 2, 1, 64, 128)
    (kr, k), (vr, v) = (rig.rows(rng, 2, 100, 1) for _ in "kv")
    k[0, 70], v[1, 37, 0, 7] = np.nan, np.inf
    dk, dv = (ctx.to_device(R.typed(x, "f32")[0]) for x in (k, v))
    qr, q = rig.rows(rng, 2, 100, 2)
    q[:, 5, 1, 3] = np.nan
    qr, _ = R.typed(q, "f32")
    dq, dout = ctx.to_device(qr), ctx.alloc(qr.size)
    skv.swiftkv_block_attention(ctx, dq, dk, dv, rig.cache, 0, [0, 0], dout, n=100, dtype=skv.F32)
    ctx.synchronize()
    out = dout.download(np.float32, (2, 100, 2, 64))
    for b, first in enumerate((64, 32)):        # the first token of the poisoned block
        assert np.isnan(out[b, first:]).all()
        assert np.isnan(out[b, 5, 1]).all()
        out[b, 5, 1] = 0
        assert np.isfinite(out[b, :first]).all()


def test_layers_and_slots_are_apart(skv, ctx):
    rng = np.random.default_rng(3)
    rig = Rig(skv, ctx, "f32", 3, 2, 1, 64, 100, layers=3)
    for layer in range(3):
        for b in range(3):
            rig.append(rng, [0], 20 + 7 * layer + b, layer=layer, seq0=b)
    for layer in (2, 0, 1):
        rig.check_attention(rng, [20 + 7 * layer + 1, 20 + 7 * layer + 2], 2, layer=layer, seq0=1, weights=True)
    for layer in range(3):
        rig.check_values([0], 20 + 7 * layer, layer=layer, seq0=0)


def test_not_a_number_reaches_what_attends_to_it(skv, ctx):
    """A NaN key or an infinite value poisons its block for the queries that see it, in either order of rows, and
    nothing else; what lies behind a sequence's end is never seen."""
    rng = np.random.default_rng(5)
    rig = Rig(skv, ctx, "f32", 3, 2, 1, 64, 128)
    (kr, k), (vr, v) = (rig.rows(rng, 3, 40, 1) for _ in "kv")
    k[0, 33], v[1, 20, 0, 7], k[2, 39, 0, 0] = np.nan, np.inf, -np.inf
    dk, dv = (ctx.to_device(R.typed(x, "f32")[0]) for x in (k, v))
    skv.swiftkv_block_append(ctx, dk, dv, rig.cache, 0, [0] * 3, n=40, dtype=skv.F32)
    qr, q = rig.rows(rng, 3, 1, 2)
    dq, dout = ctx.to_device(qr), ctx.alloc(qr.size)

    def run(at):
        skv.swiftkv_block_attention(ctx, dq, None, None, rig.cache, 0, at, dout, dtype=skv.F32)
        ctx.synchronize()
        return dout.download(np.float32, (3, 2, 64))

    assert np.isfinite(run([31, 15, 31])).all()
    got = run([32, 16, 32])
    assert np.isnan(got).all()
    skv.swiftkv_block_append(ctx, dk, dv, rig.cache, 0, [0] * 3, n=3, dtype=skv.F32)     # anew
    assert np.isfinite(run([2, 2, 2])).all()


def test_queries_out_of_range(skv, ctx):
    """An infinite query gives NaN in its own row only; huge and tiny finite ones are exact enough."""
    rng = np.random.default_rng(6)
    rig = Rig(skv, ctx, "f32", 1, 4, 1, 64, 64)
    rig.append(rng, [0], 50)
    q = rng.standard_normal((1, 1, 4, 64))
    q[0, 0, 1] *= 1e-30
    q[0, 0, 2] = 0
    q[0, 0, 3, 5] = np.inf
    raw, q = R.typed(q, "f32")
    dq, dout = ctx.to_device(raw), ctx.alloc(raw.size)
    skv.swiftkv_block_attention(ctx, dq, None, None, rig.cache, 0, 49, dout, dtype=skv.F32)
    ctx.synchronize()
    out = dout.download(np.float32, (4, 64))
    assert np.isnan(out[3]).all()
    v = rig.pages[0, 0, 0].values(50)[1]
    for h in (1, 2):
        np.testing.assert_allclose(out[h], v.mean(0), rtol=0, atol=np.abs(v).max() * 64 * 2.0 ** -24)


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_strided_rows(skv, ctx, t):
    """q, k and v as parts of one projection row, out inside a wider tensor whose other columns stay as they were."""
    rng = np.random.default_rng(8)
    rig = Rig(skv, ctx, t, 2, 4, 2, 64, 128)
    size, n, wide = (4 if t == "f32" else 2), 3, 4 * 64 + 2 * 2 * 64 + 64
    rig.append(rng, [0, 0], 30)
    x = rng.standard_normal((2, n, wide))
    raw, x = R.typed(x, t)
    dx = ctx.to_device(raw)
    q, k, v = (x[..., a:b].reshape(2, n, -1, 64) for a, b in ((0, 256), (256, 384), (384, 512)))
    out_wide = 4 * 64 + 32
    dout = ctx.to_device(np.full(2 * n * out_wide * size, 0xee, np.uint8))
    rig.note([30, 30], k, v)
    skv.swiftkv_block_attention(ctx, dx.ptr, dx.ptr + 256 * size, dx.ptr + 384 * size, rig.cache, 0, [30, 30], dout.ptr,
                                n=n, dtype=rig.dt, q_stride=wide, k_stride=wide, v_stride=wide, out_stride=out_wide)
    ctx.synchronize()
    got = dout.download(np.uint8, (2, n, out_wide * size))
    assert (got[..., 256 * size:] == 0xee).all()
    out = R.values_of(got[..., :256 * size], t, q.shape)
    rig.compare(q, [30, 30], n, out, None, None)


def test_more_sequences_than_a_launch_takes(skv, ctx):
    rng = np.random.default_rng(9)
    rig = Rig(skv, ctx, "bf16", 300, 1, 1, 64, 64)
    at = rng.integers(0, 60, 300).tolist()
    at[5] = at[290] = -1
    for p in range(1, 60):
        where = [p - 1 if p <= q else -1 for q in at]
        rig.append(rng, where, 1)
    rig.check_attention(rng, at, 1, weights=True)


@pytest.mark.parametrize("held,keep,sinks,recent", [(1, 1, 0, 1), (40, 40, 2, 3), (41, 40, 2, 3), (300, 17, 1, 4),
                                                    (300, 5, 1, 4), (511, 300, 0, 1), (64, 63, 10, 20)])
def test_evict(skv, ctx, held, keep, sinks, recent):
    rng = np.random.default_rng(held + keep)
    layers, batch, kv = 2, 3, 2
    cache = skv.BlockCache(ctx, layers, batch, kv, kv, 64, 512 * 16)
    at = [held * 16 - 5, max(1, held // 2) * 16, -1]
    w = np.exp(rng.standard_normal((layers, batch, kv, cache.blocks)) * 3).astype(np.float32)
    w[:, :, 0] = np.round(w[:, :, 0])                 # ties, zeros among them
    w[0, 0, 1, ::3] = np.nan
    w[1, 0, 1, ::2] *= -1
    dw, dk = ctx.to_device(w), ctx.alloc(layers * batch * kv * keep * 4)
    left = skv.swiftkv_block_evict(ctx, cache, 0, layers, at, keep, dw, dk, sinks=sinks, recent=recent)
    ctx.synchronize()
    got, kept = dw.download(np.float32, w.shape), dk.download(np.int32, (layers, batch, kv, keep))
    for b, p in enumerate(at):
        nb = -(-p // 16)
        assert left[b] == (p if p < 0 else p - 16 * max(0, nb - keep))
        if p < 0:
            np.testing.assert_array_equal(got[:, b], w[:, b])
            continue
        for l in range(layers):
            for h in range(kv):
                want = R.evict(w[l, b, h], nb, keep, sinks, recent)
                assert kept[l, b, h].tolist() == want + [-1] * (keep - len(want))
                np.testing.assert_array_equal(got[l, b, h, :len(want)], w[l, b, h, want])
                assert (got[l, b, h, len(want):] == 0).all()


def test_evict_of_the_longest_cache(skv, ctx):
    rng = np.random.default_rng(2)
    cache = skv.BlockCache(ctx, 1, 1, 1, 1, 64, skv.BLOCK_MAX_SEQ)
    nb = cache.blocks
    w = rng.integers(0, 50, (1, 1, 1, nb)).astype(np.float32)
    dw, dk = ctx.to_device(w), ctx.alloc(4 * 3000)
    skv.swiftkv_block_evict(ctx, cache, 0, 1, skv.BLOCK_MAX_SEQ, 3000, dw, dk, sinks=4, recent=8)
    ctx.synchronize()
    assert dk.download(np.int32, (3000,)).tolist() == R.evict(w[0, 0, 0], nb, 3000, 4, 8)


def test_decode_with_eviction(skv, ctx):
    """The operators together as a program runs them: rotate, append and attend with weights, evict when a sequence
    is full, go on; two layers, positions that run ahead of the cache's rows."""
    rng = np.random.default_rng(11)
    batch, heads, kv, dim, layers, keep = 2, 4, 2, 64, 2, 5
    rig = Rig(skv, ctx, "f32", batch, heads, kv, dim, 128, layers)
    table = skv.RotaryTable(ctx, dim, 4096, scaling=skv.RopeScaling(skv.ROPE_LINEAR, 2.0))
    half = dim // 2
    freq = 10000.0 ** (-np.arange(half) / half) / 2.0
    dw = ctx.to_device(np.zeros((layers, batch, kv, rig.cache.blocks), np.float32))
    per_layer = batch * kv * rig.cache.blocks * 4
    cached, position, wide = [0, 0], [0, 700], (heads + 2 * kv) * dim
    evictions = 0
    for step in range(30):
        n = 37 if step == 0 else 1 + step % 7
        if max(cached) + n > 128:
            w = dw.download(np.float32, (layers, batch, kv, rig.cache.blocks))
            dk = ctx.alloc(layers * batch * kv * keep * 4)
            left = skv.swiftkv_block_evict(ctx, rig.cache, 0, layers, cached, keep, dw, dk, sinks=1, recent=2)
            ctx.synchronize()
            kept = dk.download(np.int32, (layers, batch, kv, keep))
            for (l, b, h), page in rig.pages.items():
                want = R.evict(w[l, b, h], -(-cached[b] // 16), keep, 1, 2)
                assert kept[l, b, h].tolist() == want
                page.reorder(want)
            cached = left
            evictions += 1
        for layer in range(layers):
            raw, x = R.typed(rng.standard_normal((batch, n, heads + 2 * kv, dim)), "f32")
            dx = ctx.to_device(raw)
            skv.swiftkv_rotary(ctx, table, dx, dx, position, heads + kv, dim, n=n, dtype=skv.F32, x_stride=wide,
                               out_stride=wide)
            ctx.synchronize()
            turned = dx.download(np.float32, (batch, n, heads + 2 * kv, dim)).astype(np.float64)
            angle = (np.array(position)[:, None] + np.arange(n))[..., None, None] * freq
            a, b = x[:, :, :heads + kv, :half], x[:, :, :heads + kv, half:]
            want = np.concatenate([a * np.cos(angle) - b * np.sin(angle), a * np.sin(angle) + b * np.cos(angle)], -1)
            # cos and sin rounded once, two products and a sum: 4 half-steps of |a| + |b|
            assert (np.abs(turned[:, :, :heads + kv] - want) <= 4 * 2.0 ** -24 * 2 * np.abs(x).max()).all()
            np.testing.assert_array_equal(turned[:, :, heads + kv:], x[:, :, heads + kv:])
            q, k, v = turned[:, :, :heads], turned[:, :, heads:heads + kv], turned[:, :, heads + kv:]
            rig.note(cached, k, v, layer)
            dout = ctx.alloc(batch * n * heads * dim * 4)
            w_ptr = dw.ptr + layer * per_layer if n <= 8 else None
            before = dw.download(np.float32, (batch, kv, rig.cache.blocks), layer * per_layer)
            skv.swiftkv_block_attention(ctx, dx.ptr, dx.ptr + heads * dim * 4, dx.ptr + (heads + kv) * dim * 4, rig.cache,
                                        layer, cached, dout, n=n, dtype=skv.F32, weights=w_ptr, q_stride=wide,
                                        k_stride=wide, v_stride=wide)
            ctx.synchronize()
            after = dw.download(np.float32, (batch, kv, rig.cache.blocks), layer * per_layer)
            rig.compare(q, cached, n, dout.download(np.float32, q.shape).astype(np.float64), before,
                        after if n <= 8 else None, layer=layer)
        cached = [c + n for c in cached]
        position = [p + n for p in position]
    assert evictions >= 1 and min(position) > 100


def test_captured_and_replayed(skv, ctx):
    """A step with weights and an eviction in one graph, replayed with eager work between, against the same calls."""
    rng = np.random.default_rng(12)
    heads, kv, dim = 8, 2, 64

    def make():
        rig = Rig(skv, ctx, "bf16", 2, heads, kv, dim, 1024)
        rig.append(np.random.default_rng(1), [0, 0], 900)
        return rig

    (qr, _), (kr, _), (vr, _) = (make().rows(rng, 2, 2, h) for h in (heads, kv, kv))
    dq, dk, dv = (ctx.to_device(r) for r in (qr, kr, vr))

    def calls(rig, dw, dout, dkept):
        skv.swiftkv_block_attention(ctx, dq, dk, dv, rig.cache, 0, [900, 900], dout, n=2, weights=dw)
        skv.swiftkv_block_evict(ctx, rig.cache, 0, 1, [902, 902], 40, dw, dkept, sinks=1, recent=2)

    sides = []
    for _ in range(2):
        rig = make()
        dw = ctx.to_device(np.zeros((2, kv, rig.cache.blocks), np.float32))
        sides.append((rig, dw, ctx.alloc(qr.size), ctx.alloc(2 * kv * 40 * 4)))
        calls(*sides[-1])
        ctx.synchronize()
    eager, recorded = sides
    ctx.capture_begin()
    calls(*recorded)
    graph = ctx.capture_end()
    for _ in range(4):
        graph.launch()
        calls(*eager)
        ctx.synchronize()
        for i in (1, 2, 3):
            a, b = (s[i].download(np.uint8, (s[i].nbytes,)) for s in (eager, recorded))
            np.testing.assert_array_equal(a, b)
    graph.close()


def test_same_results_twice(skv, ctx):
    """Splits and weights in a fixed order: the same bits each time."""
    rng = np.random.default_rng(13)
    rig = Rig(skv, ctx, "bf16", 1, 8, 2, 128, 5000)
    rig.append(rng, [0], 4990)
    qr, _ = rig.rows(rng, 1, 1, 8)
    dq, first = ctx.to_device(qr), None
    for _ in range(20):
        dout, dw = ctx.alloc(qr.size), ctx.to_device(np.zeros((1, 2, rig.cache.blocks), np.float32))
        skv.swiftkv_block_attention(ctx, dq, None, None, rig.cache, 0, 4989, dout, weights=dw)
        ctx.synchronize()
        got = dout.download(np.uint8, (qr.size,)).tobytes() + dw.download(np.uint8, (dw.nbytes,)).tobytes()
        first = first or got
        assert got == first


def test_refusals(skv, ctx):
    """Each refused call names its fault, enqueues nothing and leaves the cache as it was."""
    rng = np.random.default_rng(14)
    rig = Rig(skv, ctx, "f32", 2, 4, 2, 64, 64)
    rig.append(rng, [0, 0], 20)
    buf = ctx.alloc(1 << 20)
    w, c = ctx.alloc(1 << 16), rig.cache

    def refused(code, f, *a, **k):
        with pytest.raises(skv.SwiftKVError) as e:
            f(ctx, *a, **k)
        assert e.value.code == code, str(e.value)

    app, att, evi = skv.swiftkv_block_append, skv.swiftkv_block_attention, skv.swiftkv_block_evict
    f = dict(dtype=skv.F32)
    refused(skv.ERANGE, app, buf, buf, c, 0, 64, **f)
    refused(skv.ERANGE, app, buf, buf, c, 0, [0, 60], n=5, **f)
    refused(skv.ERANGE, app, buf, buf, c, 1, 0, **f)
    refused(skv.ERANGE, app, buf, buf, c, 0, [0, 0, 0], **f)
    refused(skv.ERANGE, app, buf, buf, c, 0, [0, 0], seq0=1, **f)
    refused(skv.ERANGE, app, buf, buf, c, 0, 0, n=-1, **f)
    refused(skv.EINVAL, app, buf, buf, c, 0, 0, dtype=3)
    refused(skv.EINVAL, app, buf.ptr + 4, buf, c, 0, 0, **f)
    refused(skv.EINVAL, app, buf, None, c, 0, 0, **f)
    refused(skv.EINVAL, app, buf, buf, c, 0, 0, k_stride=127, **f)
    refused(skv.EINVAL, app, buf, buf, c, 0, 0, k_stride=130, **f)
    refused(skv.EINVAL, att, buf, buf, None, c, 0, 0, buf, **f)
    refused(skv.EINVAL, att, None, None, None, c, 0, 0, buf, **f)
    refused(skv.EINVAL, att, buf, None, None, c, 0, 0, None, **f)
    refused(skv.EINVAL, att, buf, None, None, c, 0, 0, buf, scale=float("nan"), **f)
    refused(skv.EINVAL, att, buf, None, None, c, 0, 0, buf, q_stride=255, **f)
    refused(skv.ERANGE, att, buf, None, None, c, 0, 0, buf, n=9, weights=w, **f)
    refused(skv.EINVAL, evi, c, 0, 1, 20, 3, None)
    refused(skv.EINVAL, evi, c, 0, 1, 20, 3, w, sinks=3, recent=1)
    refused(skv.EINVAL, evi, c, 0, 1, 20, 3, w, recent=0)
    refused(skv.EINVAL, evi, c, 0, 1, 20, 5, w)
    refused(skv.ERANGE, evi, c, 0, 2, 20, 3, w)
    refused(skv.ERANGE, evi, c, 0, 1, 65, 3, w)
    with skv.Context(0) as other:
        with pytest.raises(skv.SwiftKVError):
            app(other, buf, buf, c, 0, 0, **f)
    ctx.set_host_io(True)
    try:
        refused(skv.ESTATE, app, buf, buf, c, 0, 0, **f)
    finally:
        ctx.set_host_io(False)
    for bad in ((0, 1, 4, 2, 64, 64), (1, 0, 4, 2, 64, 64), (1, 1, 3, 2, 64, 64), (1, 1, 4, 2, 96, 64),
                (1, 1, 4, 2, 64, 0), (1, 1, 4, 2, 64, skv.BLOCK_MAX_SEQ + 1), (1, 1, 65, 1, 64, 64)):
        with pytest.raises(skv.SwiftKVError) as e:
            skv.BlockCache(ctx, *bad)
        assert e.value.code == skv.EINVAL
    rig.check_values([0, 0], 20)
    # weights first asked for during a capture would allocate
    ctx.capture_begin()
    try:
        refused(skv.ESTATE, att, buf, None, None, c, 0, 19, buf, weights=w, **f)
    finally:
        ctx.capture_end().close()
    app(ctx, buf, buf, c, 0, 0, n=0, **f)
    att(ctx, buf, None, None, c, 0, 0, buf, n=0, **f)
