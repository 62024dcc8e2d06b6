"""The block cache's attention where blocks have V scales far apart: what a row does not see, or hardly weighs, takes
nothing from the rest.  Bounds here go by each row's own visible tokens.  Long splits, whose tiles are more than one
window of the table."""
import numpy as np
import pytest

import block_ref as R
from test_gpu_block import Rig

pytestmark = pytest.mark.gpu

# Query tokens and heads on one key/value head, and weights: every form of the kernels (4, 8 and 16 rows in one
# workgroup, more rows with weights, more rows without).
FORMS = [(1, 1, False), (1, 3, True), (1, 5, False), (4, 4, False), (5, 3, True), (8, 5, True), (20, 1, False),
         (37, 2, False)]


def put(rig, at, k, v):
    """FP32 rows [n][dim] of K and V into sequence 0, on the device and in numpy."""
    (kr, k), (vr, v) = (R.typed(x[None, :, None], "f32") for x in (k, v))
    dk, dv = rig.ctx.to_device(kr), rig.ctx.to_device(vr)
    rig.skv.swiftkv_block_append(rig.ctx, dk, dv, rig.cache, 0, [at], n=k.shape[1], dtype=rig.skv.F32)
    rig.ctx.synchronize()
    rig.note([at], k, v)


def run(rig, q, at, weights):
    """Queries [n][heads][dim] at tokens at, at + 1, ... over what is cached: their values, out, block weights."""
    n = len(q)
    raw, q = R.typed(q, rig.t)
    dq, dout = rig.ctx.to_device(raw), rig.ctx.to_device(np.full(raw.size, 0xff, np.uint8))
    dw = rig.ctx.to_device(np.zeros((1, 1, rig.cache.blocks), np.float32)) if weights else None
    rig.skv.swiftkv_block_attention(rig.ctx, dq, None, None, rig.cache, 0, [at], dout, n=n, dtype=rig.dt, weights=dw)
    rig.ctx.synchronize()
    out = R.values_of(dout.download(np.uint8, (raw.size,)), rig.t, q.shape)
    return q, out, dw.download(np.float32, (rig.cache.blocks,)) if weights else None


def check(rig, q, at, out, weights):
    """Each row against its softmax over the tokens that it sees, in 64 bits.

    A weight is off by `rel` (as in block_ref, but that a query's two half floats leave 2^-23 of its largest value and a
    half float rounds by 2^-11, two of them by 2^-22), which the sums of p |v| carry, twice for their quotient.  What a
    weight rounds at the least, 2^-30 of the largest product of weight and V scale that the row sees, or with half
    floats 2^-35 of it (two of them 2^-39), meets codes of up to 127 at each token; the conversion of 32-bit byte sums
    adds less than that again."""
    n, heads, dim = q.shape
    page, prompt = rig.pages[0, 0, 0], heads * n > 16 and weights is None
    each, off = np.zeros(rig.cache.blocks), 0.0
    worst = 0.0
    for i in range(n):
        t = at + i + 1
        k, v = page.values(t)
        scales = np.repeat(page.scales[1], R.BLOCK)[:t]
        for h in range(heads):
            s = k @ q[i, h] * dim ** -0.5
            p = np.exp(s - s.max())
            p /= p.sum()
            s_max = (np.abs(k) @ np.abs(q[i, h])).max() * dim ** -0.5 * np.log2(np.e)
            q_max = np.abs(q[i, h]).max() * np.abs(k).sum(1).max() * dim ** -0.5 * np.log2(np.e)
            rel, step, floor = R.relative_bound(s_max, t), 0.0, 2.0 ** -29
            if prompt:
                rel = (np.log(2) * (130 * s_max + 2 * q_max) + t + 64) * 2.0 ** -24
                step, floor = (2.0 ** -22, 2.0 ** -39) if rig.t == "f32" else (2.0 ** -11, 2.0 ** -35)
            want, size = p @ v, p @ np.abs(v)
            bound = (2 * rel + step) * size + t * 127 * floor * (p * scales).max()
            bound += R.HALF_STEP[rig.t] * (np.abs(want) + bound) + (2.0 ** -25 if rig.t == "f16" else 2.0 ** -140)
            err = np.abs(out[i, h] - want)
            worst = max(worst, (err / bound).max()) if np.isfinite(err).all() else np.inf
            each += np.add.reduceat(np.pad(p, (0, len(each) * R.BLOCK - t)), np.arange(0, len(each) * R.BLOCK, R.BLOCK))
            off = max(off, 2 * rel + 4 * (s_max + 20) * 2.0 ** -24)
    assert worst <= 1, f"{worst:.3g} of the bound"
    if weights is not None:
        bound = off * each + (heads * n + 2) * 2.0 ** -24 * each + heads * n * 2.0 ** -126
        assert (np.abs(weights - each) <= bound).all(), f"weights: {np.abs(weights - each).max():.3g}"


def attend(rig, rng, at, n, heads, weights, q=None):
    q = rng.standard_normal((n, heads, rig.dim)) if q is None else q
    q, out, w = run(rig, q, at, weights)
    check(rig, q, at, out, w)


def rig_of(skv, ctx, t, heads, dim, tokens):
    return Rig(skv, ctx, t, 1, heads, 1, dim, tokens)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,heads,weights", FORMS)
@pytest.mark.parametrize("up", [13, 40, 100])
def test_rows_left_behind_a_restarted_sequence(skv, ctx, t, n, heads, weights, up):
    """A slot that held V rows 2^up larger, started anew with fewer rows: the blocks behind its end keep their scales,
    in the last tile and in the one behind it."""
    rng = np.random.default_rng(up + n)
    rig = rig_of(skv, ctx, t, heads, 64, 256)
    put(rig, 0, rng.standard_normal((200, 64)), rng.standard_normal((200, 64)) * 2.0 ** up)
    put(rig, 0, *rng.standard_normal((2, 90, 64)))
    for end in (10, 40, 64, 75, 90):
        if end >= n:
            attend(rig, rng, end - n, n, heads, weights)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,heads,weights", FORMS)
def test_what_is_left_behind_changes_no_bit(skv, ctx, t, n, heads, weights):
    """The same tokens in an empty slot and in slots that held large, small and no numbers."""
    seen = []
    for size in (None, 2.0 ** 110, 2.0 ** -99, np.nan):
        rng = np.random.default_rng(n)
        rig = rig_of(skv, ctx, t, heads, 64, 256)
        k, v, q = rng.standard_normal((90, 64)), rng.standard_normal((90, 64)), rng.standard_normal((n, heads, 64))
        if size is not None:
            put(rig, 0, *(rng.standard_normal((2, 250, 64)) * size))
        put(rig, 0, k, v)
        seen.append([])
        for end in (40, 65, 90):
            _, out, w = run(rig, q, end - n, weights)
            seen[-1].append(out.tobytes() + (w[:6].tobytes() if weights else b""))
    assert all(x == seen[0] for x in seen[1:])


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("n,heads,weights", FORMS)
def test_blocks_dropped_by_eviction(skv, ctx, t, n, heads, weights):
    """Dropped blocks lie right behind the kept ones."""
    rng = np.random.default_rng(n)
    rig = rig_of(skv, ctx, t, heads, 128, 256)
    k, v = rng.standard_normal((2, 112, 128))
    v[48:80] *= 2.0 ** 50                                       # blocks 3 and 4
    put(rig, 0, k, v)
    w = np.zeros((1, 1, 1, rig.cache.blocks), np.float32)
    w[..., :7] = [5, 4, 3, 0, 0.5, 6, 7]
    dw = ctx.to_device(w)
    left = skv.swiftkv_block_evict(ctx, rig.cache, 0, 1, 112, 5, dw)
    assert left == [80]
    rig.pages[0, 0, 0].reorder([0, 1, 2, 5, 6])
    for end in (80, 78, 64, 47):
        attend(rig, rng, end - n, n, heads, weights)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("n,heads,weights", [(8, 2, False), (16, 1, False), (8, 6, True), (60, 1, False), (60, 4, False),
                                             (200, 1, False)])
@pytest.mark.parametrize("at", [0, 5, 64])
def test_later_tokens_of_the_same_call(skv, ctx, t, n, heads, weights, at):
    """V rows 2^40 times those of the block before, two blocks out of three: a query takes nothing from those that come
    after it."""
    rng = np.random.default_rng(n + at)
    rig = rig_of(skv, ctx, t, heads, 64, 320)
    k, v = rng.standard_normal((2, at + n, 64))
    v *= 2.0 ** (40.0 * (np.arange(at + n) // 16 % 3))[:, None]
    put(rig, 0, k, v)
    attend(rig, rng, at, n, heads, weights)


def along_one_direction(rng, dim, height, n, heads):
    """Keys with scores height[t] for queries along one direction, with noise."""
    along = rng.standard_normal(dim)
    along /= np.linalg.norm(along)
    k = np.asarray(height)[:, None] * along + 0.02 * rng.standard_normal((len(height), dim))
    return k, dim ** 0.5 * along + 0.02 * rng.standard_normal((n, heads, dim))


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("n,heads,weights", FORMS)
@pytest.mark.parametrize("what", ["slight", "sink", "sink_last", "zero", "far"])
def test_weight_and_scale_against_each_other(skv, ctx, t, dim, n, heads, weights, what):
    """Tokens of hardly any weight with large values, tokens of nearly all the weight with small or no values."""
    rng = np.random.default_rng(dim + n)
    tokens = 330
    block = np.arange(tokens) // 16
    height, size = np.zeros(tokens), np.ones(tokens)
    if what == "slight":                                        # weight 2^-58 of the others', values 2^50 of theirs
        height[block % 5 == 1], size[block % 5 == 1] = -40.0, 2.0 ** 50
    elif what == "sink":                                        # weight 2^20 of the others', values 2^-30
        height[:16], size[:16] = 14.0, 2.0 ** -30
    elif what == "sink_last":
        height[288:304], size[288:304] = 14.0, 2.0 ** -30
    elif what == "zero":                                        # no values at all at the largest weights
        height[block % 7 == 3], size[block % 7 == 3] = 5.0, 0.0
    else:                                                       # both ends of the scales in one sequence
        size[block % 3 == 1] = 2.0 ** -90
        height[block % 4 == 2], size[block % 4 == 2] = -60.0, 2.0 ** 90
        height[96:112], size[96:112] = 3.0, 0.0
        if t == "f16":                                          # such values leave the type
            size = np.minimum(size, 1.0)
    k, q = along_one_direction(rng, dim, height, n, heads)
    rig = rig_of(skv, ctx, t, heads, dim, 384)
    put(rig, 0, k, rng.standard_normal((tokens, dim)) * size[:, None])
    for end in (330, 130, 60):
        attend(rig, rng, end - n, n, heads, weights, q)
    ctx.set_split_tokens(256)
    try:
        attend(rig, rng, tokens - n, n, heads, weights, q)
    finally:
        ctx.set_split_tokens(0)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("n,heads,weights", FORMS)
@pytest.mark.parametrize("size", [2.0 ** 125, 2.0 ** -88, 0.0])
def test_largest_and_smallest_values(skv, ctx, t, n, heads, weights, size):
    """Values whose sum leaves FP32's range though their mean does not, tiny ones, and none."""
    rng = np.random.default_rng(n)
    rig = rig_of(skv, ctx, t, heads, 64, 1100)
    v = size * np.where(rng.random((1050, 64)) < 0.5, 1.0, 0.8)
    put(rig, 0, rng.standard_normal((1050, 64)), v)
    for end in (1050, 300):
        attend(rig, rng, end - n, n, heads, weights)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("n,heads,weights", FORMS)
@pytest.mark.parametrize("height", [2.0 ** 18, -2.0 ** 18, 2.0 ** 24, 2.0 ** 29, -2.0 ** 29, 2.0 ** 60])
def test_scores_far_from_zero(skv, ctx, t, n, heads, weights, height):
    """Scores so large that FP32 has no fraction of them: the two tokens of the largest, the same in all their bits, share
    the weight, though their blocks' V scales differ.  Before them others hold it for a while."""
    rng = np.random.default_rng(n)
    dim, tokens = 64, 700
    part = 0.9 * rng.random(tokens) if height > 0 else 1.3 + rng.random(tokens)
    part[[100, 101, 390]] = 0.95 if height > 0 else 1.2
    for token in (420, 600):                    # in blocks of the same K scale, so of the same code
        part[token // 16 * 16:token // 16 * 16 + 16] = 0.5 if height > 0 else 2.0
        part[token] = 1.0
    q = np.tile(dim ** 0.25 * rng.standard_normal(dim), (n, heads, 1))
    _, q = R.typed(q, t)
    k = np.outer(part * height, q[0, 0] / (q[0, 0] @ q[0, 0] * dim ** -0.5))
    rig = rig_of(skv, ctx, t, heads, dim, 704)
    put(rig, 0, k, rng.standard_normal((tokens, dim)) * 2.0 ** (np.arange(tokens) // 16 * 7 % 13)[:, None])
    q, out, _ = run(rig, q, tokens - n, weights)
    page = rig.pages[0, 0, 0]
    keys, v = page.values(tokens)
    s = keys @ q[0, 0] * dim ** -0.5
    # the definition's own two, so far above the rest that no rounding of a score (2^-24 of it a few times) matters
    first, rest = np.flatnonzero(s == s.max()), np.sort(s)[:-2]
    assert first.tolist() == [420, 600] and rest.max() < s.max() - 0.01 * abs(height)
    want, size = v[first].mean(0), np.abs(v[first]).mean(0)
    step = 2.0 ** -20 + (0 if heads * n <= 16 or weights else 2.0 ** -22 if t == "f32" else 2.0 ** -11)
    bound = step * size + R.HALF_STEP[t] * np.abs(want) * (1 + step) + 256 * 2.0 ** -29 * page.scales[1].max()
    assert (np.abs(out - want) <= bound).all()


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,heads", [(1, 2), (40, 2)])
def test_small_values_in_channels_of_their_own(skv, ctx, t, n, heads):
    """Blocks whose scales differ by 2^12 with values in channels of their own, so that the small ones show."""
    rng = np.random.default_rng(18)
    rig = rig_of(skv, ctx, t, heads, 64, 640)
    v = rng.standard_normal((600, 64))
    large = np.arange(600) // 16 % 3 == 0
    v[large, 32:] = 0
    v[~large, :32] = 0
    v[~large] *= 2.0 ** -12
    put(rig, 0, rng.standard_normal((600, 64)), v)
    attend(rig, rng, 600 - n, n, heads, False)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 4, 70])
def test_second_window_of_the_table(skv, ctx, t, n):
    """One split of 20011 tokens and those that the call appends: a wave or team takes more tiles than the 64 whose table
    entries it reads at a time, and the appended ones lie in its second window."""
    rng = np.random.default_rng(n)
    rig = Rig(skv, ctx, t, 1, 4, 1, 64, 20100)
    rig.append(rng, [0], 20011)
    ctx.set_split_tokens(32768)
    try:
        rig.check_attention(rng, [20011], n, weights=n == 4)
        rig.check_attention(rng, [20010 + n], 1, append=False)
    finally:
        ctx.set_split_tokens(0)
