"""Rotary positions on the GPU against 64-bit rotations, and the scaled Q1.17 table of the step entries."""
import numpy as np
import pytest

import block_ref as R

pytestmark = pytest.mark.gpu


def frequencies(skv, dim, theta=10000.0, kind=0, factor=1.0, original=0, low=0.0, high=0.0):
    half = dim // 2
    base = theta * factor ** (dim / (dim - 2)) if kind == skv.ROPE_THETA else theta
    f = base ** (-np.arange(half) / half)
    if kind == skv.ROPE_LINEAR:
        f = f / factor
    if kind == skv.ROPE_BANDS:
        out = []
        for x in f:
            t = original * x / (2 * np.pi)
            s = (t - low) / (high - low)
            out.append(x if t >= high else x / factor if t <= low else (1 - s) * x / factor + s * x)
        f = np.array(out)
    return f


def rotated(x, position, f, halves, inverse, magnitude):
    """x [batch][n][heads][dim] with its first 2 * len(f) channels turned."""
    half = len(f)
    angle = (np.asarray(position)[:, None] + np.arange(x.shape[1]))[..., None, None] * f
    c, s = magnitude * np.cos(angle), magnitude * np.sin(angle) * (-1 if inverse else 1)
    y = x.copy()
    a, b = (slice(0, half), slice(half, 2 * half)) if halves else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def bound(t, want, x, half, halves, magnitude):
    """cos and sin rounded once, each product and their sum: 4 half-steps of 2^-24 of |a| + |b|, then the type's."""
    size = np.abs(x).max(-1, keepdims=True) * 2 * abs(magnitude)
    return 4 * 2.0 ** -24 * size + R.HALF_STEP[t] * (np.abs(want) + 2.0 ** -22 * size) + 2.0 ** -24 * (t == "f16")


SCALINGS = {"none": {}, "linear": dict(kind=1, factor=4.0), "theta": dict(kind=2, factor=2.5),
            "bands": dict(kind=3, factor=8.0, original=512, low=1.0, high=4.0)}


def make_scaling(skv, magnitude=1.0, kind=0, factor=1.0, original=0, low=0.0, high=0.0):
    return skv.RopeScaling(kind, factor, original, low, high, magnitude)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("heads,dim,rotary_dim,scaling,magnitude", [
    (1, 128, 128, "none", 1.0), (3, 64, 32, "linear", 1.0), (5, 80, 20, "bands", 1.25), (2, 128, 48, "theta", 1.0),
    (40, 128, 64, "bands", 1.0), (1, 2, 2, "none", 0.5), (7, 72, 64, "linear", 1.0)])
def test_rotary(skv, ctx, t, halves, heads, dim, rotary_dim, scaling, magnitude):
    rng = np.random.default_rng(dim + rotary_dim)
    sc = SCALINGS[scaling]
    table = skv.RotaryTable(ctx, rotary_dim, 40000, 10000.0, make_scaling(skv, magnitude, **sc))
    f = frequencies(skv, rotary_dim, **sc)
    size = 4 if t == "f32" else 2
    for batch, n, position, extra in ((1, 1, [39999], 0), (3, 17, [0, 31000, 5], 0), (2, 5, [100, 4], 24), (2, 3, [1, 2], 1)):
        x = rng.standard_normal((batch, n, heads * dim + extra))
        raw, x = R.typed(x, t)
        rows = x[..., :heads * dim].reshape(batch, n, heads, dim)
        dx = ctx.to_device(raw)
        for inverse in (False, True):
            dout = ctx.to_device(np.full(batch * n * (heads * dim + extra) * size, 0xee, np.uint8))
            skv.swiftkv_rotary(ctx, table, dx, dout, position, heads, dim, n=n, dtype=getattr(skv, t.upper()), halves=halves,
                               inverse=inverse, x_stride=heads * dim + extra, out_stride=heads * dim + extra)
            ctx.synchronize()
            got = dout.download(np.uint8, (batch, n, (heads * dim + extra) * size))
            assert (got[..., heads * dim * size:] == 0xee).all()
            got = R.values_of(got[..., :heads * dim * size], t, rows.shape)
            want = rotated(rows, position, f, halves, inverse, magnitude)
            err = np.abs(got - want)
            assert (err <= bound(t, want, rows, rotary_dim // 2, halves, magnitude)).all(), err.max()
            np.testing.assert_array_equal(got[..., rotary_dim:], rows[..., rotary_dim:])


def test_in_place_and_back(skv, ctx):
    """Turned in place, then back: what rounding leaves."""
    rng = np.random.default_rng(1)
    table = skv.RotaryTable(ctx, 64, 300)
    raw, x = R.typed(rng.standard_normal((2, 100, 6, 64)), "f32")
    dx = ctx.to_device(raw)
    for inverse in (False, True):
        skv.swiftkv_rotary(ctx, table, dx, dx, [200, 3], 4, 64, n=100, dtype=skv.F32, inverse=inverse, x_stride=384,
                           out_stride=384)
    ctx.synchronize()
    got = dx.download(np.float32, x.shape)
    np.testing.assert_array_equal(got[:, :, 4:], x[:, :, 4:])
    # c^2 + s^2 is 1 but for cos and sin rounded once (2 half-steps of the pair), and each turn rounds 3 times more
    assert np.abs(got - x).max() <= 10 * 2.0 ** -24 * 2 * np.abs(x).max()


def test_inverse_is_the_gradient(skv, ctx):
    """<g, turn(x + d) - turn(x - d)> / 2 against <inverse turn(g), d>: the rotation is linear, so both are exact but
    for rounding, with a magnitude other than 1 too."""
    rng = np.random.default_rng(2)
    for halves in (False, True):
        table = skv.RotaryTable(ctx, 32, 64, scaling=make_scaling(skv, 1.5))
        x, d, g = (rng.standard_normal((1, 4, 2, 64)) for _ in range(3))

        def turn(y, inverse=False):
            raw, _ = R.typed(y, "f32")
            buf, out = ctx.to_device(raw), ctx.alloc(raw.size)
            skv.swiftkv_rotary(ctx, table, buf, out, 60, 2, 64, n=4, dtype=skv.F32, halves=halves, inverse=inverse)
            ctx.synchronize()
            return out.download(np.float32, y.shape).astype(np.float64)

        diff = (g * (turn(x + d) - turn(x - d))).sum() / 2
        grad = (turn(g, True) * d).sum()
        size = np.abs(g).sum() * 1.5 * 2 * (np.abs(x).max() + np.abs(d).max())
        assert abs(diff - grad) <= 8 * 2.0 ** -24 * size


def test_more_sequences_than_a_launch_takes(skv, ctx):
    rng = np.random.default_rng(3)
    table = skv.RotaryTable(ctx, 16, 1000)
    position = rng.integers(0, 990, 600).tolist()
    raw, x = R.typed(rng.standard_normal((600, 2, 1, 16)), "f32")
    dx = ctx.to_device(raw)
    skv.swiftkv_rotary(ctx, table, dx, dx, position, 1, 16, n=2, dtype=skv.F32)
    ctx.synchronize()
    want = rotated(x, position, frequencies(skv, 16), True, False, 1.0)
    assert (np.abs(dx.download(np.float32, x.shape) - want) <= bound("f32", want, x, 8, True, 1.0)).all()


def test_scaled_q17_table(skv, ctx, oracle):
    """The step's own table with scaled frequencies: RNE(2^17 m cos|sin); unscaled it is the closed form's."""
    import helpers
    plain = skv.RopeLut.generate(ctx, 300).export()
    assert skv.RopeLut.generate_scaled(ctx, None, 300).export() == plain
    assert skv.RopeLut.generate_scaled(ctx, skv.RopeScaling(), 300).export() == plain
    # linear scaling by 2: position 2p of the scaled table is position p of the plain one
    lut = skv.RopeLut.generate_scaled(ctx, skv.RopeScaling(skv.ROPE_LINEAR, 2.0), 600)
    scaled = np.frombuffer(lut.export(), np.uint8).reshape(600, -1)
    np.testing.assert_array_equal(scaled[::2], np.frombuffer(plain, np.uint8).reshape(300, -1))


def test_refusals(skv, ctx):
    table = skv.RotaryTable(ctx, 32, 100)
    buf = ctx.alloc(1 << 16)

    def refused(code, *a, **k):
        with pytest.raises(skv.SwiftKVError) as e:
            skv.swiftkv_rotary(ctx, table, *a, dtype=k.pop("dtype", skv.F32), **k)
        assert e.value.code == code, str(e.value)

    refused(skv.ERANGE, buf, buf, 100, 1, 32)
    refused(skv.ERANGE, buf, buf, 95, 1, 32, n=6)
    refused(skv.ERANGE, buf, buf, -1, 1, 32)
    refused(skv.EINVAL, buf, buf, 0, 1, 16)
    refused(skv.EINVAL, buf, buf, 0, 0, 32)
    refused(skv.EINVAL, None, buf, 0, 1, 32)
    refused(skv.EINVAL, buf, buf, 0, 2, 32, x_stride=63)
    refused(skv.EINVAL, buf, buf, 0, 1, 32, out_stride=64)
    refused(skv.EINVAL, buf.ptr + 2, buf, 0, 1, 32)
    refused(skv.EINVAL, buf, buf, 0, 1, 32, dtype=7)
    skv.swiftkv_rotary(ctx, table, buf, buf, 99, 1, 32, n=0, dtype=skv.F32)
    for bad in ((31, 10), (0, 10), (258, 10), (32, 0), (32, skv.ROTARY_MAX_POSITIONS + 1)):
        with pytest.raises(skv.SwiftKVError):
            skv.RotaryTable(ctx, *bad)
    for bad in (skv.RopeScaling(9, 2.0), skv.RopeScaling(1, 0.5), skv.RopeScaling(3, 2.0, 0, 1.0, 4.0),
                skv.RopeScaling(3, 2.0, 4096, 4.0, 1.0), skv.RopeScaling(1, float("nan"))):
        with pytest.raises(skv.SwiftKVError):
            skv.RotaryTable(ctx, 32, 10, scaling=bad)
    with pytest.raises(skv.SwiftKVError):
        skv.RopeLut.generate_scaled(ctx, skv.RopeScaling(magnitude=2.0))
    with pytest.raises(skv.SwiftKVError):
        skv.RotaryTable(ctx, 32, 10, theta=1.0)
