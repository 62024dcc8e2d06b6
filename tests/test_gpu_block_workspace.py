"""What the block cache's attention allocates and when, and what is too large for a launch."""
import numpy as np
import pytest

from test_gpu_block import Rig

pytestmark = pytest.mark.gpu


def test_weights_allocate_once(skv, ctx):
    """The first call with weights takes what every later one needs: more queries allocate no more and can be captured."""
    rng = np.random.default_rng(19)
    rig = Rig(skv, ctx, "f32", 3, 4, 2, 64, 128)
    rig.append(rng, [0, 0, 0], 20)
    first = rig.cache.nbytes
    rig.check_attention(rng, [20, 20, 20], 1, weights=True)
    taken = 4 * 3 * 4 * skv.BLOCK_WEIGHT_QUERIES * (rig.cache.blocks + 1)
    assert rig.cache.nbytes == first + taken
    qr, q = rig.rows(rng, 3, 8, 4)
    dq, dout = ctx.to_device(qr), ctx.alloc(qr.size)
    before = np.zeros((3, 2, rig.cache.blocks), np.float32)
    dw = ctx.to_device(before)
    ctx.capture_begin()
    skv.swiftkv_block_attention(ctx, dq, None, None, rig.cache, 0, [13, 13, 13], dout, n=8, dtype=skv.F32, weights=dw)
    graph = ctx.capture_end()
    for n in (2, 8, 5):
        rig.check_attention(rng, [21 - n] * 3, n, append=False, weights=True)
    for _ in range(2):
        graph.launch()
    ctx.synchronize()
    assert rig.cache.nbytes == first + taken
    out, after = dout.download(np.float32, q.shape).astype(np.float64), dw.download(np.float32, before.shape)
    rig.compare(q, [13, 13, 13], 8, out, before, after / 2)
    graph.close()


def test_more_workgroups_than_a_launch_takes(skv, ctx):
    """Refused before the rows are appended or a tensor is read."""
    cache = skv.BlockCache(ctx, 1, 1, 256 * 64, 256, 64, 16384)
    k = np.random.default_rng(20).standard_normal((1, 256 * 64)).astype(np.float32)
    buf = ctx.to_device(k)
    skv.swiftkv_block_append(ctx, buf, buf, cache, 0, 0, dtype=skv.F32)
    got = ctx.alloc(4 * 256 * 64), ctx.alloc(4 * 256 * 64)
    values = []
    for _ in range(2):
        skv.swiftkv_block_values(ctx, cache, 0, 0, *got, dtype=skv.F32)
        ctx.synchronize()
        values.append(got[0].download(np.float32, k.shape))
        with pytest.raises(skv.SwiftKVError) as e:
            skv.swiftkv_block_attention(ctx, buf, buf, buf, cache, 0, 0, buf, n=16384, dtype=skv.F32)
        assert e.value.code == skv.ERANGE
    np.testing.assert_array_equal(*values)
    assert np.abs(values[0] - k).max() <= np.abs(k).max() / 64
