"""The paged cache on the GPU against its definition in 64 bits: rotated appends, attention of chains and trees, kept
paths, shared pages, and what the entries refuse."""
import numpy as np
import pytest

import block_ref as R
import paged_ref as P

pytestmark = pytest.mark.gpu


ROTATIONS = {"none": None, "halves": (64, True), "pairs": (32, False), "pairs_all": (64, False), "halves_48": (48, True),
             "halves_20": (20, True)}


def rotation(name):
    return None if ROTATIONS[name] is None else P.Rotation(ROTATIONS[name][0], halves=ROTATIONS[name][1])


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("name", list(ROTATIONS))
def test_append_and_values(skv, ctx, t, dim, name):
    """Rows one at a time and many at once, across steps and pages in any order; rows that no call wrote stay."""
    rig = P.Rig(skv, ctx, t, 4, 2, dim, batch=3, capacity=250, rotation=rotation(name), seed=dim)
    rig.map_all()
    at = [0, 1, 30]
    for n in (1, 2, 5, 31, 64, 1, 100):
        rig.append(at, n)
        at = [p + n for p in at]
    rig.check_values()
    rig.append([7, -1, 3], 9)           # over rows that are there; one sequence skipped
    rig.check_values()


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("name", ["halves", "pairs"])
def test_append_trees(skv, ctx, t, name):
    """A tree's rows lie in order and are turned by depth; rows without a token are not written."""
    rig = P.Rig(skv, ctx, t, 4, 2, 128, batch=4, capacity=256, rotation=rotation(name), seed=3)
    rig.map_all()
    rng = np.random.default_rng(5)
    for n, at in ((1, [0, 5, 63, 64]), (7, [1, 60, 127, 0]), (64, [100, 31, 0, 190]), (33, [3, -1, 200, 7])):
        trees = [P.random_tree(rng, n, c) for c in (n, (n + 1) // 2, n, 0)]
        rig.append(at, n, trees)
    rig.check_values()


def test_rows_of_a_fused_projection(skv, ctx):
    """q, k and v as parts of one projection's rows, out as a part of wider rows."""
    rig = P.Rig(skv, ctx, "bf16", 4, 2, 64, batch=2, capacity=128, rotation=rotation("halves"), seed=8)
    rig.map_all()
    rig.append([0, 0], 40)
    n, width, wide = 3, 8 * 64 + 8, 4 * 64 + 24
    raw, x = rig.random(2, n, width)
    fused = ctx.to_device(raw)
    out = ctx.to_device(np.full((2, n, wide), 0x7b7b, np.uint16))
    skv.swiftkv_paged_attention(ctx, fused.ptr, fused.ptr + 2 * 256, fused.ptr + 2 * 384, rig.cache, 0, [40, 11], out, n=n,
                                table=rig.table, q_stride=width, k_stride=width, v_stride=width, out_stride=wide)
    ctx.synchronize()
    q, k, v = (x[..., a:b].reshape(2, n, -1, 64) for a, b in ((0, 256), (256, 384), (384, 512)))
    rig.note([40, 11], k, v)
    got = out.download(np.uint16, (2, n, wide))
    assert (got[..., 256:] == 0x7b7b).all()
    rig.compare(q, R.values_of(got[..., :256].copy().view(np.uint8), "bf16", (2, n, 4, 64)), [40, 11])
    rig.check_values()


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(4, 4), (8, 2), (5, 1), (16, 1), (33, 1), (64, 1)])
def test_chains(skv, ctx, t, dim, heads, kv):
    """One token and more, from empty caches on, ending inside and at the ends of steps and pages."""
    rig = P.Rig(skv, ctx, t, heads, kv, dim, batch=3, capacity=320, rotation=P.Rotation(dim), seed=heads)
    rig.map_all()
    at = [0, 0, 0]
    for n in (1, 1, 30, 31, 1, 2, 3, 5, 9):
        rig.check_attention(at, n)
        at = [p + n for p in at]
    rig.check_attention([0, -1, at[2]], 40)
    rig.check_attention([64, 17, -1], 4, append=False)
    rig.check_values()


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 2), (5, 1), (16, 2)])
def test_trees(skv, ctx, t, dim, heads, kv):
    """Trees of 1 to 64 tokens and of different numbers a sequence, onto none and many cached tokens."""
    rig = P.Rig(skv, ctx, t, heads, kv, dim, batch=4, capacity=512, rotation=P.Rotation(dim, halves=dim == 64), seed=heads)
    rig.map_all()
    rig.append([0, 0, 0, 0], 400)
    rng = np.random.default_rng(heads)
    for n, at in ((1, [0, 31, 64, 399]), (2, [1, 63, 100, -1]), (3, [0, 30, 400, 7]), (8, [0, 31, 260, 400]), (13, [25, 90, 0, 57]),
                  (26, [0, 50, 399, 111]), (64, [0, 96, 33, 400])):
        trees = [P.random_tree(rng, n, c, deep) for c, deep in ((n, 0.5), (n, 0.0), ((n + 1) // 2, 0.9), (max(n - 3, 0), 0.5))]
        rig.check_attention(at, n, trees)
        rig.check_attention(at, n, trees, append=False)
    rig.check_values()


@pytest.fixture
def forced(ctx, request):
    ctx.set_paged_rows(request.param)
    yield request.param
    ctx.set_paged_rows(0)


every_shape = pytest.mark.parametrize("forced", [32, 48, 64, 128, 256], indirect=True)


@every_shape
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_every_shape(skv, ctx, t, dim, forced):
    """Each kernel for more than 16 rows on trees and chains of few and many rows, short and long sequences, rows that
    fill no chunk, splits of one step and of many; repeated calls give the same bits."""
    rig = P.Rig(skv, ctx, t, 10, 2, dim, batch=3, capacity=1600, rotation=P.Rotation(dim, halves=dim == 64), seed=forced)
    rig.map_all()
    rig.append([0, 0, 0], 1500)
    rng = np.random.default_rng(forced)
    try:
        for n, at in ((4, [0, 31, 1500]), (13, [700, -1, 64]), (64, [1500, 0, 333]), (27, [90, 1023, 5])):
            for split in (0, 256):
                ctx.set_split_tokens(split)
                trees = [P.random_tree(rng, n, c, deep) for c, deep in ((n, 0.5), ((n + 1) // 2, 0.0), (n, 0.9))]
                q, k, v = (rig.random(3, n, h, dim)[1] for h in (10, 2, 2))
                first, out = rig.attend(at, n, trees, q=q, k=k, v=v)
                rig.compare(first, out, at, trees)
                rig.check_values()
                np.testing.assert_array_equal(rig.attend(at, n, trees, q=q, k=k, v=v)[1], out)
                rig.check_attention(at, n)
        ctx.set_split_tokens(0)
        rig.check_attention([3, 0, 900], 150)
        rig.check_attention([1000, 64, -1], 150, scale=-0.2)
        rig.check_values()
    finally:
        ctx.set_split_tokens(0)


@every_shape
def test_long_scans_of_every_shape(skv, ctx, forced):
    """More steps than a window of the table holds, in one split and in several."""
    rig = P.Rig(skv, ctx, "bf16", 4, 1, 64, batch=1, capacity=17000, rotation=P.Rotation(64, 17000), seed=forced)
    rig.map_all()
    rig.append([0], 16900)
    try:
        for split in (32768, 8192, 0):
            ctx.set_split_tokens(split)
            rig.check_attention([16900], 9)
            rig.check_attention([16389], 70)
    finally:
        ctx.set_split_tokens(0)


@every_shape
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_no_numbers_in_every_shape(skv, ctx, t, forced, what):
    """A value that is no number reaches the tokens that see it, wherever in a step or a turn it stands."""
    dim, n = 64, 40
    rig = P.Rig(skv, ctx, t, 2, 1, dim, capacity=512, seed=1)
    rig.map_all()
    junk = np.full((1, 512, 1, dim), what)
    for p in (0, 77, 380):
        rig.append([0], 512, k=junk, v=junk)
        rig.append([0], p) if p else None
        tree = [[-1] + [(i - 1) // 2 for i in range(1, n)]]
        own, _, _ = P.places(tree[0])
        q, k, v = (rig.random(1, n, h, dim)[1] for h in (2, 1, 1))
        first, good = rig.attend([p], n, tree, q=q, k=k, v=v)
        rig.compare(first, good, [p], tree)
        for node in (0, 3, 17, 39):
            bad = v.copy()
            bad[0, node, 0, [1, 40]] = what
            _, out = rig.attend([p], n, tree, q=q, k=k, v=bad)
            sees = own[:, node]
            np.testing.assert_array_equal(out[0, ~sees], good[0, ~sees])
            np.testing.assert_array_equal(out[0][:, :, 2:40], good[0][:, :, 2:40])
            assert (np.isnan(out[0, sees][:, :, [1, 40]]) if np.isnan(what) else out[0, sees][:, :, [1, 40]] == what).all()


def test_a_chain_as_a_tree(skv, ctx):
    """The same tokens with parents written out and without give the same outputs, bit for bit."""
    rig = P.Rig(skv, ctx, "bf16", 8, 2, 128, batch=2, capacity=640, rotation=P.Rotation(128), seed=1)
    rig.map_all()
    rig.append([0, 0], 500)
    for n in (1, 4, 8, 16, 40):
        q, k, v = (rig.random(2, n, h, 128)[1] for h in (8, 2, 2))
        _, a = rig.attend([500, 33], n, q=q, k=k, v=v)
        _, b = rig.attend([500, 33], n, [P.chain(n)] * 2, q=q, k=k, v=v)
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("n", [1, 7, 13, 40])
def test_splits(skv, ctx, t, n):
    """Long sequences of different lengths, in the plan's splits and in forced ones; repeated calls give the same
    bits."""
    rig = P.Rig(skv, ctx, t, 4, 1, 64, batch=3, capacity=9000, rotation=P.Rotation(64, 9000), seed=n)
    rig.map_all()
    rig.append([0, 0, 0], 8900)
    rng = np.random.default_rng(n)
    trees = [P.random_tree(rng, n, c) for c in (n, n, (n + 1) // 2)]
    q, k, v = (rig.random(3, n, h, 64)[1] for h in (4, 1, 1))
    at = [8900, 2047, 300]
    try:
        for split in (0, 256, 1024):
            ctx.set_split_tokens(split)
            first, out = rig.attend(at, n, trees, q=q, k=k, v=v)
            rig.compare(first, out, at, trees)
            for _ in range(5):
                np.testing.assert_array_equal(rig.attend(at, n, trees, q=q, k=k, v=v)[1], out)
    finally:
        ctx.set_split_tokens(0)


@pytest.mark.parametrize("n", [1, 5, 8, 16])
def test_own_append_and_one_before(skv, ctx, n):
    """The attention's own append and swiftkv_paged_append leave the same rows and the same outputs."""
    rng = np.random.default_rng(n)
    rig = P.Rig(skv, ctx, "bf16", 4, 2, 128, batch=2, capacity=320, rotation=P.Rotation(128), seed=n)
    rig.map_all()
    rig.append([0, 0], 200)
    trees = [P.random_tree(rng, n, c) for c in (n, (n + 1) // 2)]
    q, k, v = (rig.random(2, n, h, 128)[1] for h in (4, 2, 2))
    at = [190, 61]
    _, a = rig.attend(at, n, trees, q=q, k=k, v=v)
    rig.check_values()
    rig.append([0, 0], 260)
    rig.append(at, n, trees, k=k, v=v)
    rig.check_values()
    first, b = rig.attend(at, n, trees, q=q, append=False)
    rig.compare(first, b, at, trees)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("heads", [1, 4, 8])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_what_is_not_seen_does_not_count(skv, ctx, t, heads, what):
    """Rows that are no numbers reach the tokens that see them and no others: drafted tokens off a token's path, and
    rows that lie behind a sequence's last token."""
    dim, n, p = 64, 6, 75
    rig = P.Rig(skv, ctx, t, heads, 1, dim, batch=1, capacity=256, seed=heads)
    rig.map_all()
    junk = np.full((1, 256, 1, dim), what)
    rig.append([0], 256, k=junk, v=junk)
    rig.append([0], p)
    #        0 - 1 - 3        token 2 is bad: it and its child 4 see it
    #          \ 2 - 4 ; 5 a root of its own
    tree = [[-1, 0, 0, 1, 2, -1]]
    q, k, v = (rig.random(1, n, h, dim)[1] for h in (heads, 1, 1))
    clean, _ = rig.attend([p], n, tree, q=q, k=k, v=v)
    good = rig.attend([p], n, tree, q=q, k=k, v=v)[1]
    rig.compare(clean, good, [p], tree)
    bad_v, bad_k = v.copy(), k.copy()
    bad_v[0, 2, 0, 3:9] = what
    _, out = rig.attend([p], n, tree, q=q, k=k, v=bad_v)
    unseen, seeing = [0, 1, 3, 5], [2, 4]
    np.testing.assert_array_equal(out[0, unseen], good[0, unseen])
    np.testing.assert_array_equal(np.isnan(out[0, seeing][:, :, 3:9]), np.isnan(what))
    if not np.isnan(what):
        assert (out[0, seeing][:, :, 3:9] == what).all()
    keep = np.r_[0:3, 9:dim]
    np.testing.assert_array_equal(out[0, seeing][:, :, keep], good[0, seeing][:, :, keep])
    bad_k[0, 2, 0, 5] = np.nan
    _, out = rig.attend([p], n, tree, q=q, k=bad_k, v=v)
    np.testing.assert_array_equal(out[0, unseen], good[0, unseen])
    assert np.isnan(out[0, seeing]).all()
    # a chain: the tokens before the bad one
    _, good = rig.attend([p], n, q=q, k=k, v=v)
    _, out = rig.attend([p], n, q=q, k=bad_k, v=bad_v)
    np.testing.assert_array_equal(out[0, :2], good[0, :2])
    assert np.isnan(out[0, 2:]).all()


@pytest.mark.parametrize("heads", [4, 8])
def test_queries_that_are_no_numbers(skv, ctx, heads):
    """Their own rows are NaN, the others as they were."""
    rig = P.Rig(skv, ctx, "bf16", heads, 1, 64, capacity=256, seed=2)
    rig.map_all()
    rig.append([0], 100)
    q = rig.random(1, 3, heads, 64)[1]
    _, good = rig.attend([97], 3, q=q, append=False)
    bad = q.copy()
    bad[0, 1, heads - 1, 7] = np.nan
    _, out = rig.attend([97], 3, q=bad, append=False)
    assert np.isnan(out[0, 1, heads - 1]).all()
    good[0, 1, heads - 1] = out[0, 1, heads - 1]
    np.testing.assert_array_equal(out, good)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("n", [1, 4, 20])
def test_scores_that_rise_and_fall(skv, ctx, t, n):
    """Large scores in rising and in falling order, of either sign of the scale, with a few tokens far above the rest
    and with many equal ones."""
    rig = P.Rig(skv, ctx, t, 4, 2, 64, capacity=1024, seed=n)
    rig.map_all()
    tokens = 900
    for slope in (-1.0, 1.0, 0.0):
        k = rig.rng.standard_normal((1, tokens, 2, 64)) * 0.1 + slope * np.linspace(-4, 4, tokens)[None, :, None, None]
        rig.append([0], tokens, k=k, v=rig.rng.standard_normal((1, tokens, 2, 64)) * 50)
        for scale in (0.0, 0.5, -0.125, 2.0 ** -40):
            q = 0.5 + rig.rng.random((1, n, 4, 64))
            rig.check_attention([tokens - n], n, append=False, scale=scale, q=q)


def test_one_token_and_none(skv, ctx):
    """A first token sees itself alone; a call of no tokens changes nothing."""
    rig = P.Rig(skv, ctx, "f16", 2, 1, 64, batch=2, capacity=64, rotation=P.Rotation(64), seed=4)
    rig.map_all()
    v = rig.random(2, 1, 1, 64)[1]
    _, out = rig.attend([0, 0], 1, v=v)
    np.testing.assert_array_equal(out, np.repeat(v, 2, 2))
    skv.swiftkv_paged_append(ctx, ctx.alloc(16), ctx.alloc(16), rig.cache, 0, [0, 0], n=0)
    skv.swiftkv_paged_attention(ctx, rig.ctx.alloc(16), None, None, rig.cache, 0, [0, 0], rig.ctx.alloc(16), n=0)
    _, out = rig.attend([1, -5], 2, [[-2, -2], [-1, 0]])
    assert (out == 0).all()
    rig.check_values()


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_keep(skv, ctx, t, dim):
    """Accepted rows move, in the layers that are named; all others stay."""
    rig = P.Rig(skv, ctx, t, 2, 2, dim, batch=4, layers=3, capacity=256, seed=dim)
    rig.map_all()
    for layer in range(3):
        rig.append([0] * 4, 256, layer=layer)
    rig.keep([10, 60, 127, 0], [[0, 1, 2, 3], [0, 2, 3, 7], [5, 6, -1, -1], [-1] * 4])
    rig.check_values()
    rig.keep([10, -3, 64, 191], [list(range(64)), list(range(64)), [63] + [-1] * 63, list(range(1, 64, 2)) + [-1] * 32])
    rig.check_values()
    rig.keep([33, 1, 2, 3], [[9], [0], [1], [63]], layer0=1, layers=2)
    rig.keep([100], [[2, 4, 6, 8, 10, 12, 14, 16]], layer0=2, layers=1, seq0=3)
    rig.check_values()


@pytest.mark.parametrize("t,dim,capacity", [("bf16", 64, 128), ("f16", 128, 64)])
def test_few_rows_of_many_heads(skv, ctx, t, dim, capacity):
    """Enough heads that a workgroup takes four: rows kept and read at every place in an octet, over pages' ends."""
    layers, batch = 32, 16
    rig = P.Rig(skv, ctx, t, 8, 8, dim, batch=batch, layers=layers, capacity=capacity, seed=dim)
    rig.map_all()
    for layer in range(layers):
        rig.append([0] * batch, capacity, layer=layer)
    places = [(5 * b) % (capacity - 9) for b in range(batch - 2)] + [-1, capacity - 9]
    for n in range(1, 10):
        got = rig.values(places, n, 0, layers)
        for b, p in enumerate(places):
            for layer in range(layers):
                for g, w in zip(got, rig.rows(layer, b, np.arange(max(p, 0), max(p, 0) + n))):
                    if p < 0:
                        assert np.isnan(g[layer, b]).all()       # as they were, 0xff
                    else:
                        np.testing.assert_array_equal(g[layer, b], w)
    room = min(capacity, 64)
    paths = [sorted(int(a) for a in rig.rng.choice(room - 9, 8, replace=False)) for _ in range(batch)]
    rig.keep([min(p, capacity - room + 9) if p >= 0 else p for p in places], paths)
    rig.check_values()


@pytest.mark.parametrize("n", [1, 5, 40, 100])
def test_sequences_that_sit_out(skv, ctx, n):
    """All of a call's sequences, or all but one long one."""
    rig = P.Rig(skv, ctx, "bf16", 8, 2, 64, batch=64, pages=60, capacity=3200, rotation=P.Rotation(64), seed=n)
    rig.map(40, list(range(50)))
    rig.append([-1] * 40 + [0] + [-1] * 23, 3000)
    _, out = rig.attend([-1] * 64, n)
    assert (out == 0).all()
    rig.check_attention([-1] * 40 + [2990] + [-7] * 23, n)


@pytest.mark.parametrize("heads", [4, 20, 40, 64])
def test_the_longest_sequence(skv, ctx, heads):
    rig = P.Rig(skv, ctx, "f16", heads, 1, 64, capacity=131072, seed=heads)
    rig.map_all()
    rig.append([0], 131072)
    rig.check_attention([131071], 1)
    if heads < 40:
        rig.check_attention([131072 - 9], 9, [[-1] + [(i - 1) // 2 for i in range(1, 9)]])


def test_shared_prefix(skv, ctx):
    """Sequences that share their first pages, each with a copy of the one that it goes on in."""
    rig = P.Rig(skv, ctx, "bf16", 4, 2, 64, batch=3, pages=9, layers=2, capacity=256, rotation=P.Rotation(64), seed=6)
    rig.map(0, [4, 2])
    for layer in range(2):
        rig.append([0], 100, layer=layer)
    for b, own in ((1, 7), (2, 0)):
        rig.map(b, [4])
        rig.cache.copy(2, own)
        for s in rig.store:
            s[:, own] = s[:, 2]
        rig.map(b, [own], first=1)
    rng = np.random.default_rng(0)
    for layer in range(2):
        trees = [P.random_tree(rng, 20, c) for c in (20, 11, 17)]
        rig.check_attention([100, 100, 100], 20, trees, layer=layer)
    rig.check_values()
    for call in (lambda: rig.append([63], 1), lambda: rig.attend([60, 100, 100], 5),
                 lambda: rig.keep([62], [[1]]), lambda: rig.cache.copy(2, 4)):
        with pytest.raises(skv.SwiftKVError) as e:
            call()
        assert e.value.code == skv.ESTATE
    rig.keep([62], [[0, 1, 4]])          # rows 0 and 1 stay on the shared page and 4 moves within its own
    rig.check_values()


def test_drafting_equals_decoding(skv, ctx):
    """Trees attended, their accepted paths kept: the cache then holds what decoding those tokens one by one leaves,
    and the accepted tokens' outputs agree."""
    layers, heads, kv, dim, prompt = 2, 8, 2, 128, 150
    rot = P.Rotation(dim)
    rigs = [P.Rig(skv, ctx, "bf16", heads, kv, dim, batch=2, layers=layers, capacity=320, rotation=rot, seed=s) for s in (1, 2)]
    drafted, plain = rigs
    rng = np.random.default_rng(9)
    for rig in rigs:
        rig.map_all()
    for layer in range(layers):
        k, v = (rng.standard_normal((2, prompt, kv, dim)) for _ in "kv")
        for rig in rigs:
            rig.append([0, 0], prompt, layer=layer, k=k, v=v)
    at = [prompt, prompt]
    for n in (6, 13, 1, 40):
        trees = [P.random_tree(rng, n, c) for c in (n, max(1, n // 2))]
        paths = []
        for tree in trees:      # from a token up to the root
            i, path = int(rng.integers(0, sum(p != P.NONE for p in tree))), []
            while i >= 0:
                path.insert(0, i)
                i = tree[i]
            paths.append(path)
        m = max(map(len, paths))
        for layer in range(layers):
            q, k, v = (rng.standard_normal((2, n, h, dim)) for h in (heads, kv, kv))
            _, out = drafted.attend(at, n, trees, layer=layer, q=q, k=k, v=v)
            for b, path in enumerate(paths):
                for j, i in enumerate(path):
                    pos = [-1, -1]
                    pos[b] = at[b] + j
                    one, got = plain.attend(pos, 1, layer=layer, q=q[:, [i]], k=k[:, [i]], v=v[:, [i]])
                    plain.compare(one, out[:, [i]] * (np.array(pos) >= 0)[:, None, None, None], pos, layer=layer, call=n)
        at = drafted.keep(at, [p + [-1] * (m - len(p)) for p in paths])
        for b in range(2):
            for layer in range(layers):
                for name, a, c in zip("kv", drafted.rows(layer, b, np.arange(at[b])), plain.rows(layer, b, np.arange(at[b]))):
                    np.testing.assert_array_equal(a, c, err_msg=name)
        drafted.check_values()
        plain.check_values()


def test_more_sequences_than_a_launch_holds(skv, ctx):
    """70 sequences, and trees of 64 tokens that a launch holds 32 of."""
    rig = P.Rig(skv, ctx, "f16", 2, 1, 64, batch=70, capacity=128, rotation=P.Rotation(64), seed=7)
    rig.map_all()
    rng = np.random.default_rng(1)
    at = [int(x) for x in rng.integers(-1, 60, 70)]
    rig.append([0] * 70, 60)
    rig.check_attention(at, 1)
    rig.check_attention(at, 64, [P.random_tree(rng, 64, int(c)) for c in rng.integers(0, 65, 70)])
    rig.append([max(p, 0) for p in at], 64, [P.random_tree(rng, 64, int(c)) for c in rng.integers(0, 65, 70)])
    rig.keep(at, [sorted(int(a) for a in rng.choice(64, 40, replace=False)) + [-1] * (i % 3) + [-1] * (2 - i % 3)
                  for i in range(70)])
    rig.check_values()


def test_offsets_beyond_32_bits(skv, ctx):
    """Pages more than 4 GiB from the first, in the second of two layers."""
    pages = 20000
    cache = skv.PagedCache(ctx, 2, pages, 1, 8, 8, 128, 256, skv.BF16)
    assert cache.nbytes > 2 ** 33
    cache.map(0, [pages - 1, 3, pages - 2])
    rng = np.random.default_rng(0)
    k, v = (R.typed(rng.standard_normal((1, 150, 8, 128)), "bf16") for _ in "kv")
    q = R.typed(rng.standard_normal((1, 1, 8, 128)), "bf16")
    skv.swiftkv_paged_append(ctx, ctx.to_device(k[0]), ctx.to_device(v[0]), cache, 1, [0], n=150)
    bufs = [ctx.alloc(k[0].nbytes) for _ in "kv"]
    skv.swiftkv_paged_values(ctx, cache, 1, [0], *bufs, n=150)
    out = ctx.alloc(q[0].nbytes)
    skv.swiftkv_paged_attention(ctx, ctx.to_device(q[0]), None, None, cache, 1, [149], out)
    ctx.synchronize()
    for buf, x in zip(bufs, (k, v)):
        np.testing.assert_array_equal(buf.download(np.uint8, x[0].shape), x[0])
    got = R.values_of(out.download(np.uint8, q[0].shape), "bf16", (8, 128))
    for h in range(8):
        want, weighted, size = P.attention(q[1][0, 0, [h]], k[1][0, :, h], v[1][0, :, h], np.ones((1, 150), bool), 128 ** -0.5)
        off = P.bound("bf16", 1, 128, want, weighted, size, 150, np.abs(v[1]).max())
        assert (np.abs(got[h] - want) <= off).all()
    cache.close()


def test_captured_steps(skv, ctx):
    """A tree's step through two layers and the move of its path in a graph: every replay, with eager work between
    them, gives the eager outputs."""
    rig = P.Rig(skv, ctx, "bf16", 8, 2, 64, batch=2, layers=2, capacity=2200, rotation=P.Rotation(64), seed=11)
    rig.map_all()
    at, n, rng = [2000, 700], 12, np.random.default_rng(2)
    for layer in range(2):
        rig.append([0, 0], 2000, layer=layer)
    tree = [P.random_tree(rng, n), P.random_tree(rng, n, 5)]
    path = [[1, 4, 9, 11], [2, 3, -1, -1]]
    x = [[rig.random(2, n, h, 64) for h in (8, 2, 2)] for _ in range(2)]
    dev = [[ctx.to_device(raw) for raw, _ in row] for row in x]
    outs = [ctx.to_device(np.zeros(x[0][0][0].size, np.uint8)) for _ in range(2)]

    def step():
        for layer in range(2):
            skv.swiftkv_paged_attention(ctx, *dev[layer], rig.cache, layer, at, outs[layer], n=n, table=rig.table,
                                        parents=sum(tree, []))
        skv.swiftkv_paged_keep(ctx, rig.cache, 0, 2, at, sum(path, []), 4)

    def state():
        ctx.synchronize()
        return [o.download(np.uint8, (x[0][0][0].size,)) for o in outs] + rig.values([0, 0], 2048, 0, 2)

    step()
    eager = state()
    ctx.capture_begin()
    step()
    graph = ctx.capture_end()
    for turn in range(4):
        for layer in range(2):
            outs[layer].zero()
        rig.append([2000, 700], n, tree)                 # what the replay has to write again
        rig.attend([1500, 100], 3, append=False)         # the same workspace, other splits
        graph.launch()
        for a, b in zip(state(), eager):
            np.testing.assert_array_equal(a, b, err_msg=f"replay {turn}")
        with pytest.raises(skv.SwiftKVError):
            rig.cache.map(0, [10 ** 6])


def test_capture_refuses_the_table(skv, ctx):
    rig = P.Rig(skv, ctx, "bf16", 1, 1, 64, capacity=64, seed=0)
    ctx.capture_begin()
    try:
        for call in (lambda: rig.cache.map(0, [0]), lambda: skv.PagedCache(ctx, 1, 1, 1, 1, 1, 64, 64), rig.cache.close):
            handle = rig.cache.handle
            with pytest.raises(skv.SwiftKVError) as e:
                call()
            assert e.value.code == skv.ESTATE
            rig.cache.handle = handle
    finally:
        ctx.capture_end()
    with pytest.raises(skv.SwiftKVError) as e:
        rig.append([0], 1)
    assert e.value.code == skv.ESTATE                    # no page: the refused call mapped nothing


def test_two_contexts_at_once(skv):
    """Two contexts' calls in flight together, each split over workgroups and joined in its own workspace."""
    ctxs = [skv.Context(0) for _ in range(2)]
    rigs = [P.Rig(skv, c, "bf16", 8, 2, 128, capacity=4096, rotation=P.Rotation(128), seed=i) for i, c in enumerate(ctxs)]
    calls = []
    for rig, c in zip(rigs, ctxs):
        rig.map_all()
        rig.append([0], 4000)
        q = rig.random(1, 2, 8, 128)
        out = c.alloc(q[0].nbytes)
        calls.append((rig, c, q, c.to_device(q[0]), out))
    for _ in range(50):
        for rig, c, q, dq, out in calls:
            skv.swiftkv_paged_attention(c, dq, None, None, rig.cache, 0, [3998], out, n=2, table=rig.table)
    for rig, c, q, dq, out in calls:
        c.synchronize()
        rig.compare(q[1], R.values_of(out.download(np.uint8, q[0].shape), "bf16", q[1].shape), [3998])
        rig.cache.close()
    for c in ctxs:
        c.close()


def test_refusals(skv, ctx):
    rig = P.Rig(skv, ctx, "bf16", 4, 2, 64, batch=2, layers=2, capacity=200, rotation=P.Rotation(64, 150), seed=0)
    rig.map(0, [0, 1, 2])
    rig.map(1, [3])
    buf = ctx.alloc(1 << 20)
    A, S, E = skv.EINVAL, skv.ESTATE, skv.ERANGE
    other = skv.Context(0)
    far = skv.RotaryTable(other, 64, 100)
    wide = skv.RotaryTable(ctx, 128, 100)

    def append(at, n=1, layer=0, k=buf, v=buf, table=None, **how):
        return lambda: skv.swiftkv_paged_append(ctx, k, v, rig.cache, layer, at, n=n, table=table, **how)

    def attend(at, n=1, layer=0, q=buf, k=buf, v=buf, out=buf, table=None, **how):
        return lambda: skv.swiftkv_paged_attention(ctx, q, k, v, rig.cache, layer, at, out, n=n, table=table, **how)

    def keep(at, accepted, m, layer0=0, layers=2, **how):
        return lambda: skv.swiftkv_paged_keep(ctx, rig.cache, layer0, layers, at, accepted, m, **how)

    def create(layers=1, pages=1, batch=1, heads=1, kv=1, dim=64, length=64, dtype=skv.BF16):
        return lambda: skv.PagedCache(ctx, layers, pages, batch, heads, kv, dim, length, dtype)

    cases = [
        (append([192]), S), (append([256]), E), (append([255], 2), E), (append([0, 64]), S), (append([0, 0, 0]), E),
        (append([0], layer=2), E), (append([0], layer=-1), E), (append([0], seq0=2), E), (append([0], -1), E),
        (append([0], 257), E), (append([0], k=None), A), (append([0], v=None), A), (append([0], k=buf.ptr + 2), A),
        (append([0], k_stride=127), A), (append([0], v_stride=132), A), (append([0], table=far), A), (append([0], table=wide), A),
        (append([150], table=rig.table), E), (append([2 ** 31 - 1]), E),
        (append([149], 2, table=rig.table), E), (append([0], 2, parents=[0, -1]), A), (append([0], 2, parents=[-1, 1]), A),
        (append([0], 2, parents=[-2, -1]), A), (append([0], 2, parents=[-1, -3]), A), (append([0], 65, parents=[-1] * 65), E),
        (append([149], 2, table=rig.table, parents=[-1, 0]), E),
        (attend([192]), S), (attend([0, 64]), S), (attend([0], q=None), A), (attend([0], out=None), A), (attend([0], k=None), A),
        (attend([0], v=None), A), (attend([0], out=buf.ptr + 8), A), (attend([0], q_stride=255), A), (attend([0], scale=np.nan), A),
        (attend([0], scale=np.inf), A), (attend([0], scale=2.0 ** -110), A), (attend([0], 2, parents=[-1, 5]), A),
        (attend([0], 65, parents=[-1] * 65), E), (attend([191], 2, k=None, v=None), S), (attend([0], layer=2), E),
        (keep([0], [0, 0], 2), A), (keep([0], [1, 0], 2), A), (keep([0], [64], 1), A), (keep([0], [-2], 1), A),
        (keep([0], [-1, 0], 2), A), (keep([0], [0] * 65, 65), E), (keep([190], [2], 1), S), (keep([0], [0], 1, layers=3), E),
        (keep([0], [0], 1, layer0=2, layers=1), E), (keep([0, 0, 0], [0] * 3, 1), E), (keep([0], [0], 1, layers=0), E),
        (lambda: skv.swiftkv_paged_values(ctx, rig.cache, 0, [190], buf, buf, n=3), S),
        (lambda: skv.swiftkv_paged_values(ctx, rig.cache, 0, [0], buf, None), A),
        (lambda: skv.swiftkv_paged_values(ctx, rig.cache, 1, [0], buf, buf, layers=2), E),
        (lambda: rig.cache.map(0, [8]), E), (lambda: rig.cache.map(0, [-2]), E), (lambda: rig.cache.map(2, [0]), E),
        (lambda: rig.cache.map(0, [0], first=4), E), (lambda: rig.cache.map(0, [0, 1, 2, 3, 4]), E), (lambda: rig.cache.map(0, [0], first=-1), E),
        (lambda: rig.cache.copy(0, 8), E), (lambda: rig.cache.copy(-1, 0), E),
        (lambda: ctx.set_paged_rows(16), A), (create(layers=0), A), (create(pages=0), A), (create(batch=0), A), (create(heads=3, kv=2), A), (create(heads=65), A),
        (create(dim=96), A), (create(length=0), A), (create(length=131073), A), (create(dtype=skv.F32), A), (create(dtype=7), A),
        (create(layers=256, pages=1 << 24, heads=256, kv=256, dim=128), skv.ENOMEM),
    ]
    for i, (call, code) in enumerate(cases):
        with pytest.raises(skv.SwiftKVError) as e:
            call()
        assert e.value.code == code, f"case {i}: {e.value}"
    for call in (append([0], 2, parents=[-1]), attend([0, 0], 1, parents=[-1]), keep([0], [0], 2), lambda: rig.cache.map(0, [0.5])):
        with pytest.raises(ValueError):
            call()
    rig.check_values()                                   # nothing was written
    mine = skv.PagedCache(other, 1, 1, 1, 1, 1, 64, 64)
    with pytest.raises(skv.SwiftKVError):
        skv.swiftkv_paged_append(ctx, buf, buf, mine, 0, [0])
    ctx.set_host_io(True)
    try:
        with pytest.raises(skv.SwiftKVError) as e:
            skv.swiftkv_paged_append(ctx, buf, buf, rig.cache, 0, [0])
        assert e.value.code == S
    finally:
        ctx.set_host_io(False)
    mine.close()
    far.close()
    other.close()


def test_pages_taken_and_given_back(skv, ctx):
    """A page goes from one sequence to another; what the former wrote behind the latter's last token is not seen."""
    rig = P.Rig(skv, ctx, "bf16", 2, 1, 64, batch=2, pages=2, capacity=128, seed=5)
    rig.map(0, [1, 0])
    junk = np.full((1, 128, 1, 64), np.nan)
    rig.append([0], 128, k=junk, v=junk)
    rig.map(0, [-1, -1])
    rig.map(1, [0, 1])
    rig.append([0], 70, seq0=1)
    rig.check_attention([70], 1, seq0=1)
    rig.check_attention([71], 5, [[-1, 0, 0, 1, 2]], seq0=1)
    with pytest.raises(skv.SwiftKVError):
        rig.append([0], 1)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("n", [1, 7, 33, 64])
def test_trees_without_tokens_come_first(skv, ctx, t, n):
    """Sequences that bring no tokens before and among ones that do, at every kind of place in a step, k and v in the
    middle of larger buffers: nothing of theirs changes, and the others' rows are as ever."""
    kv, dim = 2, 64
    rig = P.Rig(skv, ctx, t, 4, kv, dim, batch=5, capacity=256, rotation=P.Rotation(dim), seed=n)
    rig.map_all()
    rig.append([0] * 5, 190)
    rng = np.random.default_rng(n)
    for at in ([5, 63, 100, 190, 64], [31, 32, 0, 1, 127], [190, 96, 33, 5, 95]):
        trees = [P.random_tree(rng, n, c) for c in (0, 0, n, 0, (n + 1) // 2)]
        (kr, k), (vr, v) = (rig.random(7, n, kv, dim) for _ in "kv")
        row = 2 * n * kv * dim
        dk, dv = ctx.to_device(kr), ctx.to_device(vr)
        skv.swiftkv_paged_append(ctx, dk.ptr + row, dv.ptr + row, rig.cache, 0, at, n=n, table=rig.table, parents=sum(trees, []))
        ctx.synchronize()
        rig.note(at, k[1:6], v[1:6], trees)
        rig.check_values()
        rig.check_attention(at, n, trees)
        rig.check_values()


@every_shape
@pytest.mark.parametrize("halves", [True, False])
def test_the_end_of_the_rotary_table(skv, ctx, forced, halves):
    """Sequences as long as the table that bring no tokens, ones that sit out of calls of more tokens than the table has
    positions, and the last position itself."""
    dim, positions = 64, 150
    rig = P.Rig(skv, ctx, "bf16", 8, 2, dim, batch=3, capacity=320, rotation=P.Rotation(dim, positions, halves=halves), seed=forced)
    rig.map_all()
    rig.append([0] * 3, positions)
    rng = np.random.default_rng(forced)
    for n in (1, 9, 40):
        trees = [P.random_tree(rng, n, c) for c in (0, n, 0)]
        at = [positions, positions - n, positions]
        rig.append(at, n, trees)
        rig.check_values()
        rig.check_attention(at, n, trees)
        rig.check_attention(at, n, trees, append=False)
    star = [[-1] + [0] * 7, [-2] * 8, [-1] * 8]              # depths of 1, none and 0
    rig.check_attention([positions - 2, positions, positions - 1], 8, star)
    _, out = rig.attend([-1] * 3, 300)
    assert (out == 0).all()
    _, out = rig.attend([-1, -300, -7], 64, [P.chain(64)] * 3)
    assert (out == 0).all()
    rig.check_attention([0, -1, -1], positions)
    rig.check_values()


@pytest.mark.parametrize("n", [1, 7, 40])
def test_large_values(skv, ctx, n):
    """Values near bfloat16's largest, of equal and of different weights: their sums are far beyond FP32's range, their
    means are not."""
    tokens = 4096
    rig = P.Rig(skv, ctx, "bf16", 8, 2, 64, capacity=tokens, seed=n)
    rig.map_all()
    try:
        for k_size, v in ((0.0, 3e38), (0.0, -1e35), (1.0, 3e38), (1.0, None)):
            value = rig.rng.uniform(-3e38, 3e38, (1, tokens, 2, 64)) if v is None else np.full((1, tokens, 2, 64), v)
            rig.append([0], tokens, k=rig.rng.standard_normal((1, tokens, 2, 64)) * k_size, v=value)
            for split in (0, 256, 4096):
                ctx.set_split_tokens(split)
                out = rig.check_attention([tokens - n], n, append=False)
                assert np.isfinite(out).all()
    finally:
        ctx.set_split_tokens(0)


@every_shape
def test_large_values_in_every_shape(skv, ctx, forced):
    rig = P.Rig(skv, ctx, "bf16", 10, 2, 128, capacity=1600, seed=forced)
    rig.map_all()
    rig.append([0], 1500, v=np.full((1, 1500, 2, 128), 3e38))
    tree = [P.random_tree(np.random.default_rng(0), 20)]
    for how in (dict(parents=tree, v=np.full((1, 20, 2, 128), 3e38)), dict(parents=tree, v=np.full((1, 20, 2, 128), -3e38)), {}):
        rig.check_attention([1500], 20, **how)


@pytest.mark.parametrize("n", [1, 9])
def test_large_values_of_the_longest_sequence(skv, ctx, n):
    """All weights just below the 2^4 by which scores may lie above the reference value that the first ones set, of as
    many tokens as a sequence holds, in long splits and in the plan's."""
    tokens, dim = 131072, 64
    rig = P.Rig(skv, ctx, "bf16", 4, 1, dim, capacity=tokens, seed=0)
    rig.map_all()
    k = np.zeros((1, tokens, 1, dim))
    k[0, 256:, 0, 0] = 2.6875                # times log2(e): 3.877
    rig.append([0], tokens, k=k, v=np.full((1, tokens, 1, dim), 3e38))
    q = np.zeros((1, n, 4, dim))
    q[..., 0] = 1.0
    try:
        for split in (32768, 0):
            ctx.set_split_tokens(split)
            out = rig.check_attention([tokens - n], n, append=False, q=q, scale=1.0)
            assert np.isfinite(out).all()
    finally:
        ctx.set_split_tokens(0)


@pytest.mark.parametrize("n", [1, 40])
def test_small_values(skv, ctx, n):
    """Far below 1, where weights times values are near FP32's smallest numbers: 4096 tokens' 2^-127 each are 2^-115 together,
    2^-20 of these, of which the bound allows a weighted value more."""
    rig = P.Rig(skv, ctx, "bf16", 8, 2, 64, capacity=4096, seed=n)
    rig.map_all()
    rig.append([0], 4096, v=rig.rng.uniform(0.5, 1.0, (1, 4096, 2, 64)) * 2.0 ** -95)
    rig.check_attention([4096 - n], n, append=False)


def seen_no_numbers(skv, ctx, rig, p, n, heads, parents=None):
    """Values that are no numbers among the cached tokens, where they are far from the sequence's end and near it: they make
    their channels what a sum of weights above zero times values is, whatever the weights and splits; all else stays."""
    dim, kv = rig.dim, rig.kv
    at = [2, 700, p - 1]
    q = rig.random(1, n, heads, dim)[1]
    q[..., 0] = 4.0
    k, v = (rig.random(1, p, kv, dim)[1] for _ in "kv")
    try:
        for lift in (0.0, -70.0, 20.0):                      # scores of these tokens: with the others, far below, above
            kk = k.copy()
            kk[..., 0] = 0.0
            kk[0, at, :, 0] = lift
            for split in (0, 256, 4096):
                ctx.set_split_tokens(split)
                rig.append([0], p, k=kk, v=v)
                first, good = rig.attend([p], n, parents, q=q, append=False, scale=0.5) if parents is None else \
                    rig.attend([p], n, parents, q=q, k=np.zeros((1, n, kv, dim)), v=np.ones((1, n, kv, dim)), scale=0.5)
                assert np.isfinite(good).all()
                bad = v.copy()
                bad[0, at[0], :, 1], bad[0, at[1], :, 5], bad[0, at[2], :, 40] = np.inf, -np.inf, np.nan
                bad[0, at[0], :, 9], bad[0, at[1], :, 9] = np.inf, -np.inf
                bad[0, at[1:], :, 63] = np.inf
                rig.append([0], p, k=kk, v=bad)
                _, out = rig.attend([p], n, parents, q=q, append=False, scale=0.5) if parents is None else \
                    rig.attend([p], n, parents, q=q, k=np.zeros((1, n, kv, dim)), v=np.ones((1, n, kv, dim)), scale=0.5)
                for c, want in ((1, np.inf), (5, -np.inf), (40, np.nan), (9, np.nan), (63, np.inf)):
                    np.testing.assert_array_equal(out[..., c], np.full(out.shape[:-1], want), err_msg=f"channel {c}, lift {lift}, split {split}")
                rest = [c for c in range(dim) if c not in (1, 5, 9, 40, 63)]
                np.testing.assert_array_equal(out[..., rest], good[..., rest], err_msg=f"lift {lift}, split {split}")
    finally:
        ctx.set_split_tokens(0)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("n", [1, 7])
@pytest.mark.parametrize("dim", [64, 128])
def test_seen_no_numbers(skv, ctx, t, n, dim):
    rig = P.Rig(skv, ctx, t, 2, 1, dim, capacity=1600, seed=n)
    rig.map_all()
    rig.append([0], 1600)
    seen_no_numbers(skv, ctx, rig, 1500, n, 2, [P.chain(n)])
    seen_no_numbers(skv, ctx, rig, 1500, n, 2)


@every_shape
@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_seen_no_numbers_in_every_shape(skv, ctx, t, dim, forced):
    rig = P.Rig(skv, ctx, t, 4, 1, dim, capacity=1600, seed=forced)
    rig.map_all()
    rig.append([0], 1600)
    seen_no_numbers(skv, ctx, rig, 1500, 20, 4, [P.random_tree(np.random.default_rng(1), 20)])


def test_keys_of_kept_paths(skv, ctx):
    """A path of children from the root on leaves keys that are turned by the positions that they then have; one that
    leaves a generation out leaves them as the call turned them."""
    dim, p, n = 64, 90, 12
    rig = P.Rig(skv, ctx, "bf16", 2, 2, dim, batch=2, capacity=192, rotation=P.Rotation(dim), seed=3)
    rig.map_all()
    rig.append([0, 0], p)
    tree = [-1, 0, 0, 2, 2, 4, 1, 5, 5, 7, 8, -1]            # 0 - 2 - 4 - 5 - 8 - 10 is a path
    k = rig.random(2, n, 2, dim)[1]
    rig.append([p, p], n, [tree, tree], k=k)
    paths = [[0, 2, 4, 5, 8, 10], [0, 4, 5, 8, 10, -1]]
    assert rig.keep([p, p], paths) == [p + 6, p + 5]
    rig.check_values()
    for b, off in ((0, [0] * 6), (1, [0, 1, 1, 1, 1])):
        path = [a for a in paths[b] if a >= 0]
        want = rig.rotation.turn(k[b, path], p + np.arange(len(path)) + off, "bf16")
        np.testing.assert_array_equal(rig.rows(0, b, p + np.arange(len(path)))[0], want)


@pytest.mark.parametrize("cached", [0, 62, 64, 100])
def test_a_serving_program(skv, ctx, cached):
    """Steps of a drafted tree over pages' ends: pages are given to a sequence as its tokens need them, entries that have one
    keep it, and no cached token is lost."""
    layers, n, dim = 2, 4, 64
    rig = P.Rig(skv, ctx, "bf16", 8, 2, dim, batch=2, pages=12, layers=layers, capacity=384, rotation=P.Rotation(dim), seed=cached)
    free, pages, seq = list(range(12)), [], 1

    def give(tokens):
        more = [free.pop() for _ in range(-(-tokens // 64) - len(pages))]
        rig.map(seq, more, first=len(pages))
        pages.extend(more)
        return len(more)

    rig.map(0, [free.pop(3)])                                # another sequence's
    rig.append([0], 64)
    give(cached)
    for layer in range(layers if cached else 0):
        rig.append([0], cached, layer=layer, seq0=seq)
    tree, given = [skv.TREE_ROOT, 0, 0, 1], 0
    for turn in range(60):
        given += give(cached + n)
        for layer in range(layers):
            rig.check_attention([cached], n, [tree], layer=layer, seq0=seq)
        path = [[0, 1, 3], [0, 2, -1], [0, -1, -1], [-1, -1, -1]][turn % 4]
        cached = rig.keep([cached], [path], seq0=seq)[0]
        rig.check_values()
    assert given >= 1 and 64 * len(pages) >= cached


def large_scores(skv, ctx, rig, t, n, heads, tokens):
    """Scores so large that FP32 holds them in steps of 2^-5 to 2^9: equal ones weigh the same, and where half of the tokens
    are above the others by far more than a step, they alone count.  A weight is a rounding of the type off, the output
    another, and sums one of FP32 a token."""
    dim, kv = rig.dim, rig.kv
    half = tokens // 2
    k = np.zeros((1, tokens, kv, dim))
    v = rig.random(1, tokens, kv, dim)[1] + 2.0
    v = R.typed(v, t)[1]
    q = np.zeros((1, n, heads, dim))
    q[..., 0] = 1.0
    for exponent in (18, 21, 22, 23, 24, 25, 26, 27, 28, 29, 30, 32):
        for sign in (1.0, -1.0):
            for high in (0, 1):
                k[0, :, :, 0] = 1.0
                k[0, high * half:high * half + half, :, 0] += 2.0 ** -7
                rig.append([0], tokens, k=k, v=v)
                _, out = rig.attend([tokens - n], n, q=q, append=False, scale=sign * 1.37 * 2.0 ** exponent)
                assert np.isfinite(out).all(), (exponent, sign, high)
                best = high if sign > 0 else 1 - high
                for i in range(n):
                    at = np.arange(tokens - n + i + 1)
                    at = at[at >= half] if best else at[at < half]
                    for h in range(heads):
                        x = v[0, at, h // (heads // kv)]
                        want = x.mean(0)
                        off = (2 * R.HALF_STEP[t] + tokens * 2.0 ** -24 + 2.0 ** -18) * np.abs(x).mean(0)
                        err = np.abs(out[0, i, h] - want)
                        assert (err <= off).all(), (exponent, sign, high, i, h, (err / off).max())


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("n", [1, 7])
def test_large_scores(skv, ctx, t, n):
    rig = P.Rig(skv, ctx, t, 2, 1, 64, capacity=1024, seed=n)
    rig.map_all()
    try:
        for split in (0, 256, 4096):
            ctx.set_split_tokens(split)
            large_scores(skv, ctx, rig, t, n, 2, 1000)
    finally:
        ctx.set_split_tokens(0)


@every_shape
@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_large_scores_in_every_shape(skv, ctx, t, forced):
    rig = P.Rig(skv, ctx, t, 4, 1, 128, capacity=1024, seed=forced)
    rig.map_all()
    large_scores(skv, ctx, rig, t, 20, 4, 1000)


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("n", [1, 20])
def test_the_largest_and_smallest_scales(skv, ctx, t, n):
    """2^-100 weighs all tokens alike, 2^100 leaves the token with the largest score, or with a negative scale the
    smallest."""
    tokens, dim = 700, 64
    rig = P.Rig(skv, ctx, t, 4, 2, dim, capacity=tokens, seed=n)
    rig.map_all()
    k = rig.random(1, tokens, 2, dim)[1] * 0.25
    k[..., 0] = np.arange(tokens)[None, :, None] % 89        # several tokens share a score
    k[..., 1:] = 0.0
    v = rig.random(1, tokens, 2, dim)[1]
    rig.append([0], tokens, k=k, v=v)
    q = np.zeros((1, n, 4, dim))
    q[..., 0] = 1.0
    for scale in (2.0 ** -100, -2.0 ** -100, 2.0 ** 100, -2.0 ** 100):
        _, out = rig.attend([tokens - n], n, q=q, append=False, scale=scale)
        for i in range(n):
            at = np.arange(tokens - n + i + 1)
            if abs(scale) > 1:
                score = np.sign(scale) * (at % 89)
                at = at[score == score.max()]
            for h in range(4):
                x = v[0, at, h // 2]
                off = (2 * R.HALF_STEP[t] + tokens * 2.0 ** -24 + 2.0 ** -18) * np.abs(x).mean(0) + 2.0 ** -25
                assert (np.abs(out[0, i, h] - x.mean(0)) <= off).all(), (scale, i, h)
