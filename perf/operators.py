"""Rotary positions and the block cache: append, attention, eviction.

Four kinds of work around a decoder's attention, as a program that serves one layer (or evicts from all of
them) issues it:

  rotary  rotation of the query and key heads of fused projection rows by their positions (swiftkv_rotary);
  append  new K/V rows into the block cache, and the values that its codes stand for (swiftkv_block_append,
          swiftkv_block_values);
  step    n new tokens of each sequence appended, and their queries over the cache, with the attention weight
          of each block added up where the program evicts by it (swiftkv_block_attention);
  evict   all but `keep` blocks of each (layer, sequence, key/value head) dropped, the least attended first
          (swiftkv_block_evict).

A block is 16 tokens of one key/value head; its K codes and its V codes share one power-of-two scale each: the
smallest 2^e with max|x| <= 127 * 2^e.  A block that still has room when rows are appended keeps its scale unless
they need a larger one; then its codes are rounded to that one.

The sizes are the framework's own (32 heads of 128, batches of 1 to 64, contexts of 128 to 32512 tokens), with
the key/value heads shared by 1, 4, 5 or 8 query heads, and heads of 64.
"""
import importlib

import numpy as np
import torch

own = False

BLOCK = 16
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
THETA = 10000.0
MAX_POSITIONS = 32768

_kept = {}


def _package():
    return importlib.import_module("4pe_u250_amd")


def _context():
    """The one context (stream, workspace) that a program keeps for its GPU."""
    if "ctx" not in _kept:
        _kept["ctx"] = _package().Context(0)
    return _kept["ctx"]


# ---------------------------------------------------------------- cases


def _rotary(name=None, **c):
    c = {"kind": "rotary", "batch": 1, "n": 1, "position": 0, "heads": 40, "rest": 8, "head_dim": 128,
         "rotary_dim": 128, "halves": True, "scaling": "none", "inverse": False, "dtype": "bf16", **c}
    return dict(c, name=name) if name else c


def _append(name=None, **c):
    c = {"kind": "append", "batch": 1, "n": 1, "position": 0, "kv_heads": 8, "head_dim": 128, "ragged": False,
         "dtype": "bf16", "spread": 1.0, **c}
    return dict(c, name=name) if name else c


def _step(name=None, **c):
    c = {"kind": "step", "batch": 1, "n": 1, "position": 0, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "ragged": False, "weights": False, "dtype": "bf16", "spread": 1.0, **c}
    return dict(c, name=name) if name else c


def _evict(name=None, **c):
    c = {"kind": "evict", "layers": 1, "batch": 1, "kv_heads": 8, "position": 4095, "ragged": False, "keep": 128,
         "sinks": 1, "recent": 4, **c}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One token of one sequence, query and key heads of a fused projection row: latency.
        _rotary("rotary_step_b1", position=4095),
        # A full-length prompt far into a stretched context, half of each head rotated, adjacent pairs.
        _rotary("rotary_prompt_n4096", n=4096, position=28671, rotary_dim=64, halves=False, scaling="bands"),
        # The gradient of the rotation over a training batch of odd length, FP32.
        _rotary("rotary_back_n1777_f32", batch=3, n=1777, heads=36, rest=4, head_dim=64, rotary_dim=64,
                scaling="linear", inverse=True, dtype="f32"),
        # Rows of a serving batch added to caches of many lengths (tail blocks that are partly full).
        _append("append_b64_n1", batch=64, position=4095, ragged=True),
        # A prompt of odd length, all heads their own, FP32 rows with heavy channels.
        _append("append_prompt_n4095_f32", n=4095, kv_heads=32, dtype="f32", spread=20.0),
        # The first tokens of a conversation, a key/value head for each query head: the smallest step.
        _step("step_b1_p127", position=127, kv_heads=32),
        # One user at 4096 tokens, weights kept for eviction.
        _step("step_b1_p4095_weights", position=4095, weights=True),
        # The throughput workload: 64 users at 4096 tokens, weights kept.
        _step("step_b64_p4095_weights", batch=64, position=4095, weights=True),
        # Long contexts of different lengths, heavy K channels.
        _step("step_b16_p32511_f16", batch=16, position=32511, ragged=True, dtype="f16", spread=20.0),
        # A chunk of a prompt against what is cached of it.
        _step("chunk_n512_p4095", n=512, position=4095),
        # One layer of one sequence at 4096 tokens, half of it dropped.
        _evict("evict_b1_p4095"),
        # Every layer of a serving batch of long contexts, an eighth kept.
        _evict("evict_l32_b8_p32511", layers=32, batch=8, position=32511, ragged=True, keep=254, recent=16),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(lo * (hi / lo) ** rng.random() + rng.random()))


def draw(rng):
    kind = rng.choice(["rotary", "append", "step", "step", "step", "evict"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    head_dim = rng.choice([64, 128, 128])
    spread = rng.choice([1.0, 1.0, 20.0])
    batch = _log_int(rng, 1, 64)
    if kind == "rotary":
        n = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(2, 4096 // batch))
        heads, rest = rng.choice([(64, 32), (40, 16), (36, 4), (8, 0)])
        return _rotary(batch=batch, n=n, position=rng.randrange(0, MAX_POSITIONS - n), heads=heads, rest=rest,
                       head_dim=head_dim, rotary_dim=rng.choice([head_dim, head_dim, head_dim // 2, 48]),
                       halves=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "theta", "bands"]),
                       inverse=rng.random() < 0.3, dtype=dtype)
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (32, 4), (20, 4)])
    if kind == "evict":
        position = _log_int(rng, 300, 32511)
        blocks = (position + BLOCK - 1) // BLOCK
        return _evict(layers=rng.choice([1, 4, 32]), batch=min(batch, 8), kv_heads=kv_heads if kv_heads < 32 else 8,
                      position=position, ragged=rng.random() < 0.5, keep=rng.randint(8, max(8, blocks - 1)),
                      sinks=rng.randint(0, 3), recent=rng.randint(1, 5))
    if kind == "append":
        n = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(2, min(4095, 4095 * 32 // (batch * kv_heads))))
        return _append(batch=batch, n=n, position=rng.randrange(0, 4096), kv_heads=kv_heads, head_dim=head_dim,
                       ragged=rng.random() < 0.5, dtype=dtype, spread=spread)
    # Cached tokens times heads: at most those of the largest listed step.
    position = _log_int(rng, 127, min(32511, 16 * 32511 * 8 // (batch * kv_heads)))
    n = 1
    if rng.random() < 0.3:
        n = _log_int(rng, 2, 8)
    elif batch <= 2 and position <= 4095 and rng.random() < 0.4:
        n = _log_int(rng, 16, 512 // batch)
    return _step(batch=batch, n=n, position=position, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                 ragged=batch > 1 and rng.random() < 0.5, weights=n <= 8 and rng.random() < 0.5, dtype=dtype,
                 spread=spread)


def _positions(case):
    """Cached tokens of each sequence before the call: one position, or lengths from a sixteenth of it up."""
    top, batch = case["position"], case["batch"]
    if not case.get("ragged") or batch == 1:
        return torch.full((batch,), top, dtype=torch.int64)
    gen = torch.Generator().manual_seed(batch * 65537 + top)
    at = torch.randint(top // 16, top + 1, (batch,), generator=gen)
    at[0] = top
    return at


def _blocks(case):
    """Blocks of a cache that holds the case: its tokens, in whole groups of 64."""
    return (case["position"] + case.get("n", 1) + 63) // 64 * 4


# ---------------------------------------------------------------- inputs


def _generator(seed, what):
    return torch.Generator("cuda").manual_seed((seed * 1000003 + what) % (1 << 62))


def _rows(seed, what, shape, case):
    """Projection rows: normal, with one channel in 32 `spread` times as large where the case has heavy channels."""
    gen = _generator(seed, what)
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    if case["spread"] != 1.0:
        x *= 1.0 + (case["spread"] - 1.0) * (torch.rand(shape[-2:], generator=gen, device="cuda") < 1 / 32)
    return x.to(DTYPES[case["dtype"]])


def _block_weights(case, seed):
    """Attention weight gathered by each block: heavy-tailed, some blocks with the same, some with none."""
    gen = _generator(seed, 5)
    shape = (case["layers"], case["batch"], case["kv_heads"], _blocks(case))
    w = torch.randn(shape, generator=gen, device="cuda").mul_(2.0).exp_()
    w = torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.1, w.round(), w)
    held = ((_positions(case) + BLOCK - 1) // BLOCK).cuda()
    return w * (torch.arange(shape[-1], device="cuda") < held[:, None, None])


def _frequencies(case):
    """The rotary frequencies in 64 bits, with the case's scaling for long contexts, and what multiplies cos and sin."""
    half = case["rotary_dim"] // 2
    j = torch.arange(half, dtype=torch.float64)
    f = THETA ** (-j / half)
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "theta":
        return (THETA * 4.0 ** (half / (half - 1.0))) ** (-j / half), 1.0
    if case["scaling"] == "bands":
        turns = 4096.0 * f / (2.0 * torch.pi)       # full turns within the original 4096 positions
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return (1.0 - keep) * f / 8.0 + keep * f, 1.125
    return f, 1.0


def _table(case):
    """cos and sin of every position [MAX_POSITIONS][rotary_dim / 2], FP32, kept as a program keeps them; where
    `own` is true, the framework's table."""
    key = (own, case["rotary_dim"], case["scaling"])
    if key not in _kept:
        if own:
            skv = _package()
            scaling = {"none": None, "linear": skv.RopeScaling(skv.ROPE_LINEAR, 4.0),
                       "theta": skv.RopeScaling(skv.ROPE_THETA, 4.0),
                       "bands": skv.RopeScaling(skv.ROPE_BANDS, 8.0, 4096, 1.0, 4.0, 1.125)}[case["scaling"]]
            _kept[key] = skv.RotaryTable(_context(), case["rotary_dim"], MAX_POSITIONS, THETA, scaling)
        else:
            f, magnitude = _frequencies(case)
            angle = torch.arange(MAX_POSITIONS, dtype=torch.float64, device="cuda")[:, None] * f.cuda()
            _kept[key] = ((magnitude * angle.cos()).float(), (magnitude * angle.sin()).float())
    return _kept[key]


def prepare(case, seed):
    st = {"case": case}
    if case["kind"] == "rotary":
        heads, rest, dim = case["heads"], case["rest"], case["head_dim"]
        st["table"] = _table(case)
        st["x"] = _rows(seed, 1, (case["batch"], case["n"], heads + rest, dim), {**case, "spread": 1.0})
        st["out"] = torch.empty((case["batch"], case["n"], heads, dim), dtype=st["x"].dtype, device="cuda")
        st["positions"] = [case["position"] // (b + 1) for b in range(case["batch"])]
        if own:
            st["args"] = (st["x"].data_ptr(), st["out"].data_ptr())
        torch.cuda.synchronize()
        return st
    positions = _positions(case)
    st["positions"] = positions.tolist() if case["batch"] > 1 else int(positions[0])
    st["at"] = positions.cuda()
    if case["kind"] == "evict":
        st["weights"] = _block_weights(case, seed)
        st["kept"] = torch.empty(st["weights"].shape[:3] + (case["keep"],), dtype=torch.int32, device="cuda")
        if own:
            st["cache"] = _package().BlockCache(_context(), case["layers"], case["batch"], case["kv_heads"],
                                                case["kv_heads"], 64, case["position"] + 1)
        torch.cuda.synchronize()
        return st
    batch, n, top, kv, dim = case["batch"], case["n"], case["position"], case["kv_heads"], case["head_dim"]
    dtype = DTYPES[case["dtype"]]
    st["k"], st["v"] = (_rows(seed, i, (batch, n, kv, dim), case) for i in (2, 3))
    history = [_rows(seed, i, (batch, max(top, 1), kv, dim), case) for i in (6, 7)]
    if own:
        skv, ctx = _package(), _context()
        st["cache"] = skv.BlockCache(ctx, 1, batch, case.get("heads", kv), kv, dim, _blocks(case) * BLOCK)
        torch.cuda.synchronize()
        for b in range(batch):
            if int(positions[b]):
                skv.swiftkv_block_append(ctx, history[0][b].data_ptr(), history[1][b].data_ptr(), st["cache"], 0, 0,
                                         n=int(positions[b]), dtype=getattr(skv, case["dtype"].upper()), seq0=b)
        ctx.synchronize()
    else:
        st["codes"], st["scales"] = zip(*(_first_codes(x, positions, _blocks(case) + 1) for x in history))
    del history
    if case["kind"] == "append":
        st["outs"] = [torch.empty((batch, n, kv, dim), dtype=dtype, device="cuda") for _ in range(2)]
    else:
        st["q"] = _rows(seed, 4, (batch, n, case["heads"], dim), {**case, "spread": 1.0})
        st["out"] = torch.empty_like(st["q"])
        if case["weights"]:
            st["weights"] = torch.zeros((batch, kv, _blocks(case)), device="cuda")
    torch.cuda.synchronize()
    return st


# ---------------------------------------------------------------- the framework's calls


def _run_own(st):
    skv, ctx, case = _package(), _context(), st["case"]
    if case["kind"] == "rotary":
        x, out = st["args"]
        skv.swiftkv_rotary(ctx, st["table"], x, out, st["positions"], case["heads"], case["head_dim"], n=case["n"],
                           dtype=getattr(skv, case["dtype"].upper()), halves=case["halves"],
                           inverse=case["inverse"], x_stride=(case["heads"] + case["rest"]) * case["head_dim"])
        return {"out": st["out"]}
    if case["kind"] == "evict":
        skv.swiftkv_block_evict(ctx, st["cache"], 0, case["layers"], st["positions"], case["keep"],
                                st["weights"].data_ptr(), st["kept"].data_ptr(), sinks=case["sinks"],
                                recent=case["recent"])
        return {"kept": st["kept"], "weights": st["weights"]}
    dtype = getattr(skv, case["dtype"].upper())
    if case["kind"] == "append":
        k, v = st["outs"]
        skv.swiftkv_block_append(ctx, st["k"].data_ptr(), st["v"].data_ptr(), st["cache"], 0, st["positions"],
                                 n=case["n"], dtype=dtype)
        skv.swiftkv_block_values(ctx, st["cache"], 0, st["positions"], k.data_ptr(), v.data_ptr(), n=case["n"],
                                 dtype=dtype)
        return {"k": k, "v": v}
    weights = st["weights"].data_ptr() if case["weights"] else None
    skv.swiftkv_block_attention(ctx, st["q"].data_ptr(), st["k"].data_ptr(), st["v"].data_ptr(), st["cache"], 0,
                                st["positions"], st["out"].data_ptr(), n=case["n"], dtype=dtype, weights=weights)
    return {"out": st["out"], "weights": st["weights"]} if case["weights"] else {"out": st["out"]}


# ---------------------------------------------------------------- the plain forms


def _exponent(amax):
    """The smallest e with amax <= 127 * 2^e (-100 at least)."""
    m, e = torch.frexp(amax)
    return (e - 7 + (m > 127 / 128).int()).clamp_(min=-100)


def _first_codes(x, positions, blocks):
    """INT8 codes [batch][heads][blocks][16][dim] and scales [batch][heads][blocks] of rows x [batch][t][heads][dim]
    appended to an empty cache; the first positions[b] rows of sequence b count."""
    batch, t, heads, dim = x.shape
    held = torch.arange(t, device="cuda") < positions.cuda()[:, None]
    rows = torch.zeros((batch, heads, blocks * BLOCK, dim), device="cuda")
    rows[:, :, :t] = torch.where(held[:, :, None, None], x.float(), 0.0).transpose(1, 2)
    rows = rows.view(batch, heads, blocks, BLOCK, dim)
    scales = torch.ldexp(torch.ones((), device="cuda"), _exponent(rows.abs().amax((3, 4))))
    return (rows / scales[..., None, None]).round_().to(torch.int8), scales


def _plain_append(codes, scales, x, at):
    """Rows x [batch][n][heads][dim] into tokens at[b] .. at[b] + n - 1 of the codes, in place."""
    batch, n, heads, dim = x.shape
    touched = (n + 2 * BLOCK - 2) // BLOCK
    first = at // BLOCK
    seq = torch.arange(batch, device="cuda")[:, None]
    local = at[:, None] % BLOCK + torch.arange(n, device="cuda")             # [batch][n], from the first touched block
    rows = torch.zeros((batch, touched * BLOCK, heads, dim), device="cuda")
    rows[seq, local] = x.float()
    new = torch.zeros((batch, touched * BLOCK), dtype=torch.bool, device="cuda")
    new[seq, local] = True
    rows = rows.view(batch, touched, BLOCK, heads, dim)
    new = new.view(batch, touched, BLOCK, 1, 1)
    blocks = first[:, None] + torch.arange(touched, device="cuda")
    held = (torch.arange(touched, device="cuda") == 0) & (at % BLOCK > 0)[:, None]      # the block keeps rows
    old = scales.transpose(1, 2)[seq, blocks]                                # [batch][touched][heads]
    e = torch.ldexp(torch.ones((), device="cuda"), _exponent(rows.abs().amax((2, 4))))
    e = torch.where(held[:, :, None], torch.maximum(e, old), torch.where(new.any(2)[..., 0], e, old))
    kept = codes.permute(0, 2, 3, 1, 4)[seq, blocks].float()                 # [batch][touched][16][heads][dim]
    kept = (kept * (old / e)[:, :, None, :, None]).round_()
    fresh = (rows / e[:, :, None, :, None]).round_()
    codes.permute(0, 2, 3, 1, 4)[seq, blocks] = torch.where(new, fresh, kept.clamp_(-127, 127)).to(torch.int8)
    scales.transpose(1, 2)[seq, blocks] = e


def _plain_values(codes, scales, at, n):
    """The values of tokens at[b] .. at[b] + n - 1: [batch][n][heads][dim], FP32."""
    batch = codes.shape[0]
    tok = at[:, None] + torch.arange(n, device="cuda")
    seq = torch.arange(batch, device="cuda")[:, None]
    c = codes.permute(0, 2, 3, 1, 4)[seq, tok // BLOCK, tok % BLOCK].float()
    return c * scales.transpose(1, 2)[seq, tok // BLOCK][..., None]


def _plain_attention(q, codes, scales, at):
    """Attention of q [batch][n][heads][dim] over tokens 0 .. at[b] + i for query i: out and weights per block."""
    batch, n, heads, dim = q.shape
    kv, blocks = codes[0].shape[1], codes[0].shape[2] - 1       # the last block is spare
    kd, vd = ((c[:, :, :-1] * s[:, :, :-1, None, None]).view(batch, kv, blocks * BLOCK, dim)
              for c, s in zip(codes, scales))
    group = heads // kv
    rows = q.float().view(batch, n, kv, group, dim).permute(0, 2, 4, 1, 3).reshape(batch, kv, dim, n * group)
    scores = torch.matmul(kd, rows.contiguous()) * dim ** -0.5              # [batch][kv][tokens][n * group]
    last = at[:, None] + torch.arange(n, device="cuda")                      # last visible token of each query
    seen = torch.arange(blocks * BLOCK, device="cuda")[None, :, None] <= last[:, None].repeat_interleave(group, 2)
    scores = scores.masked_fill_(~seen[:, None], -torch.inf)
    p = (scores - scores.amax(2, keepdim=True)).exp_()
    p /= p.sum(2, keepdim=True)
    out = torch.matmul(p.transpose(2, 3).contiguous(), vd).view(batch, kv, n, group, dim)
    return out.transpose(1, 2).reshape(q.shape), p.view(batch, kv, blocks, BLOCK, -1).sum((3, 4))


def _plain_evict(weights, at, keep, sinks, recent):
    """Old indices of the blocks that stay [..][keep] (-1 past their number); the weights move along, in place."""
    n = weights.shape[-1]
    held = ((at + BLOCK - 1) // BLOCK)[:, None, None]                               # blocks of each sequence
    i = torch.arange(n, device="cuda")
    rank = torch.where(weights > 0, weights, 0.0)       # NaN counts as none
    rank = torch.where((i < sinks) | (i >= held - recent) | (held <= keep), torch.inf, rank)
    rank = torch.where(i < held, rank, -torch.inf)
    stays = torch.argsort(rank, dim=-1, descending=True, stable=True)[..., :keep].sort(-1).values
    stays = torch.where(torch.arange(keep, device="cuda") < held, stays, -1)
    moved = torch.where(stays >= 0, weights.gather(-1, stays.clamp(min=0)), 0.0)
    weights.zero_()[..., :keep] = moved
    return stays.to(torch.int32)


def run(st):
    if own:
        return _run_own(st)
    case = st["case"]
    if case["kind"] == "rotary":
        heads, half = case["heads"], case["rotary_dim"] // 2
        at = torch.tensor(st["positions"], device="cuda")[:, None] + torch.arange(case["n"], device="cuda")
        c, s = (t[at][:, :, None] for t in st["table"])
        x = st["x"][:, :, :heads].float()
        turned = x[..., :2 * half]
        a, b = (turned[..., :half], turned[..., half:]) if case["halves"] else (turned[..., 0::2], turned[..., 1::2])
        if case["inverse"]:
            s = -s
        pair = (a * c - b * s, a * s + b * c)
        turned = torch.cat(pair, -1) if case["halves"] else torch.stack(pair, -1).flatten(-2)
        st["out"].copy_(torch.cat([turned, x[..., 2 * half:]], -1))
        return {"out": st["out"]}
    if case["kind"] == "evict":
        st["kept"].copy_(_plain_evict(st["weights"], st["at"], case["keep"], case["sinks"], case["recent"]))
        return {"kept": st["kept"], "weights": st["weights"]}
    codes, scales, at = st["codes"], st["scales"], st["at"]
    _plain_append(codes[0], scales[0], st["k"], at)
    _plain_append(codes[1], scales[1], st["v"], at)
    if case["kind"] == "append":
        k, v = st["outs"]
        k.copy_(_plain_values(codes[0], scales[0], at, case["n"]))
        v.copy_(_plain_values(codes[1], scales[1], at, case["n"]))
        return {"k": k, "v": v}
    out, weights = _plain_attention(st["q"], codes, scales, at)
    st["out"].copy_(out)
    if not case["weights"]:
        return {"out": st["out"]}
    st["weights"] += weights
    return {"out": st["out"], "weights": st["weights"]}


def work(case):
    kind, batch = case["kind"], case["batch"]
    positions = [int(p) for p in _positions(case)]
    if kind == "evict":
        held = [(p + BLOCK - 1) // BLOCK for p in positions]
        blocks, kept = sum(held), sum(min(h, case["keep"]) for h in held)
        return {"bytes": case["layers"] * case["kv_heads"] * (4 * blocks + 8 * kept), "flops": 0}
    n, dim, size = case["n"], case["head_dim"], DTYPES[case["dtype"]].itemsize
    if kind == "rotary":
        channels = batch * n * case["heads"] * dim
        return {"bytes": 2 * size * channels + batch * n * case["rotary_dim"] * 4,
                "flops": 3 * batch * n * case["heads"] * case["rotary_dim"]}
    kv = case["kv_heads"]
    rows = batch * n * kv * dim
    if kind == "append":
        return {"bytes": 2 * rows * (size + 1 + size), "flops": 4 * rows}
    seen = sum(n * p + n * (n + 1) // 2 for p in positions)
    moved = sum(positions) * kv * (2 * dim + 8 / BLOCK) + 2 * rows * (size + 1)
    moved += 2 * batch * n * case["heads"] * dim * size
    if case["weights"]:
        moved += 8 * kv * sum((p + n + BLOCK - 1) // BLOCK for p in positions)
    return {"bytes": moved, "flops": 4 * dim * case["heads"] * seen}


# ---------------------------------------------------------------- the definition, in 64 bits


def _exact_scale(amax):
    e = torch.floor(torch.log2(amax.clamp(min=2.0 ** -93))) - 8.0
    for _ in range(3):          # floor(log2) - 8 is at most three below
        e = e + (amax > 127.0 * torch.exp2(e)).double()
    return torch.exp2(e.clamp(min=-100.0))


def _exact_values(old, new):
    """Values [t][dim...] of one sequence's rows: `old` [t0][heads][dim] appended to an empty cache, then `new`."""
    t0, n = old.shape[0], new.shape[0]
    pad = (t0 + n + BLOCK - 1) // BLOCK * BLOCK
    def blocked(x):
        return x.view(-1, BLOCK, *x.shape[1:])
    x0 = torch.zeros((pad,) + new.shape[1:], dtype=torch.float64, device="cuda")
    x1 = x0.clone()
    x0[:t0], x1[t0:t0 + n] = old.double(), new.double()
    x0, x1 = blocked(x0), blocked(x1)
    s0, s1 = (_exact_scale(x.abs().amax((1, 3), keepdim=True)) for x in (x0, x1))
    first = torch.round(x0 / s0)
    i = torch.arange(x0.shape[0], device="cuda")[:, None, None, None]
    has0, has1 = i * BLOCK < t0, (i + 1) * BLOCK > t0
    s = torch.where(has0 & has1, torch.maximum(s0, s1), torch.where(has1, s1, s0))
    return ((torch.round(first * s0 / s) + torch.round(x1 / s)) * s).view(pad, *new.shape[1:])[:t0 + n]


def exact(case, seed):
    if case["kind"] == "rotary":
        st = prepare(case, seed)
        f, magnitude = _frequencies(case)
        half = case["rotary_dim"] // 2
        x = st["x"][:, :, :case["heads"]].double()
        at = torch.tensor(st["positions"], dtype=torch.float64)[:, None] + torch.arange(case["n"])
        angle = at[..., None] * f
        turn = torch.polar(torch.full_like(angle, magnitude), angle).cuda()[:, :, None]
        turn = turn.conj() if case["inverse"] else turn
        part = x[..., :2 * half].unflatten(-1, (2, half)).transpose(-1, -2) if case["halves"] else \
            x[..., :2 * half].unflatten(-1, (half, 2))
        z = torch.view_as_real(torch.view_as_complex(part.contiguous()) * turn)
        z = (z.transpose(-1, -2) if case["halves"] else z).flatten(-2)
        return {"out": torch.cat([z, x[..., 2 * half:]], -1)}
    positions = _positions(case).tolist()
    if case["kind"] == "evict":
        w = _block_weights(case, seed).cpu().numpy()
        kept, left = np.full(w.shape[:3] + (case["keep"],), -1, np.int32), np.zeros(w.shape)
        for b, p in enumerate(positions):
            nb, keep = (p + BLOCK - 1) // BLOCK, min(case["keep"], (p + BLOCK - 1) // BLOCK)
            lo, hi = (case["sinks"], nb - case["recent"]) if nb > keep else (nb, nb)
            mid = np.argsort(-w[:, b, :, lo:hi], axis=-1, kind="stable")[..., :keep - lo - (nb - hi)] + lo
            ends = np.broadcast_to(np.r_[:lo, hi:nb], mid.shape[:2] + (lo + nb - hi,))
            kept[:, b, :, :keep] = np.sort(np.concatenate([mid, ends], -1), -1)
            left[:, b, :, :keep] = np.take_along_axis(w[:, b], kept[:, b, :, :keep].astype(np.int64), -1)
        return {"kept": kept, "weights": left}
    batch, n, top, kv, dim = case["batch"], case["n"], case["position"], case["kv_heads"], case["head_dim"]
    k, v = (_rows(seed, i, (batch, n, kv, dim), case) for i in (2, 3))
    kh, vh = (_rows(seed, i, (batch, max(top, 1), kv, dim), case) for i in (6, 7))
    if case["kind"] == "append":
        return {name: torch.stack([_exact_values(old[b, :p], new[b])[p:] for b, p in enumerate(positions)])
                for name, old, new in (("k", kh, k), ("v", vh, v))}
    q = _rows(seed, 4, (batch, n, case["heads"], dim), {**case, "spread": 1.0})
    group = case["heads"] // kv
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    weights = torch.zeros((batch, kv, _blocks(case)), dtype=torch.float64, device="cuda")
    for b, p in enumerate(positions):
        kd, vd = _exact_values(kh[b, :p], k[b]), _exact_values(vh[b, :p], v[b])
        hidden = torch.arange(p + n, device="cuda") > p + torch.arange(n, device="cuda")[:, None]
        for h in range(kv):
            rows = q[b, :, h * group:(h + 1) * group].double().transpose(0, 1).reshape(group * n, dim)
            s = torch.matmul(rows, kd[:, h].t().contiguous()) / dim ** 0.5
            w = torch.softmax(s.masked_fill_(hidden.repeat(group, 1), -torch.inf), 1)
            out[b, :, h * group:(h + 1) * group] = torch.matmul(w, vd[:, h].contiguous()).view(group, n, dim).transpose(0, 1)
            each = torch.zeros(_blocks(case) * BLOCK, dtype=torch.float64, device="cuda")
            each[:p + n] = w.sum(0)
            weights[b, h] = each.view(-1, BLOCK).sum(1)
    return {"out": out, "weights": weights} if case["weights"] else {"out": out}
