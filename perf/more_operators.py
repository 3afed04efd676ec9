"""The framework's paged-cache operators as timed cases: what a serving step does with a KV cache whose positions live in
pages that a table names.

A cache is two pools k, v [pages, kv, page, dim] in 16 bits and a table [slots, width]: position p of slot s lies in page
table[s, p // page] at p % page. A page outside the pool (-1: released) holds nothing that a row sees.

  append  a step's q|k|v rows: per-head RMS norm of queries and keys (or none), rotation of the first `rot` dims of each
          head by position (rotate-half or interleaved pairs; plain, linearly interpolated or by-parts scaled
          frequencies), queries out, keys and values into their pages
  read    positions of the cache as rows: a prefix's export
  attn    attention of each row's query heads over its slot's positions j <= pos, with a window those with
          j > pos - window or j < sinks: single tokens, a few drafted tokens and whole prompts (consecutive rows of one
          slot); rows with pos = -1 give zeros
"""
import functools
import math
import os
import random
import sys
from types import SimpleNamespace

import torch

own = False
DEV = "cuda" if torch.cuda.is_available() else "cpu"
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # a lone stream's token through a backbone layer: the smallest call
        dict(name="append_1", op="append", seqs=1, tokens=1, start=700, heads=16, kv=8, dim=128, rot=128, pairs="half",
             norm=True, scaling="none", page=64, dtype="bf16"),
        # a full GPU's decode step
        dict(name="append_224", op="append", seqs=224, tokens=1, start=2000, heads=16, kv=8, dim=128, rot=128,
             pairs="half", norm=True, scaling="none", page=64, dtype="bf16"),
        # pieces of four long prompts far into their contexts, half of each head rotated in interleaved pairs
        dict(name="append_4x512_far", op="append", seqs=4, tokens=512, start=100003, heads=32, kv=8, dim=128, rot=64,
             pairs="interleaved", norm=False, scaling="parts", page=16, dtype="fp16"),
        # a voice prefix exported
        dict(name="read_300", op="read", seqs=1, tokens=300, kv=8, dim=128, page=64, dtype="bf16"),
        # whole contexts exported, smaller heads, an odd length
        dict(name="read_16x4095", op="read", seqs=16, tokens=4095, kv=8, dim=64, page=32, dtype="fp16"),
        # a lone stream's token over its context: latency
        dict(name="attn_1", op="attn", seqs=1, tokens=1, empty=0, ctx=2048, spread=False, window=0, sinks=0, heads=16,
             kv=8, dim=128, page=64, dtype="bf16"),
        # a full GPU in steady state: bytes
        dict(name="attn_224", op="attn", seqs=224, tokens=1, empty=0, ctx=2048, spread=False, window=0, sinks=0,
             heads=16, kv=8, dim=128, page=64, dtype="bf16"),
        # drafted tokens of streams of all ages, padded to the next row bucket, small heads, small pages
        dict(name="attn_30x5_spread", op="attn", seqs=30, tokens=5, empty=10, ctx=3001, spread=True, window=0, sinks=0,
             heads=32, kv=4, dim=64, page=16, dtype="fp16"),
        # eight prompts of 200 tokens onto prefixes
        dict(name="attn_8x200", op="attn", seqs=8, tokens=200, empty=0, ctx=500, spread=False, window=0, sinks=0,
             heads=16, kv=8, dim=128, page=64, dtype="bf16"),
        # a long prompt's last piece: arithmetic
        dict(name="attn_4096_long", op="attn", seqs=1, tokens=4096, empty=0, ctx=16384, spread=False, window=0, sinks=0,
             heads=32, kv=8, dim=128, page=128, dtype="bf16"),
        # endless streams: a window and the first tokens, the pages between them released
        dict(name="window_48", op="attn", seqs=48, tokens=1, empty=0, ctx=30011, spread=False, window=1024, sinks=4,
             heads=16, kv=8, dim=128, page=64, dtype="bf16"),
        # pieces of prompts longer than the window
        dict(name="window_4x700", op="attn", seqs=4, tokens=700, empty=3, ctx=5000, spread=False, window=512, sinks=16,
             heads=32, kv=8, dim=64, page=32, dtype="fp16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "append", "read", "attn", "attn", "attn", "attn"))
    c = dict(op=op, kv=rng.choice((1, 2, 4, 8)), dim=rng.choice((64, 128, 128)), page=rng.choice((16, 32, 64, 128)),
             dtype=rng.choice(("bf16", "fp16")))
    ratio = rng.choice((1, 2, 2, 4, 5, 8))
    if op == "read":
        seqs = _log(rng, 1, 64)
        return dict(c, seqs=seqs, tokens=_log(rng, 1, 65536 // seqs))
    if op == "append":
        seqs = _log(rng, 1, 224)
        return dict(c, seqs=seqs, tokens=1 if rng.random() < 0.4 else _log(rng, 1, max(1, 4096 // seqs)),
                    start=_log(rng, 1, 200000) - 1, heads=c["kv"] * ratio,
                    rot=rng.choice((c["dim"], c["dim"], c["dim"] // 2, 16, 48)), pairs=rng.choice(("half", "interleaved")),
                    norm=rng.random() < 0.5, scaling=rng.choice(("none", "none", "linear", "parts")))
    c["heads"] = c["kv"] * ratio
    kind = rng.random()
    if kind < 0.5:  # single tokens
        seqs, tokens = _log(rng, 1, 224), 1
        ctx = _log(rng, 1, min(120000, 224 * 2048 // seqs))
    elif kind < 0.65:  # a few drafted tokens
        seqs, tokens = _log(rng, 1, 64), rng.randint(2, 8)
        ctx = tokens + _log(rng, 1, min(32000, 64 * 2048 // seqs))
    else:  # prompts
        seqs = _log(rng, 1, 16)
        tokens = _log(rng, 9, 4096 * 32 // max(32, c["heads"]) // seqs)
        ctx = tokens + _log(rng, 1, 12288) // seqs
    window = _log(rng, 16, 4096) if rng.random() < 0.4 else 0
    return dict(c, seqs=seqs, tokens=tokens, empty=rng.choice((0, 0, 1, 3)), ctx=ctx,
                spread=tokens < 9 and rng.random() < 0.5, window=window,
                sinks=rng.choice((0, 1, 4, 100)) if window else 0)


def _lengths(case):
    """Positions that each sequence holds after the step, the same for every seed (their order is the seed's)."""
    s, ctx, t = case["seqs"], case["ctx"], case["tokens"]
    if case["spread"]:
        return [max(t, ctx * (i + 1) // s) for i in range(s)]
    return [max(t, ctx - (7 * i) % 16) for i in range(s)]


def _seen(p, window, sinks):
    """Keys that a row at position p sees."""
    if not window or p < window:
        return p + 1
    return window + min(sinks, p + 1 - window)


def work(case):
    op = case["op"]
    rows, row = case["seqs"] * case["tokens"], case["kv"] * case["dim"] * 2
    if op == "append":
        return {"bytes": 2 * rows * (case["heads"] * case["dim"] * 2 + 2 * row), "flops": 0}
    if op == "read":
        return {"bytes": 2 * rows * 2 * row, "flops": 0}
    t, w, s = case["tokens"], case["window"], case["sinks"]
    keys = seen = 0
    for n in _lengths(case):
        first = max(0, n - t - w + 1) if w else 0
        keys += n - first + min(s, first)
        seen += sum(_seen(p, w, s) for p in range(n - t, n))
    return {"bytes": keys * 2 * row + 2 * (rows + case["empty"]) * case["heads"] * case["dim"] * 2,
            "flops": 4 * case["heads"] * case["dim"] * seen}


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919)


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _inv_freq(case):
    """(radians a position of each pair, factor of the rotated values), 64-bit."""
    rot, theta, factor, trained = case["rot"], 1e6, 8.0, 32768
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "parts":  # fast pairs as they are, slow ones interpolated, by their turns over the trained length
        keep = ((trained * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
        return f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1
    return f, 1.0


def _pools(case, pages, g):
    """Filled pools: keys with a few strong channels as trained ones have."""
    shape, dt = (pages, case["kv"], case["page"], case["dim"]), DT[case["dtype"]]
    k, v = _normal(g, *shape, dtype=dt), _normal(g, *shape, dtype=dt)
    k *= torch.exp(0.7 * _normal(g, case["kv"], 1, case["dim"])).to(dt)
    v *= 0.5
    return k, v


def _table(case, slots, held, g):
    """Pages for the positions in held (per slot a list of (first, end)), in no order; -1 where a slot holds nothing.
    Returns (table, pages)."""
    page = case["page"]
    width = max(-(-end // page) for spans in held.values() for _, end in spans)
    table = torch.full((slots, width), -1, dtype=torch.int32)
    n = 0
    for s, spans in held.items():
        for first, end in spans:
            a, b = first // page, -(-end // page)
            table[s, a:b] = torch.arange(n, n + b - a, dtype=torch.int32)
            n += b - a
    pages = n + 3
    order = torch.randperm(pages, generator=g, device=DEV).int()
    table = table.to(DEV)
    return torch.where(table >= 0, order[table.clamp_min(0).long()], table), pages


def prepare(case, seed):
    op, g, dt = case["op"], _gen(seed), DT[case["dtype"]]
    s = SimpleNamespace(case=dict(case), kept={})
    rng = random.Random(int(seed) * 31 + 5)
    t, w, sinks = case["tokens"], case.get("window", 0), case.get("sinks", 0)
    at = rng.sample(range(case["seqs"] + 1), case["seqs"])
    if op == "attn":
        n = _lengths(case)
        rng.shuffle(n)
        held = {}
        for i, x in zip(at, n):
            first = max(0, x - t - w + 1) if w else 0
            # the released pages lie whole between the first tokens and the window
            held[i] = [(0, x)] if first <= sinks + case["page"] else [(first, x)] + ([(0, sinks)] if sinks else [])
    elif op == "read":
        n = [t] * case["seqs"]
        held = {i: [(0, x)] for i, x in zip(at, n)}
    else:
        n = [case["start"] + t + rng.randint(0, 5) for _ in at]
        held = {i: [(x - t, x)] for i, x in zip(at, n)}
    s.table, pages = _table(case, case["seqs"] + 1, held, g)
    s.k, s.v = _pools(case, pages, g)
    e = case.get("empty", 0)
    pos = (torch.tensor(n, device=DEV)[:, None] - t + torch.arange(t, device=DEV)).flatten()
    s.slots = torch.cat([torch.tensor(at, device=DEV).repeat_interleave(t), torch.zeros(e, dtype=torch.long, device=DEV)])
    s.pos = torch.cat([pos, torch.full((e,), -1, device=DEV)]).int()
    heads, kv, dim = case.get("heads"), case["kv"], case["dim"]
    if op == "append":
        x = _normal(g, pos.numel(), heads + 2 * kv, dim)
        x[:, heads:heads + kv] *= torch.exp(0.7 * _normal(g, kv, dim))
        s.qkv = x.to(dt).flatten(1)
        s.wq, s.wk = (torch.exp(0.3 * _normal(g, dim)).to(dt) if case["norm"] else None for _ in "qk")
        s.inv_freq, s.factor = _inv_freq(case)
    elif op == "attn":
        s.q = _normal(g, s.pos.numel(), heads, dim).to(dt)
        s.scale, s.ctx = dim ** -0.5, max(n)
        # the step's runs of rows, as its host lays them out: (first row, rows, first position)
        s.runs = [(i * t, t, x - t) for i, x in enumerate(n)] + [(pos.numel() + i, 1, -1) for i in range(e)]
    return s


# ---------------------------------------------------------------- plain forms
def _place(s, slots, pos):
    """(page, offset) of positions."""
    page = s.case["page"]
    return s.table[slots, pos // page].long(), pos % page


def _plain_append(s):
    c = s.case
    heads, kv, dim, rot = c["heads"], c["kv"], c["dim"], c["rot"]
    x = s.qkv.float().view(-1, heads + 2 * kv, dim)
    qk = x[:, :heads + kv]
    if c["norm"]:
        w = torch.cat([s.wq.float().expand(heads, dim), s.wk.float().expand(kv, dim)])
        qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS) * w
    angle = s.pos.double()[:, None, None] * s.inv_freq.to(DEV)
    cos, sin = (angle.cos() * s.factor).float(), (angle.sin() * s.factor).float()
    r, rest = qk[..., :rot], qk[..., rot:]
    if c["pairs"] == "half":
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    y = torch.cat([r, rest], -1).to(s.qkv.dtype)
    page, at = _place(s, s.slots, s.pos.long())
    s.k[page, :, at] = y[:, heads:]
    s.v[page, :, at] = s.qkv.view(-1, heads + 2 * kv, dim)[:, heads + kv:]
    return y[:, :heads].contiguous(), s.k, s.v


def _plain_read(s):
    page, at = _place(s, s.slots, s.pos.long())
    return s.k[page, :, at], s.v[page, :, at]


def _plain_attn(s):
    c = s.case
    seqs, t, kv, dim, w, sinks = c["seqs"], c["tokens"], c["kv"], c["dim"], c["window"], c["sinks"]
    n, g = seqs * t, c["heads"] // kv
    slots, last = s.slots[:n:t], s.pos[t - 1:n:t].long()
    span = min(s.ctx, sinks + w + t - 1) if w else s.ctx
    j = torch.arange(span, device=DEV)  # the positions that a sequence's rows can see: the first tokens, then the window
    near = (last[:, None] + 1 - (span - sinks)).clamp_min(sinks) + j - sinks
    key = torch.where(j < sinks, j, near)
    there = key <= last[:, None]
    page, at = _place(s, slots[:, None], key.where(there, last[:, None]))
    k, v = (x[page, :, at].float().transpose(1, 2) for x in (s.k, s.v))  # [seqs, kv, span, dim]
    q = s.q[:n].float().view(seqs, t, kv, g, dim).permute(0, 2, 1, 3, 4).reshape(seqs, kv, t * g, dim)
    score = torch.matmul(q * s.scale, k.transpose(-1, -2).contiguous()).view(seqs, kv, t, g, span)
    key, p = key[:, None, None, None, :], s.pos[:n].view(seqs, 1, t, 1, 1)
    hidden = key > p
    if w:
        hidden = hidden | ((key <= p - w) & (key >= sinks))
    score = score.masked_fill(hidden, float("-inf"))
    score = torch.exp(score - score.amax(-1, keepdim=True))
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score.view(seqs, kv, t * g, span), v.contiguous()).view(seqs, kv, t, g, dim) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(n, c["heads"], dim)
    return torch.cat([o, torch.zeros(c["empty"], c["heads"], dim, device=DEV)]).to(s.q.dtype)


# ---------------------------------------------------------------- the framework's calls
@functools.lru_cache(None)
def _ops():
    at = os.path.join(os.getcwd(), "maya2-native_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from m3x import ops
    return ops


def _own_cache(s):
    """The handle on the cache that a program keeps."""
    if "cache" not in s.kept:
        s.kept["cache"] = _ops().PagedKv(s.k, s.v, s.table)
    return s.kept["cache"]


def _own_append(s):
    ops, c = _ops(), s.case
    if "rotary" not in s.kept:  # a program keeps its rotation's frequencies
        s.kept["rotary"] = ops.Rotary(s.inv_freq, interleaved=c["pairs"] == "interleaved", factor=s.factor, device=DEV)
    q = torch.empty(s.pos.numel(), c["heads"], c["dim"], dtype=s.qkv.dtype, device=DEV)
    ops.qk_norm_rope_paged(s.qkv, q, _own_cache(s), s.slots, s.pos, s.kept["rotary"], s.wq, s.wk, EPS, c["heads"])
    return q, s.k, s.v


def _own_read(s):
    shape = (s.pos.numel(), s.case["kv"], s.case["dim"])
    k, v = (torch.empty(shape, dtype=s.k.dtype, device=DEV) for _ in "kv")
    _ops().paged_read(_own_cache(s), s.slots, s.pos, k, v)
    return k, v


def _own_attn(s):
    ops, c = _ops(), s.case
    if "plan" not in s.kept:  # of a step's row layout: its layers, and steps of the same seats, share it and its workspace
        s.kept["plan"] = plan = ops.PagedPlan(s.runs, c["heads"], c["kv"], c["dim"], s.ctx, window=c["window"],
                                              sinks=c["sinks"], device=DEV)
        s.kept["ws"] = torch.empty(max(plan.workspace, 16), dtype=torch.uint8, device=DEV)
    out = torch.empty_like(s.q)
    ops.paged_attn(s.q, _own_cache(s), out, s.slots, s.pos, s.scale, s.kept["plan"], s.kept["ws"])
    return out


@torch.inference_mode()
def run(state):
    if own:
        return {"append": _own_append, "read": _own_read, "attn": _own_attn}[state.case["op"]](state)
    return {"append": _plain_append, "read": _plain_read, "attn": _plain_attn}[state.case["op"]](state)


# ---------------------------------------------------------------- 64 bits
def _rows64(s, slot, positions):
    """K and V [kv, n, dim] of a slot's positions, page by page of the table."""
    k, v = [], []
    for b in torch.unique(positions // s.case["page"]).tolist():
        inside = positions[positions // s.case["page"] == b] - b * s.case["page"]
        number = int(s.table[slot, b])
        k.append(s.k[number][:, inside])
        v.append(s.v[number][:, inside])
    return torch.cat(k, 1).double(), torch.cat(v, 1).double()


def exact(case, seed):
    s = prepare(case, seed)
    op, kv, dim = case["op"], case["kv"], case["dim"]
    if op == "read":
        found = [_rows64(s, int(s.slots[i]), s.pos[i:i + case["tokens"]].long())
                 for i in range(0, s.pos.numel(), case["tokens"])]
        return tuple(torch.cat([f[i].transpose(0, 1) for f in found]) for i in (0, 1))
    heads = case["heads"]
    if op == "append":
        x = s.qkv.double().view(-1, heads + 2 * kv, dim)
        y = x[:, :heads + kv].clone()
        if case["norm"]:
            y /= (y.pow(2).sum(-1, keepdim=True) / dim + EPS).sqrt()
            y[:, :heads] *= s.wq.double()
            y[:, heads:] *= s.wk.double()
        first, second = (slice(0, case["rot"] // 2), slice(case["rot"] // 2, case["rot"])) if case["pairs"] == "half" \
            else (slice(0, case["rot"], 2), slice(1, case["rot"], 2))
        turn = torch.polar(torch.full_like(s.inv_freq, s.factor)[None].to(DEV).expand(s.pos.numel(), -1).contiguous(),
                           torch.outer(s.pos.double(), s.inv_freq.to(DEV)))
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        k, v = s.k.double(), s.v.double()
        for r, (slot, p) in enumerate(zip(s.slots.tolist(), s.pos.tolist())):
            number = s.table[slot, p // case["page"]]
            k[number, :, p % case["page"]] = y[r, heads:]
            v[number, :, p % case["page"]] = x[r, heads + kv:]
        return y[:, :heads], k, v
    t, g, w = case["tokens"], heads // kv, case["window"]
    out = torch.zeros(s.pos.numel(), heads, dim, dtype=torch.float64, device=DEV)
    for i in range(0, case["seqs"] * t, t):
        p0, slot = int(s.pos[i]), int(s.slots[i])
        for r in range(0, t, 128):
            e = min(r + 128, t)
            lo = max(0, p0 + r - w + 1) if w else 0
            keys = torch.cat([torch.arange(min(case["sinks"], lo)), torch.arange(lo, p0 + e)]).to(DEV)
            k, v = _rows64(s, slot, keys)
            p = torch.arange(p0 + r, p0 + e, device=DEV)[:, None]
            see = (keys[None] <= p) & ((keys[None] > p - w) | (keys[None] < case["sinks"]) if w else True)
            q = s.q[i + r:i + e].double().view(e - r, kv, g, dim).permute(1, 2, 0, 3).reshape(kv, g * (e - r), dim)
            a = torch.bmm(q, k.transpose(1, 2).contiguous()).view(kv, g, e - r, -1) * s.scale
            a = torch.softmax(a.masked_fill(~see, float("-inf")), -1).view(kv, g * (e - r), -1)
            out[i + r:i + e] = torch.bmm(a, v).view(kv, g, e - r, dim).permute(2, 0, 1, 3).reshape(e - r, heads, dim)
    return out
