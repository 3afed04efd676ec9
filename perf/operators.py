"""The framework's 4-bit serving operators as timed cases: what a serving step does with a KV cache and with weights
held in 4 bits.

Four operators share one format. A group of 32 numbers is held as 32 E2M1 codes (bit 3 the sign, bits 0..2 the
magnitude 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one scale byte b that stands for 2^(b - 127): the smallest power of two s
with max|x| <= 7 s, b in [1, 252] (fp16 numbers: at most 140, so that every value is finite); codes round to the
nearest, ties to the even code, above 6 to 6. A group with a NaN or an infinity in it has b = 255 and reads as NaN.

  append  K and V rows (views of a step's q|k|v rows) quantised into a cache at (slot, position), then read back: the
          writer and the reader of the cache, as a prompt's prefix is stored and exported
  read    positions of the cache as 16-bit rows
  attn    attention of each row's query heads over its slot's positions 0 .. pos: single tokens and whole prompts
          (consecutive rows of one slot), rows with no position (pos = -1) give zeros
  linear  y = x W^T with W in 4 bits
  gated   silu(x Wg^T) * (x Wu^T) with both in 4 bits

The cache of `kv` heads of `dim` numbers, `cap` positions a slot:
  k   uint8 [slots, kv, cap, dim / 2]             byte j: dims 2j (low half) and 2j + 1
  ks  uint8 [slots, kv, cap, dim / 32]            scale bytes
  v   uint8 [slots, kv, cap / 4, 16, 4, dim / 32] four positions together: chunk c holds dims c * dim/16 ...
  vs  uint8 [slots, kv, cap / 4, dim / 32, 4]
A weight [N, K], N in tiles of 16 rows (zero rows behind N), K in steps of 128 (zeros behind K):
  codes  uint8 [N / 16, K / 128, 64, 16]  lane l's 16 bytes: row l % 16 of the tile, dims 32 (l / 16) .. + 31 of the step
  scales uint8 [N / 16, ceil(K / 512), 64, 4]  the same lane's byte of four consecutive steps
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
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # a lone stream writes its token's K/V: the smallest call
        dict(name="append_1", op="append", seqs=1, tokens=1, cap=2048, kv=8, dim=128, dtype="bf16"),
        # eight prompts of 256 tokens admitted in one step
        dict(name="append_8x256", op="append", seqs=8, tokens=256, cap=2048, kv=8, dim=128, dtype="bf16"),
        # whole contexts exported, smaller heads, an odd length
        dict(name="read_16x4095", op="read", seqs=16, tokens=4095, cap=4096, kv=8, dim=64, dtype="fp16"),
        # a lone stream's token over a long context: latency
        dict(name="attn_1", op="attn", seqs=1, tokens=1, empty=0, ctx=2048, spread=False, heads=16, kv=8, dim=128,
             dtype="bf16"),
        # a full GPU in steady state
        dict(name="attn_224", op="attn", seqs=224, tokens=1, empty=0, ctx=2048, spread=False, heads=16, kv=8, dim=128,
             dtype="bf16"),
        # streams of all ages behind four query heads a KV head, padded to the next row bucket
        dict(name="attn_61_spread", op="attn", seqs=61, tokens=1, empty=3, ctx=4000, spread=True, heads=32, kv=8,
             dim=128, dtype="fp16"),
        # two very long contexts, small heads
        dict(name="attn_2_long", op="attn", seqs=2, tokens=1, empty=0, ctx=120001, spread=False, heads=32, kv=4,
             dim=64, dtype="bf16"),
        # eight prompts of 200 tokens onto prefixes: rows of one slot
        dict(name="attn_8x200", op="attn", seqs=8, tokens=200, empty=0, ctx=500, spread=False, heads=16, kv=8, dim=128,
             dtype="bf16"),
        # one row through a backbone's q|k|v projection
        dict(name="linear_1", op="linear", rows=1, n=4096, k=1024, dtype="bf16"),
        # a small batch through a large layer: the weights are all the traffic
        dict(name="linear_9_large", op="linear", rows=9, n=16384, k=8192, dtype="fp16"),
        # the gated half of a feed-forward block, for a few rows and for a part-filled GPU
        dict(name="gated_3", op="gated", rows=3, n=2816, k=1024, dtype="fp16"),
        dict(name="gated_64", op="gated", rows=64, n=2816, k=1024, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("append", "read", "attn", "attn", "attn", "linear", "linear", "gated"))
    dtype = rng.choice(("bf16", "fp16"))
    kv, dim = rng.choice((1, 2, 4, 8)), rng.choice((64, 128, 128))
    if op in ("append", "read"):
        seqs = _log(rng, 1, 64)
        tokens = _log(rng, 1, 65536 // seqs // kv) if op == "read" else _log(rng, 1, max(1, 4096 // seqs))
        return dict(op=op, seqs=seqs, tokens=tokens, cap=-(-(tokens + rng.randint(0, 600)) // 32) * 32, kv=kv, dim=dim,
                    dtype=dtype)
    if op == "attn":
        ratio = rng.choice((1, 2, 2, 4, 5, 8))
        if rng.random() < 0.3:  # prompts
            seqs = rng.randint(1, 8)
            tokens = _log(rng, 2, 200)
            ctx = tokens + _log(rng, 1, 400)
        else:
            seqs, tokens = _log(rng, 1, 224), 1
            ctx = _log(rng, 1, min(120000, 224 * 2048 // seqs))
        return dict(op=op, seqs=seqs, tokens=tokens, empty=rng.choice((0, 0, 1, 3)), ctx=ctx,
                    spread=tokens == 1 and rng.random() < 0.5, heads=kv * ratio, kv=kv, dim=dim, dtype=dtype)
    rows = _log(rng, 1, 64)
    return dict(op=op, rows=rows, n=_log(rng, 16, 16384 if op == "linear" else 8192), k=32 * _log(rng, 2, 256),
                dtype=dtype)


def _lengths(case):
    """Positions that each sequence holds after the step, the same for every seed (their order is the seed's)."""
    s, ctx, t = case["seqs"], case["ctx"], case["tokens"]
    if case["spread"]:
        return [max(t, ctx * (i + 1) // s) for i in range(s)]
    return [max(t, ctx - (7 * i) % 16) for i in range(s)]


def work(case):
    op = case["op"]
    if op in ("append", "read"):
        numbers = 2 * case["seqs"] * case["tokens"] * case["kv"] * case["dim"]
        packed = numbers / 2 + numbers / 32
        # append's pass writes the cache and reads it back
        return {"bytes": numbers * 2 + packed if op == "read" else 2 * (numbers * 2 + packed), "flops": 0}
    if op == "attn":
        n, t = _lengths(case), case["tokens"]
        rows = case["seqs"] * t + case["empty"]
        seen = sum(sum(range(x - t + 1, x + 1)) for x in n)
        return {"bytes": sum(n) * case["kv"] * case["dim"] * 2 * (1 / 2 + 1 / 32)
                + 2 * rows * case["heads"] * case["dim"] * 2,
                "flops": 4 * case["heads"] * case["dim"] * seen}
    m, n, k = case["rows"], case["n"], case["k"]
    two = 2 if op == "gated" else 1
    return {"bytes": two * n * k * (1 / 2 + 1 / 32) + m * k * 2 + m * n * 2, "flops": 2 * two * m * n * k}


# ---------------------------------------------------------------- inputs
def _gen(seed, n=0):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + n)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rows(case, seed, g):
    """K and V rows of one call as views of its q|k|v rows, keys with a few strong channels as trained ones have."""
    rows, kv, dim = case["seqs"] * case["tokens"], case["kv"], case["dim"]
    x = _normal(g, rows, 4 * kv, dim)
    x[:, 2 * kv:3 * kv] *= torch.exp(0.7 * _normal(g, kv, dim))
    x[:, 3 * kv:] *= 0.5
    x = x.to(DT[case["dtype"]])
    return x, x[:, 2 * kv:3 * kv], x[:, 3 * kv:]


def _cache(case, slots, cap, g):
    """A filled cache: quantised keys and values, a slot at a time."""
    kv, dim = case["kv"], case["dim"]
    top = 140 if case["dtype"] == "fp16" else 252
    c = _empty_cache(case, slots, cap)
    strong = torch.exp(0.7 * _normal(g, kv, 1, dim))
    for s in range(slots):
        k, v = _normal(g, kv, cap, dim) * strong, _normal(g, kv, cap, dim) * 0.5
        codes, c.ks[s] = _quantise(k, top)
        c.k[s] = _bytes(codes)
        codes, scales = _quantise(v, top)
        c.v[s] = _bytes(codes).view(kv, cap // 4, 4, 16, dim // 32).transpose(2, 3)
        c.vs[s] = scales.view(kv, cap // 4, 4, dim // 32).transpose(2, 3)
    return c


def _empty_cache(case, slots, cap):
    kv, dim = case["kv"], case["dim"]
    new = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device=DEV)  # noqa: E731
    return SimpleNamespace(k=new(slots, kv, cap, dim // 2), ks=new(slots, kv, cap, dim // 32),
                           v=new(slots, kv, cap // 4, 16, 4, dim // 32), vs=new(slots, kv, cap // 4, dim // 32, 4))


def _weight(case, g):
    n, k = case["n"], case["k"]
    np_, kp = -(-n // 16) * 16, -(-k // 128) * 128
    w = torch.zeros(np_, kp, device=DEV)
    w[:n, :k] = _normal(g, n, k) * (k ** -0.5)
    codes, scales = _quantise(w, 252)
    steps = kp // 128
    codes = _bytes(codes).view(np_ // 16, 16, steps, 4, 16).permute(0, 2, 3, 1, 4).reshape(np_ // 16, steps, 64, 16)
    full = torch.zeros(np_, -(-steps // 4), 4, 4, dtype=torch.uint8, device=DEV)  # row, four steps, step, group
    full.view(np_, -1, 4)[:, :steps] = scales.view(np_, steps, 4)
    full = full.view(np_ // 16, 16, -1, 4, 4).permute(0, 2, 4, 1, 3).reshape(np_ // 16, -1, 64, 4)
    return codes.contiguous(), full.contiguous()


def prepare(case, seed):
    op, g = case["op"], _gen(seed)
    s = SimpleNamespace(case=dict(case), kept={})
    rng = random.Random(int(seed) * 31 + 5)
    if op in ("append", "read"):
        slots = case["seqs"] + 1
        at = rng.sample(range(slots), case["seqs"])
        first = [rng.randint(0, case["cap"] - case["tokens"]) for _ in at]
        s.slots = torch.tensor(at, device=DEV).repeat_interleave(case["tokens"])
        s.pos = (torch.tensor(first, device=DEV)[:, None] + torch.arange(case["tokens"], device=DEV)).flatten().int()
        if op == "append":
            s.cache = _empty_cache(case, slots, case["cap"])
            s.qkv, s.k, s.v = _rows(case, seed, g)
        else:
            s.cache = _cache(case, slots, case["cap"], g)
    elif op == "attn":
        n, t = _lengths(case), case["tokens"]
        rng.shuffle(n)
        s.cap = -(-max(n) // 32) * 32
        slots = case["seqs"] + 1
        s.cache = _cache(case, slots, s.cap, g)
        at = rng.sample(range(slots), case["seqs"])
        pos = (torch.tensor(n, device=DEV)[:, None] - t + torch.arange(t, device=DEV)).flatten()
        e = case["empty"]
        s.slots = torch.cat([torch.tensor(at, device=DEV).repeat_interleave(t), torch.zeros(e, dtype=torch.long, device=DEV)])
        s.pos = torch.cat([pos, torch.full((e,), -1, device=DEV)]).int()
        s.q = _normal(g, s.pos.numel(), case["heads"], case["dim"]).to(DT[case["dtype"]])
        s.ctx, s.scale = max(n), case["dim"] ** -0.5
    else:
        s.x = _normal(g, case["rows"], case["k"]).to(DT[case["dtype"]])
        s.w = _weight(case, g)
        if op == "gated":
            s.up = _weight(case, g)
    return s


# ---------------------------------------------------------------- plain forms
def _quantise(x, top):
    """(codes uint8 like x, scale bytes uint8 [..., dim / 32])."""
    x = x.float()
    grp = x.reshape(*x.shape[:-1], -1, 32)
    amax = grp.abs().amax(-1)
    good = torch.isfinite(amax)
    m, e = torch.frexp(torch.where(good, amax, torch.zeros_like(amax)))
    e = torch.where(m <= 0.875, e - 3, e - 2).clamp(-126, top - 127)  # amax = m 2^e, m in [0.5, 1)
    e = torch.where(amax == 0, torch.full_like(e, -126), e)
    a = torch.ldexp(torch.where(good[..., None], grp, torch.zeros_like(grp)).abs(), -e[..., None])
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = code + 8 * (torch.signbit(grp) & good[..., None]).to(torch.uint8)
    return code.view(x.shape), torch.where(good, e + 127, torch.full_like(e, 255)).to(torch.uint8)


def _bytes(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _halves(b):
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _values(codes, scales):
    """The float32 numbers of codes [..., dim] under scale bytes [..., dim / 32]."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    s = torch.where(scales == 255, torch.full((), float("nan"), device=codes.device),
                    torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.int() - 127))
    x = table[codes.int()].view(*codes.shape[:-1], -1, 32)
    return (x * s[..., None]).view(codes.shape)


def _dim_major(v, vs):
    """V's codes [..., cap, dim] and scale bytes [..., cap, dim / 32] from their blocks of four positions."""
    v = v.transpose(-3, -2).flatten(-2)  # [..., cap / 4, 4, dim / 2]
    return _halves(v.flatten(-3, -2)), vs.transpose(-2, -1).flatten(-3, -2)


def _plain_append(s):
    c, dim, top = s.cache, s.case["dim"], 140 if s.case["dtype"] == "fp16" else 252
    p = s.pos.long()
    codes, scales = _quantise(s.k, top)
    c.k[s.slots, :, p] = _bytes(codes)
    c.ks[s.slots, :, p] = scales
    codes, scales = _quantise(s.v, top)
    c.v[s.slots, :, p // 4, :, p % 4] = _bytes(codes).view(*codes.shape[:2], 16, dim // 32)
    c.vs[s.slots, :, p // 4, :, p % 4] = scales


def _plain_read(s):
    c, p, dt = s.cache, s.pos.long(), DT[s.case["dtype"]]
    k = _values(_halves(c.k[s.slots, :, p]), c.ks[s.slots, :, p])
    v = _values(_halves(c.v[s.slots, :, p // 4, :, p % 4].flatten(-2)), c.vs[s.slots, :, p // 4, :, p % 4])
    return k.to(dt), v.to(dt)


def _plain_attn(s):
    case, c = s.case, s.cache
    t, kv, dim = case["tokens"], case["kv"], case["dim"]
    n = case["seqs"] * t
    first = s.slots[:n:t]  # one gather of the cache per sequence
    k = _values(_halves(c.k[first]), c.ks[first])
    v = _values(*_dim_major(c.v[first], c.vs[first]))
    g = case["heads"] // kv
    q = s.q[:n].float().view(case["seqs"], t, kv, g, dim).permute(0, 2, 1, 3, 4).reshape(case["seqs"], kv, t * g, dim)
    score = torch.matmul(q, k.transpose(-1, -2)) * s.scale
    last = s.pos[:n].view(case["seqs"], 1, t, 1, 1)
    score = score.view(case["seqs"], kv, t, g, -1)
    score = score.masked_fill(torch.arange(score.shape[-1], device=DEV) > last, float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(case["seqs"], kv, t * g, -1), v).view(case["seqs"], kv, t, g, dim)
    o = o.permute(0, 2, 1, 3, 4).reshape(n, case["heads"], dim)
    return torch.cat([o, torch.zeros(case["empty"], case["heads"], dim, device=DEV)]).to(s.q.dtype)


def _plain_weight(w, n, k):
    codes, scales = w
    tiles, steps = codes.shape[:2]
    codes = _halves(codes).view(tiles, steps, 4, 16, 32).permute(0, 3, 1, 2, 4).reshape(tiles * 16, steps * 128)
    scales = scales.view(tiles, -1, 4, 16, 4).permute(0, 3, 1, 4, 2).reshape(tiles * 16, -1)[:, :steps * 4]
    return _values(codes, scales)[:n, :k]


def _plain_linear(s):
    n, k = s.case["n"], s.case["k"]
    return (s.x.float() @ _plain_weight(s.w, n, k).t()).to(s.x.dtype)


def _plain_gated(s):
    n, k = s.case["n"], s.case["k"]
    x = s.x.float()
    g, u = x @ _plain_weight(s.w, n, k).t(), x @ _plain_weight(s.up, n, k).t()
    return (g / (1 + torch.exp(-g)) * u).to(s.x.dtype)


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
        s.kept["cache"] = _ops().Kv4Cache(s.cache.k, s.cache.ks, s.cache.v, s.cache.vs)
    return s.kept["cache"]


def _own_read(s):
    shape = (s.pos.numel(), s.case["kv"], s.case["dim"])
    dt = DT[s.case["dtype"]]
    k, v = torch.empty(shape, dtype=dt, device=DEV), torch.empty(shape, dtype=dt, device=DEV)
    _ops().kv4_read(_own_cache(s), s.slots, s.pos, k, v)
    return k, v


def _own_append(s):
    _ops().kv4_append(s.k, s.v, _own_cache(s), s.slots, s.pos)
    return _own_read(s)


def _own_attn(s):
    ops = _ops()
    if "ws" not in s.kept:  # a program keeps its workspace
        s.kept["chunk"] = ops.kv4_attn_chunk(s.pos.numel(), s.case["heads"], s.case["kv"], s.ctx, s.case["dim"])
        need = ops.kv4_attn_workspace(s.pos.numel(), s.case["heads"], s.case["dim"], s.ctx, s.kept["chunk"])
        s.kept["ws"] = torch.empty(need // 4, dtype=torch.float32, device=DEV)
    out = torch.empty_like(s.q)
    ops.kv4_attn(s.q, _own_cache(s), out, s.slots, s.pos, s.scale, s.ctx, s.kept["chunk"], s.kept["ws"])
    return out


def _own_weight(s, name, w):
    if name not in s.kept:
        s.kept[name] = _ops().PackedWeight4(*w, s.case["n"], s.case["k"])
    return s.kept[name]


def _own_linear(s):
    return _ops().linear4(s.x, _own_weight(s, "w", s.w))


def _own_gated(s):
    ops = _ops()
    return ops.linear4_act(s.x, _own_weight(s, "w", s.w), _own_weight(s, "up", s.up), ops.ACT_SWIGLU)


@torch.inference_mode()
def run(state):
    op = state.case["op"]
    if own:
        return {"append": _own_append, "read": _own_read, "attn": _own_attn, "linear": _own_linear,
                "gated": _own_gated}[op](state)
    if op == "append":
        _plain_append(state)
    if op in ("append", "read"):
        return _plain_read(state)
    return {"attn": _plain_attn, "linear": _plain_linear, "gated": _plain_gated}[op](state)


# ---------------------------------------------------------------- 64 bits
def _number64(code, byte):
    """The number of one code array under its scale bytes, from the bits: sign, exponent and one mantissa bit."""
    code = code.to(torch.int64)
    ex, man = (code >> 1) & 3, (code & 1).double()
    mag = torch.where(ex == 0, 0.5 * man, (1 + 0.5 * man) * torch.pow(2.0, (ex - 1).double()))
    scale = torch.pow(2.0, byte.double() - 127)
    scale[byte == 255] = float("nan")
    return torch.where(code > 7, -mag, mag) * scale


def _row64(low_high, scale, dim):
    """Numbers of bytes [..., dim / 2] under scale bytes [..., dim / 32]."""
    x = torch.empty(*low_high.shape[:-1], dim, dtype=torch.float64, device=low_high.device)
    x[..., 0::2] = _number64(low_high % 16, scale.repeat_interleave(16, -1))
    x[..., 1::2] = _number64(low_high // 16, scale.repeat_interleave(16, -1))
    return x


def _round64(x, top):
    """Each group's numbers on the 4-bit grid of the smallest scale that holds them."""
    out = torch.empty_like(x, dtype=torch.float64)
    for j in range(0, x.shape[-1], 32):
        grp = x[..., j:j + 32].double()
        big = grp.abs().amax(-1, keepdim=True)
        e = torch.ceil(torch.log2((big / 7).clamp_min(2.0 ** -126)))
        e = torch.where(big > 7 * torch.pow(2.0, e), e + 1, torch.where(big <= 7 * torch.pow(2.0, e - 1), e - 1, e))
        s = torch.pow(2.0, e.clamp(-126, top - 127))
        a = (grp / s).abs()
        a = torch.where(a < 2, torch.round(2 * a) / 2, torch.where(a < 4, torch.round(a), 2 * torch.round(a / 2)))
        out[..., j:j + 32] = torch.sign(grp) * a.clamp_max(6) * s
    return out


def _cache64(c, slot, cap, dim):
    """K and V [kv, cap, dim] of one slot."""
    k = _row64(c.k[slot], c.ks[slot], dim)
    v = torch.stack([_row64(c.v[slot, :, :, :, i].flatten(-2), c.vs[slot, :, :, :, i], dim) for i in range(4)], 2)
    return k, v.reshape(k.shape)


def exact(case, seed):
    s = prepare(case, seed)
    op, dim = case["op"], case.get("dim")
    if op == "append":
        top = 140 if case["dtype"] == "fp16" else 252
        return _round64(s.k, top), _round64(s.v, top)
    if op == "read":
        ks, vs = [], []
        for i in range(0, s.pos.numel(), case["tokens"]):
            k, v = _cache64(s.cache, int(s.slots[i]), case["cap"], dim)
            a = int(s.pos[i])
            ks.append(k[:, a:a + case["tokens"]].transpose(0, 1))
            vs.append(v[:, a:a + case["tokens"]].transpose(0, 1))
        return torch.cat(ks), torch.cat(vs)
    if op == "attn":
        t, g = case["tokens"], case["heads"] // case["kv"]
        out = torch.zeros(s.pos.numel(), case["heads"], dim, dtype=torch.float64, device=DEV)
        for i in range(0, case["seqs"] * t, t):
            k, v = _cache64(s.cache, int(s.slots[i]), s.cap, dim)
            for r in range(i, i + t, 64):
                e = min(r + 64, i + t)
                q = s.q[r:e].double().view(e - r, case["kv"], g, dim)
                a = torch.matmul(q.permute(1, 0, 2, 3).reshape(case["kv"], -1, dim), k.transpose(-1, -2).contiguous()) * s.scale
                a = a.view(case["kv"], e - r, g, -1)
                a[(torch.arange(a.shape[-1], device=DEV)[None] > s.pos[r:e, None])[None, :, None].expand_as(a)] = float("-inf")
                a = torch.softmax(a, -1).view(case["kv"], -1, a.shape[-1])
                out[r:e] = torch.matmul(a, v).view(case["kv"], e - r, g, dim).transpose(0, 1).reshape(e - r, -1, dim)
        return out
    x, n, k = s.x.double(), case["n"], case["k"]

    def product(w):
        y = torch.empty(case["rows"], w[0].shape[0] * 16, dtype=torch.float64, device=DEV)
        steps = w[0].shape[1]
        xp = torch.zeros(case["rows"], steps * 128, dtype=torch.float64, device=DEV)
        xp[:, :k] = x
        for lane in range(16):
            at = torch.arange(4, device=DEV) * 16 + lane
            rows = w[0][:, :, at]  # [tiles, steps, 4, 16]
            sc = w[1][:, :, at].transpose(-1, -2).flatten(1, 2)[:, :steps]  # [tiles, steps, 4]
            y[:, lane::16] = xp @ _row64(rows, sc[..., None], 32).flatten(1).t()
        return y[:, :n]

    if op == "linear":
        return product(s.w)
    a, b = product(s.w), product(s.up)
    return a * torch.sigmoid(a) * b
