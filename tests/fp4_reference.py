"""The 4-bit group format and the operators over it in float64 (numpy), written from their definitions: the expected
results of the tests of the 4-bit cache and weights."""
import numpy as np
import torch

GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


def quantise(x, top):
    """(values, codes, scale bytes) of float64 x [..., 32 n]; groups with a non-finite number are NaN (code 0, byte
    255)."""
    x = np.asarray(x, dtype=np.float64)
    g = x.reshape(*x.shape[:-1], -1, 32)
    ok = np.isfinite(g).all(-1)
    amax = np.where(ok, np.abs(np.where(np.isfinite(g), g, 0)).max(-1), 0)
    byte = np.full(amax.shape, 1, dtype=np.int64)
    while True:  # the smallest power of two that holds the group
        grow = (amax > 7 * np.ldexp(1.0, byte - 127)) & (byte < top)
        if not grow.any():
            break
        byte[grow] += 1
    a = np.abs(np.where(ok[..., None], g, 0)) / np.ldexp(1.0, byte - 127)[..., None]
    d = np.abs(np.minimum(a, 6.0)[..., None] - GRID)
    best = d.min(-1, keepdims=True)
    cand = d == best  # one or two neighbours; of two the even code
    even = cand & (np.arange(8) % 2 == 0)
    code = np.where(cand.sum(-1) > 1, even.argmax(-1), cand.argmax(-1))
    neg = np.signbit(g) & ok[..., None]
    val = np.where(neg, -1.0, 1.0) * GRID[code] * np.ldexp(1.0, byte - 127)[..., None]
    val = np.where(ok[..., None], val, np.nan)
    code = np.where(ok[..., None], code + 8 * neg, 0)
    byte = np.where(ok, byte, 255)
    return val.reshape(x.shape), code.reshape(x.shape).astype(np.uint8), byte.astype(np.uint8)


def top_of(dtype):
    return 140 if dtype == torch.float16 else 252


def pack_nibbles(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def values_of(codes, byte):
    """Values of codes [..., 32 n] under scale bytes [..., n]."""
    with np.errstate(over="ignore", invalid="ignore"):
        s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(np.int64) - 127))
    v = np.where(codes > 7, -1.0, 1.0) * GRID[codes & 7]
    return (v.reshape(*codes.shape[:-1], -1, 32) * s[..., None]).reshape(codes.shape)


def unpack_nibbles(b):
    out = np.empty(b.shape[:-1] + (2 * b.shape[-1],), dtype=np.uint8)
    out[..., 0::2] = b & 15
    out[..., 1::2] = b >> 4
    return out


def cache_values(cache, slot):
    """(K, V) [kv_heads, cap, D] float64 of one slot of an ops.Kv4Cache."""
    k, ks = cache.k[slot].cpu().numpy(), cache.ks[slot].cpu().numpy()
    v, vs = cache.v[slot].cpu().numpy(), cache.vs[slot].cpu().numpy()
    KV, cap, half = k.shape
    rows = np.empty((KV, cap, half), dtype=np.uint8)
    scales = np.empty_like(ks)
    per = half // 16
    for p in range(4):
        for c in range(16):
            rows[:, p::4, c * per:(c + 1) * per] = v[:, :, c, p]
        scales[:, p::4] = vs[:, :, :, p]
    return values_of(unpack_nibbles(k), ks), values_of(unpack_nibbles(rows), scales)


def weight_values(codes, scales, N, K):
    """[N, K] float64 of a packed weight's bytes."""
    codes, scales = codes.cpu().numpy(), scales.cpu().numpy()
    tiles, steps = codes.shape[:2]
    w = np.empty((tiles * 16, steps * 128))
    for lane in range(64):
        row, g = lane % 16, lane // 16
        for s in range(steps):
            w[row::16, 128 * s + 32 * g:128 * s + 32 * g + 32] = values_of(
                unpack_nibbles(codes[:, s, lane]), scales[:, s // 4, lane, s % 4][:, None])
    return w[:N, :K]


def attention(q, K, V, pos, scale):
    """(out, A, dS) [heads, D] of one row's queries over keys 0 .. pos of its slot (K, V [kv_heads, cap, D]): the
    output, sum p |v| and a bound of the scores' fp32 rounding."""
    H, D = q.shape
    KV = K.shape[0]
    G = H // KV
    out, mag, ds = np.zeros((H, D)), np.zeros((H, D)), np.zeros((H, 1))
    if pos < 0:
        return out, mag, ds
    for h in range(H):
        k, v = K[h // G, :pos + 1], V[h // G, :pos + 1]
        with np.errstate(invalid="ignore"):
            s = k @ q[h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[h], mag[h] = p @ v, p @ np.abs(v)
            # a score sums D exact products in fp32 (D + 2 roundings with the scaling), an exponent adds two more
            ds[h] = (D + 4) * 2.0 ** -24 * ((np.abs(k) @ np.abs(q[h])).max() * abs(scale) + 1)
    return out, mag, ds


def attention_bound(out, mag, ds, dtype, keys):
    """How far a kernel's output may be off: the weights rounded to the 16-bit type, the scores' fp32 rounding in
    numerator and denominator, the fp32 sums over the keys, and the store's half step.

    The rounded weights p (1 + d), |d| <= h, stand in numerator and denominator: sum p (1 + d) v / sum p (1 + d) - out =
    sum p d (v - out) / sum p (1 + d), at most h / (1 - h) (sum p |v| + |out|) for weights that sum to 1. Either sum is
    off by at most 2^-24 a key and term (the denominator's takes two keys at a time, within 3.4 * 2^-24)."""
    h = torch.finfo(dtype).eps / 2
    sums = (2 * keys + 16) * 2.0 ** -24
    return h / (1 - h) * (mag + np.abs(out)) + 2 * ds * mag + sums * mag + h * np.abs(out) + 1e-30 + \
        (2.0 ** -25 if dtype == torch.float16 else 0)  # half a step of fp16's smallest numbers
