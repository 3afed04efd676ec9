"""The 4-bit KV cache (append, fused norm + RoPE + append, read, attention) and the 4-bit weights (pack, linear, gated)
on the GPU against float64 evaluations of their definitions."""
import numpy as np
import pytest
import torch

import fp4_reference as R

pytestmark = pytest.mark.gpu
DTYPES = (torch.bfloat16, torch.float16)


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _f64(t):
    return t.detach().cpu().double().numpy()


def _rows(rows, KV, D, dtype, seed):
    """K, V [rows, KV, D] with a few strong channels."""
    g = _g(seed)
    k = torch.randn(rows, KV, D, generator=g) * torch.exp(0.7 * torch.randn(KV, D, generator=g))
    return k.to(dtype), (torch.randn(rows, KV, D, generator=g) * 0.5).to(dtype)


def _filled(gpu, S, KV, cap, D, dtype, seed, stale=None):
    """A cache whose every position holds quantised numbers; stale: a byte that fills it first."""
    from m3x import ops
    c = ops.Kv4Cache.empty(S, KV, cap, D, gpu)
    k, v = _rows(S * cap, KV, D, dtype, seed)
    slots = torch.arange(S).repeat_interleave(cap).to(gpu)
    pos = torch.arange(cap, dtype=torch.int32).repeat(S).to(gpu)
    ops.kv4_append(k.to(gpu), v.to(gpu), c, slots, pos)
    return c


def _equal(a, b):
    return np.array_equal(a, b, equal_nan=True)


# ---------------------------------------------------------------- format
def _special(dtype):
    """Rows of 32 numbers at the edges of the format: zeros, signs, ties, scale borders, smallest and largest numbers,
    non-finite ones."""
    fi = torch.finfo(dtype)
    rows = [torch.zeros(32), -torch.zeros(32)]
    ties = torch.tensor([0.25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6])
    for s in (1.0, 2.0 ** -5, 2.0 ** 6):
        rows += [torch.cat([ties, -ties, ties * 1.01, -ties * 0.99]) * s]
    for top in (7.0, 7.0 * (1 + fi.eps), 7.0 * (1 - fi.eps), 3.5, 1.75, 6.0, 1.0):
        rows += [torch.linspace(-top, top, 32)]
    rows += [torch.linspace(-1, 1, 32) * fi.max, torch.linspace(0, 1, 32) * fi.max * 0.87, torch.full((32,), fi.tiny),
             torch.arange(32) * fi.smallest_normal * fi.eps, torch.full((32,), -fi.max)]
    for bad in (float("nan"), float("inf"), float("-inf")):
        r = torch.randn(32, generator=_g(1))
        r[5] = bad
        rows += [r]
    x = torch.stack(rows).to(dtype)
    return torch.cat([x, torch.randn(64, 32, generator=_g(2)).to(dtype)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_append_format(gpu, dtype, D):
    """Bytes in the cache and numbers read back, against the definition; every group is exact."""
    from m3x import ops
    x = _special(dtype)
    x = x[:len(x) // (D // 32) * (D // 32)].reshape(-1, 1, D)
    rows, cap = x.shape[0], 128
    c = ops.Kv4Cache.empty(2, 1, cap, D, gpu)
    perm = torch.randperm(rows, generator=_g(3))
    kx, vx = x, x[perm]
    pos = torch.randperm(cap, generator=_g(4))[:rows].int()
    slots = torch.ones(rows, dtype=torch.long)
    ops.kv4_append(kx.to(gpu), vx.to(gpu), c, slots.to(gpu), pos.to(gpu))
    K, V = R.cache_values(c, 1)
    for got, src, codes_of in ((K, kx, c.k), (V, vx, None)):
        val, code, byte = R.quantise(_f64(src[:, 0]), R.top_of(dtype))
        assert _equal(got[0, pos.long().numpy()], val)
        if codes_of is not None:
            assert np.array_equal(c.k[1, 0].cpu().numpy()[pos.long().numpy()], R.pack_nibbles(code))
            assert np.array_equal(c.ks[1, 0].cpu().numpy()[pos.long().numpy()], byte)
    assert not any(t[0].any() for t in (c.k, c.ks, c.v, c.vs))  # the other slot is untouched
    k2, v2 = torch.empty_like(kx, device=gpu), torch.empty_like(kx, device=gpu)
    ops.kv4_read(c, slots.to(gpu), pos.to(gpu), k2, v2)
    assert _equal(_f64(k2), R.quantise(_f64(kx), R.top_of(dtype))[0])
    assert _equal(_f64(v2), R.quantise(_f64(vx), R.top_of(dtype))[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_every_number(gpu, dtype):
    """Every 16-bit number next to a fixed largest one, at two scales."""
    from m3x import ops
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    for big in (6.5, 0.02):
        x = bits[torch.isfinite(bits) & (bits.abs() <= big)]
        n = len(x) // 31 // 4 * 4
        x = torch.cat([torch.full((n, 1), big).to(dtype), x[:n * 31].view(n, 31)], 1).view(-1, 1, 128)
        rows = x.shape[0]
        c = ops.Kv4Cache.empty(1, 1, -(-rows // 32) * 32, 128, gpu)
        at = torch.zeros(rows, dtype=torch.long, device=gpu), torch.arange(rows, dtype=torch.int32, device=gpu)
        ops.kv4_append(x.to(gpu), x.to(gpu), c, *at)
        val = R.quantise(_f64(x), R.top_of(dtype))[0]
        k, v = torch.empty_like(x, device=gpu), torch.empty_like(x, device=gpu)
        ops.kv4_read(c, *at, k, v)
        assert _equal(_f64(k), val) and _equal(_f64(v), val)
        s = 2.0 ** np.ceil(np.log2(big / 7))
        assert np.abs(val - _f64(x)).max() <= s


@pytest.mark.parametrize("dtype,KV,D", [(torch.bfloat16, 3, 128), (torch.float16, 8, 64), (torch.bfloat16, 1, 64)])
def test_append_read_indexing(gpu, dtype, KV, D):
    """Strided views of joint rows, shuffled slots and positions; rows outside the cache are neither written nor read,
    and nothing beside the written rows changes."""
    from m3x import ops
    S, cap, rows = 5, 96, 70
    g = _g(KV)
    joint = torch.randn(rows, 2 * KV + 1, D, generator=g).to(dtype).to(gpu)
    k, v = joint[:, 1:1 + KV], joint[:, 1 + KV:]
    flat = torch.randperm(S * cap, generator=g)[:rows]
    slots, pos = flat // cap, (flat % cap).int()
    slots[3], pos[7], pos[9], slots[11], slots[20] = -1, -1, cap, S, 2 ** 40
    pos[30] = 2 ** 31 - 1
    out = [3, 7, 9, 11, 20, 30]
    c = ops.Kv4Cache.empty(S, KV, cap, D, gpu)
    for t in (c.k, c.ks, c.v, c.vs):
        t.fill_(0x5A)
    ops.kv4_append(k, v, c, slots.to(gpu), pos.to(gpu))
    full = [R.cache_values(c, s) for s in range(S)]
    inside = [r for r in range(rows) if r not in out]
    fill = R.values_of(np.full((1, 32), 10, np.uint8), np.full((1, 1), 0x5A, np.uint8))[0, 0]
    kq, vq = R.quantise(_f64(k), R.top_of(dtype))[0], R.quantise(_f64(v), R.top_of(dtype))[0]
    for s in range(S):
        ek = np.full((KV, cap, D), np.nan)
        ev = np.full((KV, cap, D), np.nan)
        ek[..., 0::2], ev[..., 0::2] = fill, fill  # byte 0x5A: codes 10 and 5
        fill5 = R.values_of(np.full((1, 32), 5, np.uint8), np.full((1, 1), 0x5A, np.uint8))[0, 0]
        ek[..., 1::2], ev[..., 1::2] = fill5, fill5
        for r in inside:
            if slots[r] == s:
                ek[:, pos[r]], ev[:, pos[r]] = kq[r], vq[r]
        assert np.array_equal(full[s][0], ek) and np.array_equal(full[s][1], ev)
    dst = torch.full((KV, rows, 2 * D), 7.0, dtype=dtype, device=gpu)
    ko, vo = dst[:, :, :D].transpose(0, 1), dst[:, :, D:].transpose(0, 1)
    ops.kv4_read(c, slots.to(gpu), pos.to(gpu), ko, vo)
    assert not ko[out].any() and not vo[out].any()
    assert np.array_equal(_f64(ko)[inside], kq[inside]) and np.array_equal(_f64(vo)[inside], vq[inside])


@pytest.mark.parametrize("D,H,KV", [(128, 16, 8), (64, 6, 2), (128, 3, 1)])
def test_qk_norm_rope_kv4(gpu, D, H, KV):
    """The bits of qk_norm_rope_cache followed by kv4_append."""
    from m3x import ops
    rows, cap, S = 21, 64, 3
    g = _g(D + H)
    bf = torch.bfloat16
    qkv = torch.randn(rows, (H + 2 * KV) * D + 8, generator=g).to(bf).to(gpu)[:, :(H + 2 * KV) * D]
    cos, sin = torch.randn(cap, D, generator=g).to(bf).to(gpu), torch.randn(cap, D, generator=g).to(bf).to(gpu)
    wq, wk = torch.randn(D, generator=g).to(bf).to(gpu), torch.randn(D, generator=g).to(bf).to(gpu)
    flat = torch.randperm(S * cap, generator=g)[:rows]
    slots, pos = (flat // cap).to(gpu), (flat % cap).int().to(gpu)
    kc, vc = torch.zeros(S, KV, cap, D, dtype=bf, device=gpu), torch.zeros(S, KV, cap, D, dtype=bf, device=gpu)
    q0, q1 = torch.empty(rows, H, D, dtype=bf, device=gpu), torch.empty(rows, H, D, dtype=bf, device=gpu)
    ops.qk_norm_rope_cache(qkv, q0, kc, vc, slots, pos, cos, sin, wq, wk, 1e-6, H, KV)
    a, b = ops.Kv4Cache.empty(S, KV, cap, D, gpu), ops.Kv4Cache.empty(S, KV, cap, D, gpu)
    ops.kv4_append(kc[slots, :, pos.long()], vc[slots, :, pos.long()], a, slots, pos)
    ops.qk_norm_rope_kv4(qkv, q1, b, slots, pos, cos, sin, wq, wk, 1e-6, H)
    assert torch.equal(q0, q1)
    for x in ("k", "ks", "v", "vs"):
        assert torch.equal(getattr(a, x), getattr(b, x)), x
    # rows outside the cache: q still comes out, nothing is written
    before = [getattr(b, x).clone() for x in ("k", "ks", "v", "vs")]
    ops.qk_norm_rope_kv4(qkv, q1, b, torch.full_like(slots, S), pos, cos, sin, wq, wk, 1e-6, H)
    ops.qk_norm_rope_kv4(qkv, q1, b, slots, torch.full_like(pos, -1), cos, sin, wq, wk, 1e-6, H)
    assert all(torch.equal(getattr(b, x), t) for x, t in zip(("k", "ks", "v", "vs"), before))


# ---------------------------------------------------------------- attention
def _attend(q, c, slots, pos, scale, max_ctx, chunk, out=None):
    from m3x import ops
    need = ops.kv4_attn_workspace(q.shape[0], q.shape[1], q.shape[2], max_ctx, chunk)
    ws = torch.full((need // 4,), float("nan"), device=q.device) if need else None
    out = torch.full_like(q, float("nan")) if out is None else out
    ops.kv4_attn(q, c, out, slots, pos, scale, max_ctx, chunk, ws)
    return out


def _check(got, q, c, slots, pos, scale):
    vals = {}
    worst = 0.0
    got, q64 = _f64(got), _f64(q)
    for r in range(len(pos)):
        s, p = int(slots[r]), int(pos[r])
        if not 0 <= s < c.slots or p < 0:
            assert not got[r].any(), r
            continue
        if s not in vals:
            vals[s] = R.cache_values(c, s)
        out, mag, ds = R.attention(q64[r], *vals[s], p, scale)
        assert np.array_equal(np.isnan(out), np.isnan(got[r])), r
        bound = R.attention_bound(out, mag, ds, q.dtype, p + 1)
        bad = np.abs(got[r] - out) - bound
        worst = max(worst, float(np.nanmax(np.abs(got[r] - out) / bound)) if not np.isnan(out).all() else 0.0)
        assert not (bad > 0).any(), (r, s, p, float(np.nanmax(bad)))
    print(f"[fp4] attention error at most {worst:.3f} of its bound", flush=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("KV,G", [(1, 1), (2, 2), (3, 4), (1, 5), (2, 16), (1, 20)])
def test_attn_heads(gpu, dtype, D, KV, G):
    """Head layouts at ragged lengths, one of them zero, with one split and with several."""
    S, cap = 4, 320
    c = _filled(gpu, S, KV, cap, D, dtype, 10 * G + KV)
    pos = torch.tensor([0, 299, -1, 130, 31, 64, 319])
    slots = torch.tensor([2, 0, 1, 3, 1, 4, 3])  # slot 4 does not exist
    q = torch.randn(len(pos), KV * G, D, generator=_g(G)).to(dtype).to(gpu)
    scale = D ** -0.5
    for chunk in (128, 384):
        got = _attend(q, c, slots.to(gpu), pos.int().to(gpu), scale, cap, chunk)
        _check(got, q, c, slots, pos, scale)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64)])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 160, 255, 256,
                               257, 384, 500, 512])
def test_attn_lengths(gpu, dtype, D, n):
    """Every kind of length against the tiles and the splits; strided queries and outputs, what lies beside them kept."""
    KV, G, cap = 2, 2, 512
    c = _filled(gpu, 2, KV, cap, D, dtype, n)
    q = torch.randn(2, KV * G + 1, D, generator=_g(n)).to(dtype).to(gpu)[:, :KV * G]
    big = torch.full((2, 2 * KV * G, D + 8), 3.0, dtype=dtype, device=gpu)
    out = big[:, ::2, :D]
    slots, pos = torch.tensor([1, 0]), torch.tensor([n - 1, (n - 1) // 2])
    for max_ctx, chunk in ((n, 128), (cap, 128), (cap, 512)):
        got = _attend(q, c, slots.to(gpu), pos.int().to(gpu), 0.11, max_ctx, chunk, out)
        _check(got, q, c, slots, pos, 0.11)
        assert (big[:, 1::2] == 3).all() and (big[..., D:] == 3).all()


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 128), (torch.bfloat16, 64)])
@pytest.mark.parametrize("G", [1, 2, 3, 8])
def test_attn_prompt_rows(gpu, dtype, D, G):
    """Rows of one slot at consecutive positions, among single rows: each row right, and the same bits as alone."""
    KV, cap, S = 2, 288, 4
    c = _filled(gpu, S, KV, cap, D, dtype, G)
    runs = [(0, 5, 1), (1, 0, 37), (2, 100, 1), (3, 250, 38), (2, 101, 3), (0, 7, 2)]  # slot, first position, rows
    slots = torch.cat([torch.full((n,), s) for s, _, n in runs] + [torch.full((3,), 0)])
    pos = torch.cat([torch.arange(p, p + n) for _, p, n in runs] + [torch.zeros(3, dtype=torch.long)])
    q = torch.randn(len(pos), KV * G, D, generator=_g(G)).to(dtype).to(gpu)
    for chunk in (128, 384):
        got = _attend(q, c, slots.to(gpu), pos.int().to(gpu), D ** -0.5, cap, chunk)
        _check(got, q, c, slots, pos, D ** -0.5)
        order = torch.randperm(len(pos), generator=_g(5))
        alone = _attend(q[order], c, slots[order].to(gpu), pos[order].int().to(gpu), D ** -0.5, cap, chunk)
        assert torch.equal(alone, got[order])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("stale", [0xFF, 0xFE, 0x7F])
def test_attn_what_a_row_does_not_see(gpu, dtype, D, stale):
    """Stale bytes behind the last position, and a prompt's later keys and values that are NaN or infinite, have no part
    in a row's result; a row that sees them is NaN where the definition says so."""
    from m3x import ops
    KV, G, cap = 2, 2, 160
    c = ops.Kv4Cache.empty(3, KV, cap, D, gpu)
    for t in (c.k, c.ks, c.v, c.vs):
        t.fill_(stale)
    k, v = _rows(45, KV, D, dtype, 3)
    k[40, 0, 3] = float("nan")  # keys 40 (head 0) and 43 (head 1), values 41 (head 1, group 0) and 42 (last group)
    k[43, 1, 0] = float("inf")
    v[41, 1, 5] = float("nan")
    v[42, :, D - 1] = float("-inf")
    ops.kv4_append(k.to(gpu), v.to(gpu), c, torch.full((45,), 1, device=gpu), torch.arange(45, dtype=torch.int32, device=gpu))
    pos = torch.cat([torch.arange(34, 45), torch.tensor([0, 12, 31, 32])])
    slots = torch.ones(len(pos), dtype=torch.long)
    q = torch.randn(len(pos), KV * G, D, generator=_g(4)).to(dtype).to(gpu)
    for chunk in (128, 256):
        got = _attend(q, c, slots.to(gpu), pos.int().to(gpu), 0.1, cap, chunk)
        _check(got, q, c, slots, pos, 0.1)
        assert torch.isfinite(got[:6]).all()


def test_attn_extreme_scores(gpu):
    """Scores far apart, all equal, zero scale, and queries at infinity or NaN."""
    dtype, D, KV = torch.bfloat16, 128, 1
    c = _filled(gpu, 1, KV, 256, D, dtype, 9)
    q = torch.randn(7, 2, D, generator=_g(9))
    q[0] *= 1000
    q[1] *= -3000
    q[2] = 0
    q[3, 0, 7] = float("inf")
    q[4, 1, 7] = float("nan")
    q[5] *= 1e-30
    q = q.to(dtype).to(gpu)
    slots, pos = torch.zeros(7, dtype=torch.long), torch.tensor([200, 255, 100, 50, 50, 33, 180])
    for scale in (0.09, 0.0):
        rows = [0, 1, 2, 5, 6]
        got = _attend(q, c, slots.to(gpu), pos.int().to(gpu), scale, 256, 128)
        _check(got[rows], q[rows], c, slots[rows], pos[rows], scale)
        assert torch.isnan(got[3, 0]).all() and torch.isfinite(got[3, 1]).all()
        assert torch.isnan(got[4, 1]).all() and torch.isfinite(got[4, 0]).all()


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128)])
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.2, 1e-30, -1e-40, 2.0, -2.0])
def test_attn_scales(gpu, dtype, D, scale):
    """Any finite scale: 0 (every weight the same), negative, one below the smallest normal number, large."""
    c = _filled(gpu, 2, 2, 288, D, dtype, 3)
    pos, slots = torch.tensor([0, 31, 40, 41, 42, 287]), torch.tensor([1, 0, 1, 1, 1, 0])
    q = torch.randn(len(pos), 4, D, generator=_g(4)).to(dtype).to(gpu)
    for chunk in (128, 384):
        _check(_attend(q, c, slots.to(gpu), pos.int().to(gpu), scale, 288, chunk), q, c, slots, pos, scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_read_every_scale(gpu, dtype):
    """Each code at each scale byte reads as its number rounded to the type, whichever type it was written from."""
    from m3x import ops
    c = ops.Kv4Cache.empty(1, 1, 256, 64, gpu)
    code = torch.arange(64) % 16
    kb = (code[0::2] | code[1::2] << 4).to(torch.uint8)
    c.k.copy_(kb.expand(1, 1, 256, 32))
    c.ks.copy_(torch.arange(256).to(torch.uint8)[None, None, :, None].expand(1, 1, 256, 2))
    k = torch.empty(256, 1, 64, dtype=dtype, device=gpu)
    ops.kv4_read(c, torch.zeros(256, dtype=torch.long, device=gpu), torch.arange(256, dtype=torch.int32, device=gpu), k,
                 torch.empty_like(k))
    mag = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
    want = torch.cat([mag, -mag])[code] * 2.0 ** (torch.arange(256, dtype=torch.float64)[:, None] - 127)
    want = want.float().to(dtype)  # exact in fp32, one rounding to the type
    assert torch.equal(k[:255, 0].cpu(), want[:255]) and k[255].isnan().all()


def test_attn_long_split(gpu):
    """A long context in many splits (offsets of its last slot past 2^31 are in test_attn_far_slot)."""
    dtype, D = torch.bfloat16, 64
    cap = 9600
    c = _filled(gpu, 1, 1, cap, D, dtype, 2)
    q = torch.randn(2, 3, D, generator=_g(2)).to(dtype).to(gpu)
    slots, pos = torch.zeros(2, dtype=torch.long), torch.tensor([cap - 1, 5000])
    for chunk in (128, 1024):
        got = _attend(q, c, slots.to(gpu), pos.int().to(gpu), D ** -0.5, cap, chunk)
        _check(got, q, c, slots, pos, D ** -0.5)


def test_attn_far_slot(gpu):
    """A cache whose byte offsets pass 2^32: its last slot's last positions."""
    from m3x import ops
    dtype, D, KV, cap = torch.bfloat16, 128, 8, 65536
    S = 140  # 140 * 8 * 65536 * 64 bytes = 4.7e9
    c = ops.Kv4Cache.empty(S, KV, cap, D, gpu)
    k, v = _rows(40, KV, D, dtype, 1)
    at = torch.full((40,), S - 1, device=gpu), torch.arange(cap - 40, cap, dtype=torch.int32, device=gpu)
    ops.kv4_append(k.to(gpu), v.to(gpu), c, *at)
    ko, vo = torch.empty_like(k, device=gpu), torch.empty_like(k, device=gpu)
    ops.kv4_read(c, *at, ko, vo)
    kq, vq = R.quantise(_f64(k), 252)[0], R.quantise(_f64(v), 252)[0]
    assert np.array_equal(_f64(ko), kq) and np.array_equal(_f64(vo), vq)
    q = torch.randn(1, 16, D, generator=_g(2)).to(dtype).to(gpu)
    got = _f64(_attend(q, c, at[0][:1], at[1][-1:].contiguous(), 0.09, cap, 4096))[0]
    K, V = np.zeros((KV, cap, D)), np.zeros((KV, cap, D))
    K[:, -40:], V[:, -40:] = kq.transpose(1, 0, 2), vq.transpose(1, 0, 2)
    out, mag, ds = R.attention(_f64(q)[0], K, V, cap - 1, 0.09)
    assert (np.abs(got - out) <= R.attention_bound(out, mag, ds, dtype, cap)).all()


def test_step_in_a_graph_and_on_another_stream(gpu):
    """Append, attend, read and the 4-bit products captured on a side stream and replayed with eager work between the
    replays, the inputs changed each time: every replay has the eager result's bits."""
    from m3x import ops
    dtype, D, KV, H, cap, rows = torch.bfloat16, 128, 2, 4, 256, 3
    g = _g(1)
    c, e = _filled(gpu, 4, KV, cap, D, dtype, 1), _filled(gpu, 4, KV, cap, D, dtype, 1)
    w = ops.pack_weight4(torch.randn(H * D, H * D, generator=g).to(dtype).to(gpu))
    qkv = torch.empty(rows, H + 2 * KV, D, dtype=dtype, device=gpu)
    slots, pos = torch.tensor([2, 0, 3], device=gpu), torch.zeros(rows, dtype=torch.int32, device=gpu)
    ws = torch.empty(ops.kv4_attn_workspace(rows, H, D, cap, 128) // 4, device=gpu)
    out, y = torch.empty(rows, H, D, dtype=dtype, device=gpu), torch.empty(rows, H * D, dtype=dtype, device=gpu)
    ko, vo = torch.empty(rows, KV, D, dtype=dtype, device=gpu), torch.empty(rows, KV, D, dtype=dtype, device=gpu)

    def step(cache):
        ops.kv4_append(qkv[:, H:H + KV], qkv[:, H + KV:], cache, slots, pos)
        ops.kv4_attn(qkv[:, :H], cache, out, slots, pos, 0.09, cap, 128, ws)
        ops.linear4(out.view(rows, -1), w, y)
        ops.kv4_read(cache, slots, pos, ko, vo)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    qkv.normal_()
    with torch.cuda.stream(side):
        step(c)
        step(e)  # the capture's warm-up writes rows that the later passes see
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(c)
    for i in range(5):
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(dtype))
        pos.copy_(torch.tensor([i, 250 + i, 127 + i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, y, ko, vo)]
        step(e)
        torch.cuda.synchronize()
        for a, b in zip(got, (out, y, ko, vo)):
            assert torch.equal(a, b), i


# ---------------------------------------------------------------- weights
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,K", [(1, 32), (16, 128), (33, 672), (40, 1024), (17, 2816)])
def test_pack_weight4(gpu, dtype, N, K):
    from m3x import ops
    w = torch.randn(N, K + 8, generator=_g(N + K)).to(dtype)[:, :K]
    w[0, :3] = 0
    w[N - 1, K - 32:] = 0
    p = ops.pack_weight4(w.to(gpu))
    val, code, byte = R.quantise(_f64(w), R.top_of(dtype))
    assert np.array_equal(R.weight_values(p.codes, p.scales, N, K), val)
    full = R.weight_values(p.codes, p.scales, p.codes.shape[0] * 16, p.codes.shape[1] * 128)
    assert not full[N:].any() and not full[:, K:].any()
    assert p.memory_bytes() == p.codes.numel() + p.scales.numel()
    x = _special(dtype).reshape(1, -1)
    p = ops.pack_weight4(x.to(gpu))
    assert _equal(R.weight_values(p.codes, p.scales, *x.shape), R.quantise(_f64(x), R.top_of(dtype))[0])


def _product_bound(x, w, dtype):
    """K products summed in fp32 (any order), then one half step of the type."""
    y = x @ w.T
    h = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0
    return y, (x.shape[1] + 8) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T), h, tiny


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (1, 4096, 1024), (1, 17, 96), (2, 100, 160), (3, 2816, 1024), (5, 33, 672),
                                   (7, 48, 2048), (8, 1000, 512), (9, 16, 8192), (13, 250, 384), (16, 64, 4128),
                                   (17, 65, 256), (31, 200, 1024), (33, 130, 1056), (48, 31, 640), (64, 1024, 2816),
                                   (65, 80, 128), (130, 47, 544), (300, 256, 1024)])
def test_linear4(gpu, dtype, M, N, K):
    from m3x import ops
    g = _g(M * 31 + N + K)
    x = torch.randn(M, K + 16, generator=g).to(dtype)[:, 8:8 + K].to(gpu)
    p = ops.pack_weight4((torch.randn(N, K, generator=g) * K ** -0.5).to(dtype).to(gpu))
    w = R.weight_values(p.codes, p.scales, N, K)
    y, sums, h, tiny = _product_bound(_f64(x), w, dtype)
    big = torch.full((M, N + 5), 3.0, dtype=dtype, device=gpu)
    for out in (None, big[:, 2:2 + N]):
        got = _f64(ops.linear4(x, p, out))
        assert (np.abs(got - y) <= sums + h * (np.abs(y) + sums) + tiny).all()
    assert (big[:, :2] == 3).all() and (big[:, 2 + N:] == 3).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,I,K", [(1, 2816, 1024), (3, 50, 96), (16, 128, 2048), (20, 33, 512), (64, 2816, 1024),
                                   (100, 17, 352)])
def test_linear4_act(gpu, dtype, M, I, K):
    """silu(g) u and gelu(g): the slopes are at most 1.13, so a product's error passes at most 1.13 times; the activations
    themselves are within 2^-20 of their value."""
    from scipy.special import erf
    from m3x import ops
    g = _g(M + I + K)
    x = (torch.randn(M, K, generator=g) * 2).to(dtype).to(gpu)
    p = ops.pack_weight4((torch.randn(2 * -(-I // 16) * 16, K, generator=g) * K ** -0.5).to(dtype).to(gpu))
    half = p.N // 2
    pg, pu = p.rows(0, I), p.rows(half, half + I)
    w = R.weight_values(p.codes, p.scales, p.N, K)
    a, da, h, tiny = _product_bound(_f64(x), w[:I], dtype)
    b, db, _, _ = _product_bound(_f64(x), w[half:half + I], dtype)
    act = a / (1 + np.exp(-a))
    for kind, up, y, off in ((ops.ACT_SWIGLU, pu, act * b, 1.13 * da * (np.abs(b) + db) + np.abs(act) * db),
                             (ops.ACT_GELU, None, 0.5 * a * (1 + erf(a / 2 ** 0.5)), 1.13 * da)):
        # erff's absolute error near -1 is about an ulp of 1, times |a| / 2
        off = off + 2.0 ** -20 * np.abs(y) + (np.abs(a) * 2.0 ** -23 if up is None else 0)
        got = _f64(ops.linear4_act(x, pg, up, kind))
        assert (np.abs(got - y) <= off + h * (np.abs(y) + off) + tiny).all()


def test_linear4_no_numbers(gpu):
    """A NaN group makes its own output column NaN, an infinite input its own row non-finite; nothing else changes."""
    from m3x import ops
    dtype = torch.bfloat16
    w = torch.randn(40, 256, generator=_g(1))
    w[7, 200] = float("nan")
    x = torch.randn(5, 256, generator=_g(2))
    clean = ops.linear4(x.to(dtype).to(gpu), ops.pack_weight4(torch.nan_to_num(w).to(dtype).to(gpu)))
    x[3, 100] = float("inf")
    got = ops.linear4(x.to(dtype).to(gpu), ops.pack_weight4(w.to(dtype).to(gpu)))
    keep_r, keep_c = [0, 1, 2, 4], [i for i in range(40) if i != 7]
    assert torch.isnan(got[:, 7]).all() and not torch.isfinite(got[3]).any()
    assert torch.equal(got[keep_r][:, keep_c], clean[keep_r][:, keep_c])


def test_no_rows(gpu):
    from m3x import ops
    c = ops.Kv4Cache.empty(1, 2, 32, 64, gpu)
    z = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=gpu)
    at = torch.empty(0, dtype=torch.long, device=gpu), torch.empty(0, dtype=torch.int32, device=gpu)
    ops.kv4_append(z, z, c, *at)
    ops.kv4_read(c, *at, z, z)
    ops.kv4_attn(z, c, z, *at, 1.0, 32, 128, None)
    p = ops.pack_weight4(torch.zeros(16, 64, dtype=torch.bfloat16, device=gpu))
    assert ops.linear4(torch.empty(0, 64, dtype=torch.bfloat16, device=gpu), p).shape == (0, 16)
