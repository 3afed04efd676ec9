"""Attention over the 4-bit cache at the ends of its numbers' range: scores and scales far from 1, against float64
evaluations under bounds for scores that are exact in fp32."""
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


def _attend(q, c, slots, pos, scale, chunk):
    from m3x import ops
    need = ops.kv4_attn_workspace(q.shape[0], q.shape[1], q.shape[2], c.cap, chunk)
    ws = torch.full((max(need, 16) // 4,), float("nan"), device=q.device)
    out = torch.full_like(q, float("nan"))
    ops.kv4_attn(q, c, out, slots.to(q.device), pos.int().to(q.device), scale, c.cap, chunk, ws)
    return out


def _exact_scores(gpu, dtype, seed):
    """A cache and queries whose scores are exact in fp32 in any order of summation: half of the dimensions give every
    key 2^22 (32 products of 4 and 2^15), four others multiples of 0.5 up to 24, so all partial sums are multiples of 0.5
    below 2^23. Every group's largest number is 4 or 6: its scale is 1 and the numbers are the format's."""
    from m3x import ops
    S, KV, cap, D, H = 2, 2, 288, 64, 4
    g = _g(seed)
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6])
    k = torch.zeros(S * cap, KV, D)
    k[..., :32] = 4
    k[..., 32:36] = grid[torch.randint(0, 8, (S * cap, KV, 4), generator=g)] * (
        1 - 2 * torch.randint(0, 2, (S * cap, KV, 4), generator=g))
    k[..., 63] = 6
    v = torch.randn(S * cap, KV, D, generator=g)
    c = ops.Kv4Cache.empty(S, KV, cap, D, gpu)
    ops.kv4_append(k.to(dtype).to(gpu), v.to(dtype).to(gpu), c, torch.arange(S, device=gpu).repeat_interleave(cap),
                   torch.arange(cap, dtype=torch.int32, device=gpu).repeat(S))
    assert np.array_equal(R.cache_values(c, 1)[0], _f64(k.view(S, cap, KV, D)[1].transpose(0, 1)))
    slots = torch.tensor([1, 0, 0, 0, 1] + [1] * 11)
    pos = torch.tensor([287, 0, 31, 140, 5] + list(range(120, 131)))
    q = torch.zeros(len(pos), H, D)
    q[..., :32] = 32768.0
    q[..., 32:36] = 1 - 2 * torch.randint(0, 2, (len(pos), H, 4), generator=g)
    return c, q.to(dtype).to(gpu), slots, pos


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.09, 1.0, 4.0, -4.0, 7.0, 1e7, -1e12, 2.0 ** 100, 2.0 ** 127])
def test_attn_far_scores(gpu, dtype, scale):
    """Scores of 2^22 that differ by multiples of 0.5, times scales from ordinary ones to the largest: the weights are
    those of the differences. A difference is exact and its product with the scale's factor is off by 2^-22 relative; a
    weight above fp32's smallest has an exponent of at most 160, so its exponent is off by less than 2^-14 and, in
    natural units, the score's part by less."""
    c, q, slots, pos = _exact_scores(gpu, dtype, 5)
    vals = [R.cache_values(c, s) for s in range(c.slots)]
    for chunk in (128, 384):
        got = _f64(_attend(q, c, slots, pos, scale, chunk))
        for r in range(len(pos)):
            out, mag, ds = R.attention(_f64(q[r]), *vals[int(slots[r])], int(pos[r]), scale)
            bound = R.attention_bound(out, mag, np.full_like(ds, 2.0 ** -14), dtype, int(pos[r]) + 1)
            assert (np.abs(got[r] - out) <= bound).all(), (chunk, r, float(np.nanmax(np.abs(got[r] - out) / bound)))


@pytest.mark.parametrize("scale", [0.0, 1e-40, -1e-38])
def test_attn_scores_past_the_scale(gpu, scale):
    """Raw scores of some 2^105 under scale 0, or under one so small that their products with it are below 2^-22: every
    weight is the same."""
    from m3x import ops
    dtype, D, cap = torch.bfloat16, 64, 160
    g = _g(2)
    k, v = torch.randn(cap, 1, D, generator=g) * 2.0 ** 60, torch.randn(cap, 1, D, generator=g)
    c = ops.Kv4Cache.empty(1, 1, cap, D, gpu)
    zero = torch.zeros(cap, dtype=torch.long, device=gpu)
    ops.kv4_append(k.to(dtype).to(gpu), v.to(dtype).to(gpu), c, zero, torch.arange(cap, dtype=torch.int32, device=gpu))
    q = (torch.randn(3, 2, D, generator=g) * 2.0 ** 42).to(dtype).to(gpu)
    if scale == -1e-38:
        q = q * 2.0 ** -8
    pos = torch.tensor([159, 40, 70])
    V = R.cache_values(c, 0)[1][0]
    for chunk in (128, 256):
        got = _f64(_attend(q, c, torch.zeros(3, dtype=torch.long), pos, scale, chunk))
        for r, p in enumerate(pos.tolist()):
            out, mag = V[:p + 1].mean(0), np.abs(V[:p + 1]).mean(0)
            bound = R.attention_bound(out, mag, 2.0 ** -14, dtype, p + 1)
            assert (np.abs(got[r] - out) <= bound).all(), (r, float((np.abs(got[r] - out) / bound).max()))


def test_attn_largest_values(gpu):
    """Values at the format's largest, 6 x 2^125, whose plain sum passes fp32: the weighted mean is never larger than
    they are, and keys of either sign cancel."""
    from m3x import ops
    dtype, D, KV, cap = torch.bfloat16, 128, 2, 512
    top = 6 * 2.0 ** 125
    c = ops.Kv4Cache.empty(1, KV, cap, D, gpu)
    g = _g(7)
    k = torch.randn(cap, KV, D, generator=g)
    v = torch.full((cap, KV, D), top)
    v[:, 1, ::2] *= 1 - 2 * (torch.arange(cap) % 2)[:, None].float()
    ops.kv4_append(k.to(dtype).to(gpu), v.to(dtype).to(gpu), c, torch.zeros(cap, dtype=torch.long, device=gpu),
                   torch.arange(cap, dtype=torch.int32, device=gpu))
    assert (c.vs == 252).all()
    K, V = R.cache_values(c, 0)
    pos = torch.tensor([1, 5, 300, 301, 302, 511])
    slots = torch.zeros(len(pos), dtype=torch.long)
    q = torch.randn(len(pos), 4, D, generator=g).to(dtype).to(gpu)
    for scale in (0.0, 0.09):
        for chunk in (128, 512):
            got = _f64(_attend(q, c, slots, pos, scale, chunk))
            for r, p in enumerate(pos.tolist()):
                out, mag, ds = R.attention(_f64(q[r]), K, V, p, scale)
                bound = R.attention_bound(out, mag, ds, dtype, p + 1)
                assert (np.abs(got[r] - out) <= bound).all(), (r, scale, chunk)
