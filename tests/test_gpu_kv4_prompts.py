"""Attention over the 4-bit cache where one workgroup takes several candidate rows: prompts in one call large enough
for each such count, whose chains start anywhere, cross the workgroups' parts and follow one another through the same
sums."""
import numpy as np
import pytest
import torch

import fp4_reference as R

pytestmark = pytest.mark.gpu


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _f64(t):
    return t.detach().cpu().double().numpy()


def _candidates(rows, kv_heads, splits, G):
    """Candidate rows a workgroup takes: doubled while 4096 workgroups are left, at most 16 // G."""
    n = 1
    while n < 16 // G and rows * kv_heads * splits >= 4096 * n:
        n *= 2
    return min(n, 16 // G)


def _attention(q, K, V, pos, scale):
    """R.attention of one slot's rows at once: q [rows, heads, D], K, V [kv_heads, cap, D], pos [rows]."""
    n, H, D = q.shape
    KV = K.shape[0]
    G = H // KV
    out, mag, ds = np.zeros((n, H, D)), np.zeros((n, H, D)), np.zeros((n, H, 1))
    seen = np.arange(K.shape[1])[None] <= pos[:, None]
    for h in range(H):
        s = np.where(seen, q[:, h] @ K[h // G].T * scale, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[:, h], mag[:, h] = p @ V[h // G], p @ np.abs(V[h // G])
        size = np.where(seen, np.abs(q[:, h]) @ np.abs(K[h // G]).T, 0).max(-1, keepdims=True)
        ds[:, h] = (D + 4) * 2.0 ** -24 * (size * scale + 1)
    return out, mag, ds


@pytest.mark.parametrize("G,runs,chunk,want", [
    # G query heads a kv head; prompts (rows each, repeated); keys a split; candidates a workgroup
    (1, [200] * 8, 384, 4), (1, [200] * 8, 128, 16), (1, [33] * 41, 384, 4),
    (2, [200] * 8, 384, 4), (2, [199, 1, 1, 7] * 8, 128, 8), (2, [97] * 9, 384, 2),
    (3, [200] * 8, 384, 4), (3, [201, 2] * 8, 128, 5), (3, [130] * 6, 384, 2),
    (5, [200] * 8, 384, 3), (5, [3, 1, 4, 1, 5, 9, 2, 6] * 20, 384, 2), (8, [200] * 8, 128, 2), (16, [200] * 4, 128, 1)])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 64), (torch.bfloat16, 128)])
def test_prompts_share_workgroups(gpu, dtype, D, G, runs, chunk, want):
    """Every row against float64, and bit for bit as in a shuffled call, where hardly any two rows share a pass."""
    from m3x import ops
    KV, cap, S = 8, 288, 6
    rows = sum(runs) + 3
    splits = -(-cap // chunk)
    assert _candidates(rows, KV, splits, G) == want
    g = _g(G + len(runs))
    c = ops.Kv4Cache.empty(S, KV, cap, D, gpu)
    k, v = torch.randn(S * cap, KV, D, generator=g), torch.randn(S * cap, KV, D, generator=g) * 0.5
    ops.kv4_append(k.to(dtype).to(gpu), v.to(dtype).to(gpu), c, torch.arange(S, device=gpu).repeat_interleave(cap),
                   torch.arange(cap, dtype=torch.int32, device=gpu).repeat(S))
    slots, pos = [torch.tensor([2, S, 0])], [torch.tensor([17, 3, -1])]  # the first prompt starts at row 3
    for i, n in enumerate(runs):
        slots.append(torch.full((n,), i % S))
        pos.append(torch.arange(n) + int(torch.randint(0, cap - n + 1, (1,), generator=g)))
    slots, pos = torch.cat(slots), torch.cat(pos)
    q = torch.randn(rows, KV * G, D, generator=g).to(dtype).to(gpu)
    scale = D ** -0.5

    def attend(order):
        need = ops.kv4_attn_workspace(rows, KV * G, D, cap, chunk)
        ws = torch.full((need // 4,), float("nan"), device=gpu) if need else None
        out = torch.full_like(q, float("nan"))
        ops.kv4_attn(q[order], c, out, slots[order].to(gpu), pos[order].int().to(gpu), scale, cap, chunk, ws)
        return out

    got = attend(torch.arange(rows))
    order = torch.randperm(rows, generator=g)
    assert torch.equal(attend(order), got[order])
    assert not got[1:3].any()
    for s in range(S):
        at = [r for r in range(rows) if slots[r] == s and pos[r] >= 0]
        if not at:
            continue
        out, mag, ds = _attention(_f64(q[at]), *R.cache_values(c, s), pos[at].numpy(), scale)
        keys = (pos[at].numpy() + 1)[:, None, None]
        bound = R.attention_bound(out, mag, ds, dtype, keys)
        off = np.abs(_f64(got[at]) - out) / bound
        assert off.max() <= 1, (s, at[int(off.max((1, 2)).argmax())], float(off.max()))


@pytest.mark.parametrize("G", [1, 2, 20])
def test_positions_past_the_context(gpu, G):
    """A position at or past max_ctx, the largest int among them, sees the keys below max_ctx."""
    from m3x import ops
    KV, D, cap, ctx = 2, 128, 128, 70
    g = _g(3)
    c = ops.Kv4Cache.empty(2, KV, cap, D, gpu)
    k, v = (torch.randn(2 * cap, KV, D, generator=g).bfloat16().to(gpu) for _ in "kv")
    ops.kv4_append(k, v, c, torch.arange(2, device=gpu).repeat_interleave(cap),
                   torch.arange(cap, dtype=torch.int32, device=gpu).repeat(2))
    slots = torch.tensor([0, 0, 0, 0, 1, 1, 0], device=gpu)
    pos = torch.tensor([67, 68, 69, 70, 127, 2 ** 31 - 2, 2 ** 31 - 1], dtype=torch.int32, device=gpu)
    q = torch.randn(7, KV * G, D, generator=g).bfloat16().to(gpu)
    out, ref = torch.empty_like(q), torch.empty_like(q)
    ops.kv4_attn(q, c, out, slots, pos, 0.1, ctx, 128, None)
    ops.kv4_attn(q, c, ref, slots, pos.clamp(max=ctx - 1), 0.1, ctx, 128, None)
    assert torch.equal(out, ref) and torch.isfinite(out).all()
