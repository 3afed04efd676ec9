"""What the 4-bit entry points refuse, on the CPU: the binding's ValueErrors (raised before a library call) and the C
ABI's status codes (returned before a launch)."""
import ctypes

import pytest
import torch

P = ctypes.c_void_p(4096)  # never read: every call below is refused, or has no rows


def _cache(S=2, KV=2, cap=64, D=128):
    from m3x import ops
    return ops.Kv4Cache.empty(S, KV, cap, D, "cpu")


def _at(n):
    return torch.zeros(n, dtype=torch.long), torch.zeros(n, dtype=torch.int32)


def test_cache_shapes():
    from m3x import ops
    for D, cap in ((96, 64), (32, 64), (256, 64), (128, 40), (64, 0)):
        with pytest.raises(ValueError):
            _cache(cap=cap, D=D)
    c = _cache()
    assert (c.slots, c.kv_heads, c.cap, c.head_dim) == (2, 2, 64, 128)
    assert c.memory_bytes() == 2 * 2 * 64 * (128 + 8)
    with pytest.raises(ValueError):
        ops.Kv4Cache(c.k.to(torch.int8), c.ks, c.v, c.vs)
    with pytest.raises(ValueError):
        ops.Kv4Cache(c.k, c.ks[:1], c.v, c.vs)
    with pytest.raises(ValueError):
        ops.Kv4Cache(c.k, c.ks, c.v.transpose(3, 4), c.vs)
    with pytest.raises(ValueError):
        ops.Kv4Cache(c.k, c.ks, c.v, c.ks)


def test_rows_refused():
    from m3x import ops
    c, bf = _cache(), torch.bfloat16
    ok = torch.zeros(3, 2, 128, dtype=bf)
    for k, v in ((ok[:2], ok), (ok, ok[:, :1]), (ok.float(), ok.float()), (ok, ok.half()), (ok[..., :64], ok),
                 (ok, torch.zeros(3, 2, 256, dtype=bf)[..., ::2]), (torch.zeros(3, 2, 132, dtype=bf)[..., :128], ok)):
        with pytest.raises(ValueError):
            ops.kv4_append(k, v, c, *_at(3))
        with pytest.raises(ValueError):
            ops.kv4_read(c, *_at(3), k, v)
    slots, pos = _at(3)
    for s, p in ((slots.int(), pos), (slots, pos.long()), (slots[:2], pos), (slots[None], pos[None])):
        with pytest.raises(ValueError):
            ops.kv4_append(ok, ok, c, s, p)
    with pytest.raises(ValueError, match="device"):
        ops.kv4_append(ok, ok, c, slots, pos)
    with pytest.raises(ValueError, match="device"):
        ops.kv4_read(c, slots, pos, ok, ok)
    with pytest.raises(TypeError):
        ops.kv4_append(ok, ok, (c.k, c.v), slots, pos)


def test_attn_refused():
    from m3x import ops
    c = _cache()
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    at = _at(3)
    ws = torch.zeros(1 << 16)
    for args in ((q[:, :3], c, q[:, :3], *at, 1.0, 64, 128, ws), (q, c, q.half(), *at, 1.0, 64, 128, ws),
                 (q, c, q, *at, 1.0, 65, 128, ws), (q, c, q, *at, 1.0, 0, 128, ws), (q, c, q, *at, 1.0, 64, 100, ws),
                 (q, c, q, *at, 1.0, 64, 0, ws), (q[:, :0], c, q[:, :0], *at, 1.0, 64, 128, ws),
                 (q, c, q, *at, 1.0, 64, 128, ws[1:]), (q, c, q, *at, 1.0, 64, 128, ws[::2])):
        with pytest.raises(ValueError):
            ops.kv4_attn(*args)


def test_attn_workspace():
    from m3x import ops
    assert ops.kv4_attn_workspace(3, 4, 128, 1000, 1024) == 0
    assert ops.kv4_attn_workspace(3, 4, 128, 1025, 1024) == 3 * 4 * 2 * 130 * 4
    assert ops.kv4_attn_workspace(300, 64, 128, 1 << 20, 128) == 300 * 64 * 8192 * 130 * 4  # past 2^32
    assert ops.kv4_attn_workspace(0, 4, 128, 1000, 128) == 0
    for rows, ctx in ((1, 1), (1, 2048), (224, 2048), (2, 120001), (1600, 500)):
        chunk = ops.kv4_attn_chunk(rows, 16, 8, ctx)
        assert chunk >= 128 and chunk % 128 == 0


def test_weights_refused():
    from m3x import ops
    w = torch.zeros(20, 64, dtype=torch.bfloat16)
    for bad in (w[:, :40], w[None], w[:, ::2], w.to(torch.int8), torch.zeros(20, 68)[:, :64], w[:0]):
        with pytest.raises(ValueError):
            ops.pack_weight4(bad)
    with pytest.raises(ValueError, match="device"):
        ops.pack_weight4(w)
    p = ops.PackedWeight4(torch.zeros(2, 1, 64, 16, dtype=torch.uint8), torch.zeros(2, 1, 64, 4, dtype=torch.uint8), 20, 64)
    assert p.rows(16, 20).N == 4
    for a, b in ((8, 20), (16, 21), (16, 16)):
        with pytest.raises(ValueError):
            p.rows(a, b)
    with pytest.raises(ValueError):
        ops.PackedWeight4(p.codes, p.scales, 40, 64)
    with pytest.raises(ValueError):
        ops.PackedWeight4(p.codes, p.scales, 20, 60)
    x = torch.zeros(3, 64, dtype=torch.bfloat16)
    for xx, y in ((x[:, :32], None), (x.float(), None), (x[0], None), (torch.zeros(3, 68, dtype=x.dtype)[:, :64], None),
                  (x, torch.zeros(3, 21, dtype=x.dtype)), (x, torch.zeros(3, 20)), (x, torch.zeros(20, 3, dtype=x.dtype).t())):
        with pytest.raises(ValueError):
            ops.linear4(xx, p, y)
    with pytest.raises(TypeError):
        ops.linear4(x, w)
    with pytest.raises(ValueError):
        ops.linear4_act(x, p, None, ops.ACT_SWIGLU)
    with pytest.raises(ValueError):
        ops.linear4_act(x, p, p.rows(0, 16), ops.ACT_SWIGLU)
    with pytest.raises(ValueError):
        ops.linear4_act(x, p, p, ops.ACT_NONE)


def _kv4(kw):
    """The cache argument of a call whose keyword arguments may change its fields."""
    from m3x.ops import Kv4CacheArgs
    a = dict(k4=4096, ks4=4096, v4=4096, vs4=4096, nslots=1, kv_heads=2, head_dim=128, cap=64)
    a.update({n: kw.pop(n) for n in list(kw) if n in a})
    return Kv4CacheArgs(*a.values())


def _append(L, **kw):
    c = _kv4(kw)
    a = dict(k=P, sk_r=256, sk_h=128, v=P, sv_r=256, sv_h=128, slots=P, pos=P, rows=1, dtype=0)
    assert set(kw) <= set(a)
    return L.m3x_kv4_append(ctypes.addressof(c), *{**a, **kw}.values(), None)


def _attn(L, **kw):
    c = _kv4(kw)
    a = dict(q=P, sq_b=512, sq_h=128, out=P, so_b=512, so_h=128, slots=P, pos=P, scale=1.0, rows=1, heads=4, max_ctx=64,
             chunk=128, workspace=None, ws_bytes=0, dtype=0)
    assert set(kw) <= set(a)
    return L.m3x_kv4_attn(ctypes.addressof(c), *{**a, **kw}.values(), None)


def _read(L, **kw):
    c = _kv4(kw)
    a = dict(slots=P, pos=P, k=P, sk_r=256, sk_h=128, v=P, sv_r=256, sv_h=128, rows=1, dtype=0)
    assert set(kw) <= set(a)
    return L.m3x_kv4_read(ctypes.addressof(c), *{**a, **kw}.values(), None)


def _rope(L, **kw):
    c = _kv4(kw)
    a = dict(qkv=P, s_qkv=1024, q_out=P, s_qo_b=512, s_qo_h=128, slots=P, pos=P, cos=P, sin=P, s_cos=128, wq=P, wk=P,
             eps=1e-6, rows=1, heads=4)
    assert set(kw) <= set(a)
    return L.m3x_qk_norm_rope_kv4(ctypes.addressof(c), *{**a, **kw}.values(), None)


def _linear(L, **kw):
    a = dict(x=P, ldx=64, codes=P, scales=P, y=P, ldy=20, M=1, N=20, K=64, dtype=0)
    assert set(kw) <= set(a)
    return L.m3x_linear4(*{**a, **kw}.values(), None)


ODD = ctypes.c_void_p(4098)


@pytest.mark.parametrize("call,kw,status", [
    (_append, dict(rows=0), 0), (_append, dict(rows=-1), -1), (_append, dict(head_dim=96), -5), (_append, dict(cap=40), -1),
    (_append, dict(nslots=0), -1), (_append, dict(kv_heads=0), -1), (_append, dict(dtype=2), -5),
    (_append, dict(k=None), -2), (_append, dict(vs4=None), -2), (_append, dict(slots=None), -2), (_append, dict(sk_r=12), -1),
    (_append, dict(sv_h=4), -1), (_append, dict(v=ODD), -1), (_append, dict(k4=4098), -1),
    (_append, dict(cap=(1 << 30) + 32), -1), (_attn, dict(cap=(1 << 30) + 32), -1),
    (_append, dict(rows=2 ** 31 - 1, kv_heads=64), -1), (_append, dict(rows=1 << 25, kv_heads=8), -1),
    (_read, dict(rows=0), 0), (_read, dict(rows=-1), -1), (_read, dict(cap=40), -1), (_read, dict(k4=None), -2),
    (_read, dict(v=None), -2), (_read, dict(k=ODD), -1), (_read, dict(sv_r=3), -1), (_read, dict(dtype=2), -5),
    (_rope, dict(rows=0), 0), (_rope, dict(rows=-1), -1), (_rope, dict(heads=0), -1), (_rope, dict(head_dim=32), -5),
    (_rope, dict(cos=None), -2), (_rope, dict(wk=ODD), -1), (_rope, dict(s_cos=4), -1), (_rope, dict(ks4=4104), -1),
    (_attn, dict(rows=0), 0), (_attn, dict(rows=-1), -1), (_attn, dict(heads=0), -1), (_attn, dict(heads=5), -5),
    (_attn, dict(head_dim=256), -5), (_attn, dict(dtype=2), -5), (_attn, dict(max_ctx=65), -1), (_attn, dict(max_ctx=0), -1),
    (_attn, dict(chunk=64), -1), (_attn, dict(chunk=0), -1), (_attn, dict(out=None), -2), (_attn, dict(pos=None), -2),
    (_attn, dict(sq_h=100), -1), (_attn, dict(out=ODD), -1), (_attn, dict(cap=256, max_ctx=256), -2),
    (_attn, dict(cap=256, max_ctx=256, workspace=P, ws_bytes=100), -3),
    (_attn, dict(cap=256, max_ctx=256, workspace=ODD, ws_bytes=1 << 20), -1),
    (_attn, dict(heads=131072, kv_heads=2), -1), (_attn, dict(rows=(1 << 20) + 1), -1), (_attn, dict(cap=1 << 25, max_ctx=1 << 25, workspace=P, ws_bytes=1 << 40), -1),
    (_linear, dict(M=0), 0), (_linear, dict(M=-1), -1), (_linear, dict(N=0), -1), (_linear, dict(K=48), -1),
    (_linear, dict(ldx=60), -1), (_linear, dict(x=ODD), -1), (_linear, dict(codes=None), -2), (_linear, dict(y=None), -2),
    (_linear, dict(dtype=2), -5), (_linear, dict(M=2 ** 31 - 1), -1), (_linear, dict(N=1 << 27), -1)])
def test_status(call, kw, status):
    from m3x._lib import lib
    assert call(lib(), **kw) == status


def test_weight_sizes():
    from m3x._lib import lib
    L = lib()
    assert L.m3x_packed_weight4_bytes(20, 672, 0) == 2 * 6 * 1024 and L.m3x_packed_weight4_bytes(20, 672, 1) == 2 * 2 * 256
    assert L.m3x_packed_weight4_bytes(20, 48, 0) == -1 and L.m3x_packed_weight4_bytes(0, 32, 0) == -1
    assert L.m3x_kv4_append(None, P, 256, 128, P, 256, 128, P, P, 1, 0, None) == -2
    assert L.m3x_linear4_act(P, 64, P, P, None, None, P, 20, 1, 20, 64, 0, 0, None) == -2
    assert L.m3x_linear4_act(P, 64, P, P, P, P, P, 20, 1, 20, 64, -1, 0, None) == -5
    assert L.m3x_pack_weight4(P, 64, 20, 48, P, P, 0, None) == -1 and L.m3x_pack_weight4(P, 64, 20, 64, P, P, 3, None) == -5
