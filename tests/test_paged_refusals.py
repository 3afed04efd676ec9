"""What the paged entry points refuse, on the CPU: the binding's errors (raised before a library call) and the C ABI's
status codes (returned before a launch); tiles, plans, frequencies and the page pool's bookkeeping."""
import ctypes
import math

import numpy as np
import pytest
import torch

P = ctypes.c_void_p(4096)  # never read: every call below is refused, or has no rows


def _cache(pages=5, KV=2, page=16, D=128, slots=2, width=4, dtype=torch.bfloat16):
    from m3x import ops
    return ops.PagedKv.empty(pages, KV, page, D, torch.zeros(slots, width, dtype=torch.int32), dtype)


def _at(n):
    return torch.zeros(n, dtype=torch.long), torch.zeros(n, dtype=torch.int32)


def test_cache_shapes():
    from m3x import ops
    c = _cache()
    assert (c.pages, c.page_size, c.kv_heads, c.head_dim, c.slots, c.cap) == (5, 16, 2, 128, 2, 64)
    assert c.memory_bytes() == 2 * 5 * 2 * 16 * 128 * 2
    for kw in (dict(D=96), dict(D=256), dict(page=8), dict(page=48), dict(page=512), dict(pages=0), dict(width=0),
               dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            _cache(**kw)
    t = c.table
    for k, v, table in ((c.k, c.v[:4], t), (c.k, c.v.half(), t), (c.k.transpose(1, 2), c.v.transpose(1, 2), t),
                        (c.k[..., :64], c.v[..., :64], t), (c.k, c.v, t.long()), (c.k, c.v, t[:, :2]), (c.k, c.v, t[0]),
                        (c.k[0], c.v[0], t), (c.k[::2], c.v[:3], t),
                        (c.k, c.v, torch.zeros(1, (1 << 26) + 1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.PagedKv(k, v, table)
    both = torch.zeros(5, 2, 2, 16, 128, dtype=torch.bfloat16)
    assert ops.PagedKv(both[:, 0], both[:, 1], t)._args.page_stride == 2 * 2 * 16 * 128


def test_rows_refused():
    from m3x import ops
    c, bf = _cache(), torch.bfloat16
    ok = torch.zeros(3, 2, 128, dtype=bf)
    for k, v in ((ok[:2], ok), (ok, ok[:, :1]), (ok.half(), ok.half()), (ok, ok.half()), (ok[..., :64], ok),
                 (ok, torch.zeros(3, 2, 256, dtype=bf)[..., ::2]), (torch.zeros(3, 2, 132, dtype=bf)[..., :128], ok)):
        with pytest.raises(ValueError):
            ops.paged_append(k, v, c, *_at(3))
        with pytest.raises(ValueError):
            ops.paged_read(c, *_at(3), k, v)
    slots, pos = _at(3)
    for s, p in ((slots.int(), pos), (slots, pos.long()), (slots[:2], pos), (slots[None], pos[None])):
        with pytest.raises(ValueError):
            ops.paged_append(ok, ok, c, s, p)
    with pytest.raises(ValueError, match="device"):
        ops.paged_append(ok, ok, c, slots, pos)
    with pytest.raises(ValueError, match="device"):
        ops.paged_read(c, slots, pos, ok, ok)
    with pytest.raises(TypeError):
        ops.paged_append(ok, ok, (c.k, c.v), slots, pos)


def test_qk_norm_rope_refused():
    from m3x import ops
    c, bf = _cache(D=64), torch.bfloat16
    rot = ops.Rotary([1.0] * 32, device="cpu")
    qkv, q, w = torch.zeros(3, 8 * 64, dtype=bf), torch.zeros(3, 4, 64, dtype=bf), torch.ones(64, dtype=bf)
    for a in ((qkv[:, :-64], q, rot, w, w, 4), (qkv, q[:, :3], rot, w, w, 4), (qkv.half(), q, rot, w, w, 4),
              (qkv, q.half(), rot, w, w, 4), (qkv, q, rot, w, None, 4), (qkv, q, rot, None, w, 4),
              (qkv, q, rot, w[:32], w, 4), (qkv, q, rot, w.float(), w, 4), (qkv, q, None, w, w, 4),
              (qkv, q, ops.Rotary([1.0] * 40, device="cpu"), w, w, 4), (qkv, q, rot, w, w, 0),
              (torch.zeros(3, 8 * 64 + 4, dtype=bf)[:, :512], q, rot, w, w, 4)):
        with pytest.raises(ValueError):
            ops.qk_norm_rope_paged(a[0], a[1], c, *_at(3), a[2], a[3], a[4], 1e-6, a[5])
    with pytest.raises(ValueError, match="device"):
        ops.qk_norm_rope_paged(qkv, q, c, *_at(3), rot, w, w, 1e-6, 4)


def test_attn_refused():
    from m3x import ops
    c = _cache()
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    at = _at(3)
    plan = ops.PagedPlan([(0, 3, 0)], 4, 2, 128, 64, device="cpu")
    for args in ((q[:, :3], c, q[:, :3], *at, 1.0, plan), (q, c, q.half(), *at, 1.0, plan),
                 (q.half(), c, q.half(), *at, 1.0, plan), (q[:2], c, q[:2], *_at(2), 1.0, plan),
                 (q, c, q, *at, float("nan"), plan), (q, c, q, *at, 2.0 ** 127, plan),
                 (q, _cache(KV=1), q, *at, 1.0, plan), (q, _cache(D=64), q, *at, 1.0, plan)):
        with pytest.raises(ValueError):
            ops.paged_attn(*args)
    with pytest.raises(ValueError, match="device"):
        ops.paged_attn(q, c, q, *at, 1.0, plan)
    with pytest.raises(TypeError):
        ops.paged_attn(q, c, q, *at, 1.0, None)
    split = ops.PagedPlan([(0, 3, 0)], 4, 2, 128, 1 << 16, device="cpu")
    assert split.workspace > 0
    ws = torch.zeros(split.workspace + 16, dtype=torch.uint8)
    for w in (None, ws[:split.workspace - 1], ws[1:], torch.zeros(2 * split.workspace, dtype=torch.uint8)[::2]):
        with pytest.raises(ValueError):
            ops.paged_attn(q, c, q, *at, 1.0, split, w)


def test_plan_refused():
    from m3x import ops
    for a in (([(0, 1, 0)], 3, 2, 128, 64), ([(0, 1, 0)], 0, 1, 128, 64), ([(-1, 2, 0)], 4, 2, 128, 64),
              ([(0, -1, 0)], 4, 2, 128, 64), ([(0, 1 << 31, 0)], 4, 2, 128, 64), ([(4, 2, 0), (0, 5, 0)], 4, 2, 128, 64),
              ([(1, 1, 0), (1, 1, 0)], 4, 2, 128, 64)):
        with pytest.raises(ValueError):
            ops.PagedPlan(*a, device="cpu")
    for kw in (dict(window=-1), dict(sinks=-1), dict(window=1 << 31)):
        with pytest.raises(ValueError):
            ops.PagedPlan([(0, 1, 0)], 4, 2, 128, 64, device="cpu", **kw)
    with pytest.raises(ValueError):
        ops.PagedPlan.reserve(0, 4, 2, 128, 64, device="cpu")
    assert ops.PagedPlan([], 4, 2, 128, 64, device="cpu").launches == []


@pytest.mark.parametrize("H,KV", [(16, 8), (8, 8), (32, 4), (71, 1), (300, 2)])
def test_tiles(H, KV):
    """Every row of the runs in one tile, tiles within a run and within the columns, the longest contexts first."""
    from m3x import ops
    G = H // KV
    rng = np.random.default_rng(H)
    for _ in range(20):
        runs, at = [], 0
        for _ in range(rng.integers(1, 30)):
            n = int(rng.choice([0, 1, 1, 1, 2, 5, 16, 17, 33, 64, 65, 129, 400]))
            runs.append((at, n, int(rng.integers(-1, 3000))))
            at += n + int(rng.integers(0, 2))
        for narrow, wide in (ops.paged_tiles(runs, H, KV), ops.paged_tiles(runs, H, KV, cut=32)):
            seen = []
            ends = []
            for t, most in ((narrow, 32), (wide, 128)):
                for a, n in t:
                    if n == 0:
                        continue
                    assert n == 1 or n * G <= most
                    r = [x for x in runs if x[0] <= a and a + n <= x[0] + x[1]]
                    assert len(r) == 1
                    seen += range(a, a + n)
                    if most == 128:
                        ends.append(r[0][2] + a + n - r[0][0])
            assert sorted(seen) == [r for a, n, _ in runs for r in range(a, a + n)]
            assert ends == sorted(ends, reverse=True)


@pytest.mark.parametrize("D", [64, 128])
def test_plans(D):
    """Every row of a plan's runs is in one tile of one launch, whatever its layout, window and largest context."""
    from m3x import ops
    rng = np.random.default_rng(D)
    for H, KV in ((16, 8), (8, 8), (32, 4), (24, 1), (71, 1), (300, 2)):
        for _ in range(60):
            runs, at = [], int(rng.integers(0, 3))
            sizes = rng.choice([1, 1, 1, 2, 5, 6, 17, 33, 65, 300], int(rng.integers(1, 50))) if rng.integers(3) else [1] * 40
            for n in sizes:
                runs.append((at, int(n), int(rng.integers(-n - 1, rng.choice([2, 500, 4000])))))
                at += n + int(rng.integers(0, 2))
            window = int(rng.choice([0, 0, 1, 100, 5000]))
            plan = ops.PagedPlan([runs[i] for i in rng.permutation(len(runs))], H, KV, D, int(rng.choice([0, 50, 4000])),
                                 window=window, sinks=int(rng.choice([0, 4, 900])) if window else 0, device="cpu")
            seen = []
            for tiles, n, tile_rows, cols, splits in plan.launches:
                assert cols in ((16, 32, 48, 128) if D == 64 else (16, 32, 128)) and 1 <= splits <= 256 and n <= 65535
                for a, x in [(r, 1) for r in range(n)] if tiles is None else tiles.tolist():
                    m, s = x & 0xFFFF, x >> 16
                    assert 1 <= m <= tile_rows and 0 <= s <= splits and any(f <= a and a + m <= f + k for f, k, _ in runs)
                    seen += range(a, a + m)
            assert sorted(seen) == [r for f, k, _ in runs for r in range(f, f + k)] and plan.rows == runs[-1][0] + runs[-1][1]


def test_splits():
    """At least one workgroup, none with fewer keys than the kernels' least, within the ABI's limit."""
    from m3x import ops
    for blocks in (0, 1, 8, 100, 256, 257, 640, 641, 5000):
        for keys in (0, 1, 100, 2048, 120000, 1 << 30):
            for cols in (16, 32, 128):
                s = ops.paged_attn_splits(blocks, keys, cols, keys // 2, blocks * cols)
                assert 1 <= s <= 256 and (s == 1 or s * 128 <= keys)
    assert ops.paged_attn_splits(30, 3000, 48, 1) <= 11 and ops.paged_attn_splits(1, 383, 16) == ops.paged_attn_splits(1, 767, 32) == 1 and ops.paged_attn_splits(160, 3000, 48, 1500) == 3
    assert ops.paged_attn_splits(1792, 2048, 16) == 1 and ops.paged_attn_splits(8, 2048, 16) == 8


def test_rotary():
    """Frequencies as exact binary fractions of a turn; the scalings' formulas."""
    from fractions import Fraction
    from m3x import ops
    pi = Fraction(314159265358979323846264338327950288419716939937510582097494459, 10 ** 62)
    f = [1.0, 0.1, 1e-6, 3.0, 7.5, 2.0 ** -40, 0.0, -0.25]
    for x, w in zip(f, ops.Rotary(f, device="cpu").freq.tolist()):
        want = Fraction(x) / (2 * pi) * 2 ** 64
        off = (w - want) % 2 ** 64
        assert min(off, 2 ** 64 - off) <= Fraction(1, 2) + Fraction(1, 1 << 40)
    for bad in ([1.0] * 7, [1.0] * 9, [1.0] * 72, [float("inf")] * 8, torch.ones(2, 8)):
        with pytest.raises(ValueError):
            ops.Rotary(bad, device="cpu")
    with pytest.raises(ValueError):
        ops.Rotary([1.0] * 8, factor=float("inf"), device="cpu")
    plain, one = ops.rotary_freqs(64, 1e4)
    assert one == 1 and torch.allclose(plain, torch.tensor([1e4 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64))
    assert torch.equal(ops.rotary_freqs(64, 1e4, "linear", by=4.0)[0], plain / 4)
    base = ops.rotary_freqs(64, 1e4, "base", by=4.0)[0]
    assert base[0] == 1 and abs(base[-1] / (plain[-1] / 4) - 1) < 1e-12
    parts, factor = ops.rotary_freqs(64, 1e4, "parts", by=4.0, trained=4096)
    assert factor == pytest.approx(0.1 * math.log(4) + 1) and parts[0] == plain[0] and parts[-1] == plain[-1] / 4
    assert ((parts <= plain) & (parts >= plain / 4)).all()
    for kw in (dict(kind="other"), dict(kind="parts", by=2.0), dict(kind="linear", by=0.5),
               dict(kind="parts", by=2.0, trained=10, fast=1.0, slow=2.0)):
        with pytest.raises(ValueError):
            ops.rotary_freqs(64, 1e4, **kw)
    for dim, theta in ((3, 1e4), (2, 1e4), (64, 0.0)):
        with pytest.raises(ValueError):
            ops.rotary_freqs(dim, theta)


def _args(**kw):
    from m3x.ops import PagedKvArgs
    a = dict(k=4096, v=4096, table=4096, page_stride=2 * 16 * 128, pages=4, page_size=16, kv_heads=2, head_dim=128, slots=3,
             width=4, dtype=0)
    a.update(kw)
    return ctypes.byref(PagedKvArgs(*(a[n] for n, _ in PagedKvArgs._fields_)))


def test_status_codes():
    """The C ABI: statuses instead of launches."""
    from m3x._lib import lib
    from m3x.ops import RotaryArgs
    L = lib()
    rot = lambda **kw: ctypes.byref(RotaryArgs(*({**dict(freq=4096, dim=128, i=0, f=1.0), **kw}).values()))  # noqa: E731
    append = lambda c, k=P, n=1, s=128: L.m3x_paged_append(c, k, s, s, P, s, s, P, P, n, None)  # noqa: E731
    assert append(_args(), n=0) == 0 and append(None) == -2 and append(_args(), k=None) == -2
    assert append(_args(), n=-1) == -1 and append(_args(), s=4) == -1 and append(_args(), k=ctypes.c_void_p(4100)) == -1
    assert append(_args(), n=2 ** 31 - 1) == -1  # more threads than a launch holds
    for kw, st in ((dict(head_dim=96), -5), (dict(page_size=24), -5), (dict(page_size=512), -5), (dict(dtype=2), -5),
                   (dict(pages=0), -1), (dict(width=0), -1), (dict(width=(1 << 26) + 1), -1), (dict(k=0), -2),
                   (dict(table=0), -2), (dict(page_stride=2 * 16 * 128 - 8), -1), (dict(page_stride=2 * 16 * 128 + 4), -1),
                   (dict(k=4104), -1), (dict(table=4098), -1), (dict(kv_heads=70000, page_stride=1 << 40), -1)):
        assert append(_args(**kw)) == st, kw
    read = lambda c, n=1: L.m3x_paged_read(c, P, P, P, 128, 128, P, 128, 128, n, None)  # noqa: E731
    assert read(_args(), 0) == 0 and read(None) == -2 and read(_args(), -1) == -1 and read(_args(head_dim=32)) == -5
    far = ctypes.c_void_p(1 << 30)
    qkn = lambda r=None, q=far, qkv=P, wq=P, wk=P, n=1, h=4: L.m3x_qk_norm_rope_paged(  # noqa: E731
        _args(), qkv, 1024, q, 512, 128, P, P, r or rot(), wq, wk, 1e-6, n, h, None)
    assert qkn(n=0) == 0 and qkn(qkv=None) == -2 and qkn(wq=None) == -2 and qkn(wk=None) == -2 and qkn(h=0) == -1
    assert qkn(rot(dim=8)) == -1 and qkn(rot(dim=144)) == -1 and qkn(rot(dim=72)) == -1 and qkn(rot(freq=0)) == -2
    assert qkn(q=P) == -1 and qkn(q=ctypes.c_void_p(4096 + 512)) == -1  # over the rows themselves
    assert L.m3x_qk_norm_rope_paged(_args(), P, 1024, far, 512, 128, P, P, None, P, P, 1e-6, 1, 4, None) == -2

    def attn(c=None, q=P, tiles=None, n=3, tr=1, cols=16, scale=1.0, rows=3, heads=4, window=0, sinks=0, splits=1, ws=None,
             wb=0, arrived=None, s=128):
        return L.m3x_paged_attn(c or _args(), q, 4 * s, s, P, 4 * s, s, P, P, tiles, n, tr, cols, scale, rows, heads, window,
                                sinks, splits, ws, wb, arrived, None)
    assert attn(rows=0) == 0 and attn(n=0) == 0 and attn(q=None) == -2 and attn(heads=3) == -5 and attn(heads=0) == -1
    for kw in (dict(rows=-1), dict(n=-1), dict(scale=float("nan")), dict(scale=2.0 ** 127), dict(window=-1), dict(sinks=-1),
               dict(splits=0), dict(splits=257), dict(s=4), dict(n=4), dict(tr=2), dict(cols=64), dict(cols=48), dict(heads=1 << 20),
               dict(tiles=ctypes.c_void_p(4098)), dict(tiles=P, n=65536, rows=1 << 20),
               dict(tiles=P, tr=1 << 15, cols=128, rows=1 << 20), dict(q=ctypes.c_void_p(4104))):
        assert attn(**kw) == -1, kw
    assert attn(splits=2) == -2 and attn(splits=2, ws=P, wb=1 << 30) == -2 and attn(splits=2, ws=P, arrived=P, wb=10) == -3
    assert attn(splits=2, ws=ctypes.c_void_p(4100), arrived=P, wb=1 << 30) == -1
    need = L.m3x_paged_attn_workspace(3, 2, 4, 1, 16, 128, 2)
    assert need == 3 * 2 * 16 * 2 * 130 * 4 and L.m3x_paged_attn_workspace(3, 2, 4, 1, 16, 128, 1) == 0
    assert L.m3x_paged_attn_workspace(65535, 8, 64, 16, 128, 128, 64) == 65535 * 8 * 128 * 64 * 130 * 4  # past 2^32


# ---------------------------------------------------------------- the page pool
def _pool(pages=10, page=16, slots=4, cap=100):
    from m3x.pages import PagePool
    return PagePool(pages, page, slots, cap, "cpu")


def _sound(p):
    """Each page is free or named as often as its count says, and never both."""
    named = p._host[p._host >= 0]
    assert np.array_equal(np.bincount(named, minlength=p.pages), p._uses)
    assert sorted(p._free) == [i for i in range(p.pages) if p._uses[i] == 0]


def test_pool_grow_and_release():
    p = _pool()
    assert p.width == 7 and p.free_pages == 10
    p.grow([(0, 1), (1, 33), (2, 0)])
    assert [p.held(s) for s in range(4)] == [1, 3, 0, 0] and p.has(1, 33) and p.has(1, 48) and not p.has(1, 49)
    p.grow([(0, 16), (1, 48)])
    assert p.free_pages == 6
    with pytest.raises(RuntimeError, match="exhausted"):
        p.grow([(0, 100), (1, 100)])
    assert p.free_pages == 6 and p.held(0) == 1  # nothing taken
    with pytest.raises(ValueError):
        p.grow([(0, 113)])
    _sound(p)
    p.release(1)
    assert p.held(1) == 0 and p.free_pages == 9
    _sound(p)
    p.grow([(3, 20), (3, 40), (3, 5)])  # the same slot again
    assert p.held(3) == 3 and p.free_pages == 6
    _sound(p)
    for bad in ((0, 16, 4, 100), (4, 16, 0, 100), (4, 16, 4, 0)):
        with pytest.raises(ValueError):
            _pool(*bad)


def test_pool_trim():
    p = _pool()
    p.grow([(0, 100)])
    p.trim(0, 15)
    assert p.held(0) == 7
    p.trim(0, 50, keep=4)  # page 0 holds the first 4 and stays, pages 1 and 2 go
    assert p.held(0) == 5 and p._host[0, 0] >= 0 and (p._host[0, 1:3] == -1).all() and p._host[0, 3] >= 0
    p.trim(0, 50, keep=4)
    p.trim(0, 20, keep=4)
    assert p.held(0) == 5 and not p.has(0, 20) and p.has(0, 16)
    p.trim(0, 1000)
    assert p.free_pages == 9 or p.held(0) <= 1
    _sound(p)
    p.release(0)
    assert p.free_pages == 10
    _sound(p)


def test_pool_share():
    p = _pool()
    p.grow([(0, 40)])
    copy = p.share(1, 0, 40)
    assert copy == (p._host[0, 2], p._host[1, 2]) and copy[0] != copy[1]
    assert (p._host[1, :2] == p._host[0, :2]).all() and p.free_pages == 6
    assert p.share(2, 0, 32) is None and p.free_pages == 6
    with pytest.raises(ValueError):
        p.share(2, 0, 16)
    with pytest.raises(ValueError):
        p.share(3, 0, 60)
    _sound(p)
    p.release(0)
    assert p.free_pages == 7  # the partly filled page; the others are still named
    p.grow([(1, 100), (2, 80)])
    with pytest.raises(RuntimeError, match="exhausted"):
        p.share(3, 1, 20)
    assert p.held(3) == 0
    _sound(p)
    for s in (1, 2):
        p.release(s)
    assert p.free_pages == 10
    _sound(p)


def test_pool_outside():
    """Slots and lengths outside the table are refused, with nothing changed."""
    p = _pool()
    p.grow([(0, 112)])
    for s in (-1, 4):
        for call in (lambda: p.held(s), lambda: p.has(s, 1), lambda: p.grow([(1, 5), (s, 5)]), lambda: p.trim(s, 5),
                     lambda: p.release(s), lambda: p.share(s, 0, 5), lambda: p.share(1, s, 0)):
            with pytest.raises(IndexError):
                call()
    assert p.has(0, 112) and not p.has(0, 113) and p.has(1, 0) and p.has(1, -3)
    with pytest.raises(ValueError):
        p.share(1, 0, 113)
    assert p.held(1) == 0 and p.free_pages == 3
    _sound(p)


def test_pool_random():
    """A long run of grows, trims, shares and releases keeps the counts."""
    rng = np.random.default_rng(1)
    p = _pool(pages=40, slots=8, cap=200)
    length = [0] * 8
    for _ in range(2000):
        s, t = (int(x) for x in rng.choice(8, 2, replace=False))
        op = rng.integers(5)
        try:
            if op == 0:
                p.release(s)
                length[s] = 0
            elif op == 1:
                p.release(s)
                length[s] = 0
                n = int(rng.integers(0, length[t] + 1))
                if p.has(t, n):
                    p.share(s, t, n)
                    length[s] = n
            elif op == 2:
                p.trim(s, max(0, length[s] - 30), int(rng.integers(0, 20)))
            else:
                n = min(200, length[s] + int(rng.integers(1, 40)))
                p.grow([(s, n)])
                length[s] = n
        except RuntimeError:
            pass
        _sound(p)


@pytest.mark.parametrize("few", [None, True, False])
def test_reserved(few, monkeypatch):
    """A reserved plan holds the tiles of any layout of its rows: each row once, within a run and within its launch."""
    from m3x import ops
    if few is not None:
        monkeypatch.setattr(ops.PagedPlan, "_few", lambda *a: few)
    rng = np.random.default_rng(2)
    for H, KV, rows in ((16, 8, 1), (16, 8, 2), (16, 8, 64), (16, 8, 300), (32, 4, 40), (32, 2, 50), (64, 1, 90), (24, 2, 33),
                        (8, 8, 64), (40, 1, 7), (150, 1, 9)):
        plan = ops.PagedPlan.reserve(rows, H, KV, 64, 1500, device="cpu")
        assert len(plan.launches) <= 3
        for i in range(200):
            runs, at = [], 0
            while at < rows:
                n = min(rows - at, (2, 3, 17, 33)[i] if i < 4 else int(rng.choice([1, 1, 2, 3, 5, 9, 17, 33, 100])))
                runs.append((at, n, int(rng.integers(-50, 3000))))
                at += n
            seen = []
            for tiles, (_, room, tile_rows, _, splits) in zip(plan.tiles(runs), plan.launches):
                assert tiles.shape == (room, 2)
                for a, x in tiles.tolist():
                    n, s = x & 0xFFFF, x >> 16
                    assert n <= tile_rows and s <= splits
                    assert n == 0 or any(f <= a and a + n <= f + m for f, m, _ in runs)
                    seen += range(a, a + n)
            assert sorted(seen) == list(range(rows))
    one = ops.PagedPlan.reserve(40, 16, 8, 128, 2048, device="cpu", single=True)
    assert len(one.launches) == 1 and one.launches[0][1:4] == (40, 1, 16) and one.launches[0][4] > 1
    even, uneven = (one.tiles([(r, 1, p) for r, p in enumerate(at)])[0] for at in ([2000] * 40, range(100, 2060, 49)))
    assert even[:, 0].tolist() == list(range(40)) and uneven[:, 0].tolist() == list(range(39, -1, -1))
    with pytest.raises(ValueError):
        one.tiles([(0, 2, 5)])
    with pytest.raises(ValueError):
        plan.tiles([(r, 1, 0) for r in range(30)])
    with pytest.raises(ValueError):
        plan.tiles([(8, 2, 0)])
    with pytest.raises(ValueError):
        plan.tiles([(0, 2, 0), (1, 1, 0)])
