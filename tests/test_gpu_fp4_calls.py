"""The 4-bit entry points as callers combine them: calls in flight on two streams, two captured graphs over one
workspace, launches past 65535 workgroups and rows, rows at one place, repeated rows, a row's bits under other rows."""
import numpy as np
import pytest
import torch

import fp4_reference as R

pytestmark = pytest.mark.gpu


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _f64(t):
    return t.detach().cpu().double().numpy()


def _filled(gpu, S, KV, cap, D, dtype, seed):
    from m3x import ops
    c = ops.Kv4Cache.empty(S, KV, cap, D, gpu)
    k, v = (torch.randn(S * cap, KV, D, generator=_g(seed + i)).to(dtype).to(gpu) for i in range(2))
    ops.kv4_append(k, v, c, torch.arange(S, device=gpu).repeat_interleave(cap),
                   torch.arange(cap, dtype=torch.int32, device=gpu).repeat(S))
    return c


def _attention(gpu, c, rows, H, seed, dtype, chunk):
    """A call's arguments: queries, output, places and workspace of its own."""
    from m3x import ops
    g = _g(seed)
    q = torch.randn(rows, H, c.head_dim, generator=g).to(dtype).to(gpu)
    slots = torch.randint(0, c.slots, (rows,), generator=g).to(gpu)
    pos = torch.randint(0, c.cap, (rows,), generator=g).int().to(gpu)
    ws = torch.empty(ops.kv4_attn_workspace(rows, H, c.head_dim, c.cap, chunk), dtype=torch.uint8, device=gpu)
    out = torch.empty_like(q)
    return lambda: ops.kv4_attn(q, c, out, slots, pos, 0.1, c.cap, chunk, ws), out, ws


def test_two_streams(gpu):
    """Two attention calls and two products in flight at once, each on its own stream with its own workspace."""
    from m3x import ops
    c = _filled(gpu, 3, 4, 2048, 128, torch.bfloat16, 1)
    a, b = (_attention(gpu, c, 24, 8, s, torch.bfloat16, 256) for s in (1, 2))
    w = ops.pack_weight4(torch.randn(2048, 1024, generator=_g(3)).bfloat16().to(gpu))
    x = [torch.randn(9, 1024, generator=_g(4 + i)).bfloat16().to(gpu) for i in range(2)]
    want = []
    for (run, out, _), xi in zip((a, b), x):
        run()
        want.append((out.clone(), ops.linear4(xi, w)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(8):
        ys = []
        for (run, out, ws), xi, s in zip((a, b), x, streams):
            with torch.cuda.stream(s):
                out.zero_()
                ws.fill_(255)
                run()
                ys.append(ops.linear4(xi, w))
        torch.cuda.synchronize()
        for (_, out, _), y, (o, yo) in zip((a, b), ys, want):
            assert torch.equal(out, o) and torch.equal(y, yo)


def test_two_graphs_one_workspace(gpu):
    """Graphs of different shapes that share a workspace, replayed in turn with eager calls on it between."""
    from m3x import ops
    c = _filled(gpu, 3, 2, 1024, 64, torch.float16, 5)
    H, chunk = 8, 128
    ws = torch.empty(ops.kv4_attn_workspace(20, H, 64, c.cap, chunk), dtype=torch.uint8, device=gpu)
    calls = []
    for rows, seed in ((20, 1), (3, 2)):
        g = _g(seed)
        q = torch.randn(rows, H, 64, generator=g).half().to(gpu)
        slots, pos = torch.randint(0, 3, (rows,), generator=g).to(gpu), torch.zeros(rows, dtype=torch.int32, device=gpu)
        out = torch.empty_like(q)
        run = lambda q=q, out=out, slots=slots, pos=pos: ops.kv4_attn(  # noqa: E731
            q, c, out, slots, pos, 0.2, c.cap, chunk, ws)
        run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
        calls.append((run, graph, out, pos, g))
    for i in range(4):
        for run, graph, out, pos, g in calls:
            pos.copy_(torch.randint(-1, c.cap, pos.shape, generator=g).int())
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone()
            out.fill_(float("nan"))
            run()
            torch.cuda.synchronize()
            assert torch.equal(got, out), i


@pytest.mark.parametrize("D", [64, 128])
def test_large_counts(gpu, D):
    """262144 rows of one kv head written, read back and, 100000 of them, attended over short contexts."""
    from m3x import ops
    S, cap, rows = 8, 32768, 262144
    g = _g(D)
    c = ops.Kv4Cache.empty(S, 1, cap, D, gpu)
    k, v = (torch.randn(rows, 1, D, generator=g).bfloat16() for _ in "kv")
    place = torch.randperm(rows, generator=g)
    slots, pos = (place // cap).to(gpu), (place % cap).int().to(gpu)
    ops.kv4_append(k.to(gpu), v.to(gpu), c, slots, pos)
    ko, vo = torch.empty_like(k, device=gpu), torch.empty_like(k, device=gpu)
    ops.kv4_read(c, slots, pos, ko, vo)
    for a, b in ((k, ko), (v, vo)):
        for at in (slice(0, 3000), slice(rows - 3000, rows)):
            assert np.array_equal(_f64(b[at]), R.quantise(_f64(a[at]), 252)[0])
    n = 100000
    q = torch.randn(n, 2, D, generator=g).bfloat16().to(gpu)
    s, p = torch.randint(0, S, (n,), generator=g), torch.randint(-1, 40, (n,), generator=g)
    out = torch.full_like(q, float("nan"))
    ops.kv4_attn(q, c, out, s.to(gpu), p.int().to(gpu), 0.1, 64, 512, None)
    assert not out[(p < 0).to(gpu)].any() and torch.isfinite(out).all()
    vals = {}
    for r in list(range(0, 60)) + list(range(n - 60, n)):
        if p[r] < 0:
            continue
        i = int(s[r])
        if i not in vals:  # the first 64 positions are enough
            at = torch.full((64,), i, device=gpu), torch.arange(64, dtype=torch.int32, device=gpu)
            kk, vv = (torch.empty(64, 1, D, dtype=torch.bfloat16, device=gpu) for _ in "kv")
            ops.kv4_read(c, *at, kk, vv)
            vals[i] = [_f64(t).transpose(1, 0, 2) for t in (kk, vv)]
        o, mag, ds = R.attention(_f64(q[r]), *vals[i], int(p[r]), 0.1)
        assert (np.abs(_f64(out[r]) - o) <= R.attention_bound(o, mag, ds, torch.bfloat16, int(p[r]) + 1)).all(), r


def test_many_rows_product(gpu):
    """70001 rows through a narrow layer: K products summed in fp32, one half step of the type."""
    from m3x import ops
    M, N, K = 70001, 40, 64
    x = torch.randn(M, K, generator=_g(1)).bfloat16().to(gpu)
    p = ops.pack_weight4(torch.randn(N, K, generator=_g(2)).bfloat16().to(gpu))
    w = torch.from_numpy(R.weight_values(p.codes, p.scales, N, K))
    y = x.cpu().double() @ w.T
    off = (K + 8) * 2.0 ** -24 * (x.cpu().double().abs() @ w.abs().T)
    got = ops.linear4(x, p).cpu().double()
    assert ((got - y).abs() <= off + 2.0 ** -8 * (y.abs() + off)).all()


def test_rows_at_one_place(gpu):
    """Rows of one call at one place, and rows of a repeated (stride 0) source: nothing else of the cache changes, and
    equal rows leave their own numbers."""
    from m3x import ops
    KV, D, cap = 2, 128, 64
    c = _filled(gpu, 2, KV, cap, D, torch.bfloat16, 9)
    before = [t.clone() for t in (c.k, c.ks, c.v, c.vs)]
    k = torch.randn(1, KV, D, generator=_g(1)).bfloat16().to(gpu)
    slots = torch.ones(100, dtype=torch.long, device=gpu)
    pos = torch.full((100,), 17, dtype=torch.int32, device=gpu)
    ops.kv4_append(k.expand(100, KV, D), k.expand(100, KV, D), c, slots, pos)
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    ops.kv4_read(c, slots[:1], pos[:1], ko, vo)
    want = R.quantise(_f64(k), 252)[0]
    assert np.array_equal(_f64(ko), want) and np.array_equal(_f64(vo), want)
    k, v = (torch.randn(100, KV, D, device=gpu).bfloat16() for _ in "kv")
    ops.kv4_append(k, v, c, slots, pos)
    for now, old in zip((c.k, c.ks), before[:2]):
        now[1, :, 17] = old[1, :, 17]
    c.v[1, :, 4, :, 1], c.vs[1, :, 4, :, 1] = before[2][1, :, 4, :, 1], before[3][1, :, 4, :, 1]
    assert all(torch.equal(a, b) for a, b in zip((c.k, c.ks, c.v, c.vs), before))


def _product(x, w):
    """(sums, bound of K products summed in fp32 in any order), float64."""
    return x @ w.T, (x.shape[1] + 8) * 2.0 ** -24 * (np.abs(x) @ np.abs(w).T)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(4, 4200, 160), (7, 4200, 160), (9, 8300, 1056), (14, 8300, 1056), (3, 33000, 96),
                                   (40, 6000, 1056), (200, 3000, 160), (530, 2000, 1056), (130, 3700, 1184),
                                   (224, 4800, 8192)])
def test_linear4_groups(gpu, dtype, M, N, K):
    """Every grouping of tiles and rows a product is dealt out in, with rows, columns and inputs that end inside one,
    and numbers beside x that are not finite."""
    from m3x import ops
    g = _g(M + N + K)
    wide = torch.full((M + 1, K + 16), float("nan"), dtype=dtype)
    wide[:M, 8:8 + K] = torch.randn(M, K, generator=g).to(dtype)
    x = wide.to(gpu)[:M, 8:8 + K]
    p = ops.pack_weight4((torch.randn(N, K, generator=g) * K ** -0.5).to(dtype).to(gpu))
    y, off = _product(_f64(x), R.weight_values(p.codes, p.scales, N, K))
    h, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0
    big = torch.full((M + 1, N + 3), 3.0, dtype=dtype, device=gpu)
    for out in (None, big[:M, 1:1 + N]):
        got = _f64(ops.linear4(x, p, out))
        assert (np.abs(got - y) <= off + h * (np.abs(y) + off) + tiny).all()
    assert (big[M] == 3).all() and (big[:, :1] == 3).all() and (big[:, 1 + N:] == 3).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(4, 4200, 160), (7, 4200, 160), (40, 3000, 160), (130, 3700, 1184), (40, 6000, 1056),
                                   (70, 14000, 2080)])
def test_linear4_act_groups(gpu, dtype, M, N, K):
    """The same of silu(g) u: the slope is at most 1.13, so a product's error passes at most 1.13 times; the activation
    is within 2^-20 of its value."""
    from m3x import ops
    g = _g(M + N + K + 1)
    x = (torch.randn(M, K, generator=g) * 2).to(dtype).to(gpu)
    pg, pu = (ops.pack_weight4((torch.randn(N, K, generator=g) * K ** -0.5).to(dtype).to(gpu)) for _ in "gu")
    a, da = _product(_f64(x), R.weight_values(pg.codes, pg.scales, N, K))
    b, db = _product(_f64(x), R.weight_values(pu.codes, pu.scales, N, K))
    act = a / (1 + np.exp(-a))
    y = act * b
    off = 1.13 * da * (np.abs(b) + db) + np.abs(act) * db + 2.0 ** -20 * np.abs(y)
    h, tiny = torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0
    got = _f64(ops.linear4_act(x, pg, pu, ops.ACT_SWIGLU))
    assert (np.abs(got - y) <= off + h * (np.abs(y) + off) + tiny).all()


def test_rows_of_x_stay_apart(gpu):
    """An infinity in one row of x changes that row alone, also where K ends inside a step, whatever the grouping."""
    from m3x import ops
    for M, N, K in ((6, 4200, 160), (16, 100, 96), (40, 6000, 1056), (130, 3700, 1184)):
        x = torch.randn(M, K, generator=_g(M)).bfloat16().to(gpu)
        p = ops.pack_weight4(torch.randn(N, K, generator=_g(N)).bfloat16().to(gpu))
        clean = ops.linear4(x, p)
        x[M - 2, K - 1] = float("inf")
        got = ops.linear4(x, p)
        rest = [r for r in range(M) if r != M - 2]
        w = R.weight_values(p.codes, p.scales, N, K)[:, K - 1]
        assert torch.equal(got[rest], clean[rest])
        want = torch.from_numpy(np.where(w == 0, np.nan, np.copysign(np.inf, w))).bfloat16().to(gpu)
        assert torch.equal(torch.nan_to_num(got[M - 2], nan=7.0), torch.nan_to_num(want, nan=7.0))
