"""The paged cache's operators on the GPU against 64 bits: attention over the range of heads, types, pages, lengths and
windows with every place that a row does not see holding NaN; writers and reader."""
import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _spans(p0, n, window, sinks, page):
    """What a slot holds for a run of n rows from p0: with a window no more than the rows see."""
    last = p0 + n
    first = max(0, p0 - window + 1) if window else 0
    return [(0, last)] if first <= sinks else ([(0, sinks)] if sinks else []) + [(first, last)]


def _case(runs, H, KV, D, page, dtype, window=0, sinks=0, seed=0, gap=0):
    """runs: (rows, first position). Returns CPU tensors of a call whose runs lie one behind the other, `gap` rows that
    no run holds between them, each run its own slot."""
    slots, pos, laid, held, at = [], [], [], {}, 0
    for s, (n, p0) in enumerate(runs):
        laid.append((at, n, p0))
        slots += [s + 1] * n + [0] * gap
        pos += list(range(p0, p0 + n)) + [5] * gap
        at += n + gap
        if p0 + n > 0:
            held[s + 1] = _spans(max(p0, 0), n + min(p0, 0), window, sinks, page)
    width = max([1] + [-(-end // page) for spans in held.values() for _, end in spans]) + 1
    table, pages = R.table_for(held, len(runs) + 2, page, width, seed)
    k, v = R.pools(table, pages, held, KV, page, D, dtype, seed + 1)
    q = R.normal(seed + 2, at, H, D).to(dtype)
    return q, k, v, table, torch.tensor(slots), torch.tensor(pos, dtype=torch.int32), laid


def _run(gpu, q, k, v, table, slots, pos, laid, scale, window=0, sinks=0, splits=None, ctx=None, cut=None):
    """cut: prompts in narrow tiles, or wide ones (None: as the plan decides)."""
    from m3x import ops

    class Plan(ops.PagedPlan):
        def _few(self, *a):
            return super()._few(*a) if cut is None else cut
    cache = ops.PagedKv(k.to(gpu), v.to(gpu), table.to(gpu))
    plan = Plan(laid, q.shape[1], k.shape[1], k.shape[3], ctx or cache.cap, window=window, sinks=sinks, device=gpu)
    if splits:
        plan.launches = [(*x[:4], splits) for x in plan.launches]
        plan._finish(torch.device(gpu))
    ws = torch.full((max(plan.workspace, 16),), 255, dtype=torch.uint8, device=gpu)
    out = torch.full_like(q, 7.0).to(gpu)
    ops.paged_attn(q.to(gpu), cache, out, slots.to(gpu), pos.to(gpu), scale, plan, ws)
    return out.cpu()


def _check(gpu, case, scale, window=0, sinks=0, **kw):
    q, k, v, table, slots, pos, laid = case
    want, bound = R.attention(q, k, v, table, slots, pos, scale, window, sinks, laid)
    inside = torch.zeros(len(q), dtype=torch.bool)
    for a, n, _ in laid:
        inside[a:a + n] = True
    for cut in (True, False):
        got = _run(gpu, *case, scale, window, sinks, cut=cut, **kw)
        assert (got[~inside] == 7).all()
        worst = R.within(got[inside], want[inside], bound[inside])
        assert worst <= 1, (cut, worst)
    return got


LENGTHS = [(1, 0), (1, 1), (1, 15), (1, 16), (1, 31), (1, 32), (1, 130), (1, 700), (1, -1)]


@pytest.mark.parametrize("H,KV,D,page,dtype", [(16, 8, 128, 64, BF), (4, 4, 64, 16, FP), (10, 2, 128, 16, FP),
                                               (8, 1, 64, 256, BF), (17, 1, 128, 32, BF), (71, 1, 64, 128, FP),
                                               (64, 2, 128, 32, BF)])
@pytest.mark.parametrize("splits", [1, 3])
def test_single_rows(gpu, H, KV, D, page, dtype, splits):
    case = _case(LENGTHS, H, KV, D, page, dtype)
    _check(gpu, case, D ** -0.5, splits=splits)


@pytest.mark.parametrize("H,KV,D,page,dtype", [(16, 8, 128, 64, BF), (4, 4, 64, 16, FP), (10, 2, 128, 16, BF),
                                               (8, 1, 64, 32, BF), (6, 2, 128, 256, FP)])
@pytest.mark.parametrize("splits", [1, 5])
def test_runs(gpu, H, KV, D, page, dtype, splits):
    """Drafted tokens, prompts and single rows in one call, runs that begin before position 0, rows in no run."""
    runs = [(3, 40), (1, 300), (2, 0), (70, 0), (1, -1), (65, 190), (4, 61), (130, 7), (40, -3), (5, -9)]
    _check(gpu, _case(runs, H, KV, D, page, dtype, gap=2, seed=3), D ** -0.5, splits=splits)


@pytest.mark.parametrize("D,page,dtype", [(128, 64, BF), (64, 16, FP), (128, 16, FP), (64, 128, BF)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 3), (64, 4), (100, 40), (333, 1), (10000, 7)])
@pytest.mark.parametrize("splits", [1, 4])
def test_windows(gpu, D, page, dtype, window, sinks, splits):
    """Pages that no row sees are released; what lies beside the window in a page that some row needs is NaN."""
    runs = [(1, 500), (1, 3), (3, 410), (80, 0), (90, 350), (1, -1), (130, 30)]
    case = _case(runs, 8, 2, D, page, dtype, window, sinks, seed=5)
    _check(gpu, case, D ** -0.5, window, sinks, splits=splits)


@pytest.mark.parametrize("n,p0", [(1, 300), (4, 200), (100, 250)])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_holes(gpu, n, p0, dtype):
    """Positions in no page (an entry of -1 or past the pool) are seen by no row, wherever they are."""
    q, k, v, table, slots, pos, laid = _case([(n, p0)], 4, 2, 128, 16, dtype)
    for b, bad in ((0, -1), (3, 1 << 20), (7, -5), (8, -1), (p0 // 16, -1)):
        table[1, b] = bad
    _check(gpu, (q, k, v, table, slots, pos, laid), 0.1, splits=2)
    table[1] = -1
    assert (_check(gpu, (q, k, v, table, slots, pos, laid), 0.1) == 0).all()


def test_outside(gpu):
    """Slots outside the cache give zeros, positions past the table's end see what there is."""
    q, k, v, table, slots, pos, laid = _case([(1, 20), (2, 30), (90, 30)], 4, 2, 64, 16, BF)
    table = table[:, :3].contiguous()  # 48 positions
    slots[0] = len(table)
    pos[1:3] = torch.tensor([2 ** 31 - 2, 2 ** 31 - 1], dtype=torch.int32)
    laid[1] = (1, 1, 0)
    got = _run(gpu, q, k, v, table, slots, pos, laid, 0.125)
    assert (got[0] == 0).all() and (got[2] == 7).all()
    k[table[2, 2].long(), :, :] = R.normal(1, 2, 16, 64).to(BF)  # the page is full for a row past the end
    v[table[2, 2].long(), :, :] = R.normal(2, 2, 16, 64).to(BF)
    got = _run(gpu, q, k, v, table, slots, pos, laid, 0.125)
    pos[1] = 47
    want, bound = R.attention(q, k, v, table, slots, pos, 0.125, runs=laid)
    assert R.within(got[3:], want[3:], bound[3:]) <= 1 and R.within(got[1], want[1], bound[1]) <= 1


@pytest.mark.parametrize("n,p0,window,sinks", [(4, 60, 0, 0), (100, 10, 0, 0), (4, 60, 20, 5), (100, 40, 30, 5), (1, 90, 20, 5)])
@pytest.mark.parametrize("dtype,D", [(BF, 128), (FP, 64), (FP, 128), (BF, 64)])
@pytest.mark.parametrize("cut", [False, True])
def test_wild_values(gpu, n, p0, window, sinks, dtype, D, cut):
    """An infinite or NaN value reaches the rows that see its position and no other."""
    q, k, v, table, slots, pos, laid = _case([(n, p0)], 4, 2, D, 16, dtype)
    bad = {p0 + n // 2: float("inf"), p0 + 3 * n // 4: float("nan"), 25: float("-inf"), 3: float("nan")}
    if not window:
        del bad[25], bad[3]
    clean = v.clone()
    for j, x in bad.items():
        v[table[1, j // 16].long(), 1, j % 16, 5] = x
        clean[table[1, j // 16].long(), 1, j % 16, 5] = 0.5
    got = _run(gpu, q, k, v, table, slots, pos, laid, 0.1, window, sinks, cut=cut)
    want, bound = R.attention(q, k, clean, table, slots, pos, 0.1, window, sinks, laid)
    hit = torch.zeros(got.shape, dtype=torch.bool)
    for r in range(n):
        hit[r, 2:, 5] = any(j in bad for j in R.see(p0 + r, window, sinks))
    assert not torch.isfinite(got[hit]).any() and torch.isfinite(got[~hit]).all()
    assert R.within(got[~hit], want[~hit], bound[~hit]) <= 1


@pytest.mark.parametrize("n", [1, 3, 70])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_scores(gpu, n, dtype):
    """Negative and zero scales, scores of any size, keys that are infinite where no row sees them."""
    q, k, v, table, slots, pos, laid = _case([(n, 100)], 4, 2, 128, 32, dtype)
    big = (q * 30, k * 30, v)
    for scale in (-0.1, 0.0, 0.5, 1e-30):
        _check(gpu, (q, k, v, table, slots, pos, laid), scale)
    want, bound = R.attention(*big, table, slots, pos, 3.0, runs=laid)  # one key has all the weight unless two are near
    for cut in (True, False):
        assert R.within(_run(gpu, *big, table, slots, pos, laid, 3.0, cut=cut), want, bound) <= 1
    if n == 1:
        table2 = table.clone()
        k2 = k.clone()
        k2[table[1, 101 // 32].long(), :, 101 % 32] = float("inf")
        _check(gpu, (q, k2, v, table2, slots, pos, laid), 0.1)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_large_values(gpu, dtype):
    """Values at the format's largest: their means are finite."""
    for n in (1, 40):
        q, k, v, table, slots, pos, laid = _case([(n, 999)], 2, 1, 128, 64, dtype)
        v = torch.where(torch.isfinite(v), torch.sign(v) * torch.finfo(dtype).max, v)
        v = v.abs()
        u = R.unit(dtype)
        for cut in (True, False):
            got = _run(gpu, q, k, v, table, slots, pos, laid, 0.1, splits=2, cut=cut)
            assert torch.isfinite(got).all() and (got.double() >= torch.finfo(dtype).max * (1 - 4 * u)).all()


@pytest.mark.parametrize("window,sinks", [(20, 100), (1, 1), (3, 64), (50, 2 ** 31 - 1), (2 ** 31 - 1, 5)])
def test_more_sinks_than_window(gpu, window, sinks):
    case = _case([(1, 300), (5, 90), (150, 40), (70, 230), (1, 2)], 4, 2, 128, 16, BF, window, sinks, seed=8)
    for splits in (1, 3):
        _check(gpu, case, 0.1, window, sinks, splits=splits)


@pytest.mark.parametrize("cut", [False, True])
@pytest.mark.parametrize("n", [1, 6, 90])
def test_wild_queries(gpu, n, cut):
    """An infinite or NaN query spoils its own row and head alone."""
    q, k, v, table, slots, pos, laid = _case([(n, 200), (n, 77)], 4, 2, 128, 32, BF)
    want, bound = R.attention(q, k, v, table, slots, pos, 0.1, runs=laid)
    bad = torch.zeros(len(q), 4, dtype=torch.bool)
    for r, h, x in ((0, 1, float("nan")), (n // 2, 2, float("inf")), (2 * n - 1, 0, float("nan"))):
        q[r, h, 3], bad[r, h] = x, True
    got = _run(gpu, q, k, v, table, slots, pos, laid, 0.1, splits=2, cut=cut)
    assert R.within(got[~bad], want[~bad], bound[~bad]) <= 1 and torch.isnan(got[bad]).any()


def test_far_pages(gpu):
    """Pages more than 2^32 bytes into the pools: written, read and attended as near ones."""
    from m3x import ops
    KV, page, D, pages = 8, 256, 128, 9000  # 4.7 GB a pool
    if torch.cuda.mem_get_info()[0] < 16e9:
        pytest.skip("needs 10 GB")
    near, far = torch.tensor([3, 1, 5]), torch.tensor([8999, 8500, 8998])
    table = torch.stack([near, far]).int()
    k, v = (torch.empty(pages, KV, page, D, dtype=BF, device=gpu) for _ in "kv")
    cache = ops.PagedKv(k, v, table.to(gpu))
    n = 700
    x = R.normal(1, 2, n, KV, D).to(BF).to(gpu)
    pos = torch.arange(n, dtype=torch.int32, device=gpu)
    out = []
    for s in (0, 1):
        slots = torch.full((n,), s, dtype=torch.long, device=gpu)
        ops.paged_append(x[0], x[1], cache, slots, pos)
        a, b = torch.empty_like(x[0]), torch.empty_like(x[1])
        ops.paged_read(cache, slots, pos, a, b)
        assert torch.equal(a, x[0]) and torch.equal(b, x[1])
        q = R.normal(2, 230, 16, D).to(BF).to(gpu)
        rows = slots[:230], torch.cat([pos[:100], pos[500:630]])
        for runs in ([(r, 1, 0) for r in range(230)], [(0, 100, 0), (100, 130, 500)]):
            for few in (True, False):
                class Plan(ops.PagedPlan):
                    def _few(self, *a):
                        return few
                plan = Plan(runs, 16, KV, D, 700, device=gpu)
                ws = torch.empty(max(16, plan.workspace), dtype=torch.uint8, device=gpu)
                out.append(torch.empty_like(q))
                ops.paged_attn(q, cache, out[-1], *rows, 0.1, plan, ws)
    for a, b in zip(out[:4], out[4:]):
        assert torch.equal(a, b)
    want, bound = R.attention(q.cpu(), k[:6].cpu(), v[:6].cpu(), table[:1], torch.zeros(230, dtype=torch.long), rows[1].cpu(), 0.1)
    for a in out[:4]:
        assert R.within(a, want, bound) <= 1


def test_strides(gpu):
    """q and out as views of wider rows, pools as a view of joined ones, a plan's rows in any order."""
    from m3x import ops
    q, k, v, table, slots, pos, laid = _case([(1, 50), (60, 33), (4, 70)], 8, 2, 64, 32, BF)
    joined = torch.stack([k, v], 1).to(gpu)
    cache = ops.PagedKv(joined[:, 0], joined[:, 1], table.to(gpu))
    wide = torch.zeros(len(q), 8, 96, dtype=BF, device=gpu)
    wide[:, :, :64] = q.to(gpu)
    out = torch.full((8, len(q), 64), 3.0, dtype=BF, device=gpu)
    plan = ops.PagedPlan(laid[::-1], 8, 2, 64, 100, device=gpu)
    ops.paged_attn(wide[:, :, :64], cache, out.transpose(0, 1), slots.to(gpu), pos.to(gpu), 0.125, plan,
                   torch.empty(plan.workspace, dtype=torch.uint8, device=gpu) if plan.workspace else None)
    want, bound = R.attention(q, k, v, table, slots, pos, 0.125, runs=laid)
    assert R.within(out.transpose(0, 1), want, bound) <= 1


@pytest.mark.parametrize("H,KV,D,rows", [(32, 4, 64, 5), (32, 4, 64, 6), (24, 1, 64, 2), (40, 1, 64, 1), (48, 1, 64, 1),
                                         (33, 1, 128, 1), (40, 1, 128, 1)])
@pytest.mark.parametrize("splits", [1, 2, 7, 11])
def test_middling_columns(gpu, H, KV, D, rows, splits):
    """33 to 48 columns a tile, splits that fill no batch of eight."""
    case = _case([(rows, 1500), (rows, 31), (1, 0), (rows, 640), (rows, -rows)], H, KV, D, 32, FP, seed=5)
    _check(gpu, case, D ** -0.5, splits=splits)


def test_shared_pages(gpu):
    """Slots that name the same pages: each reads them as its own."""
    q, k, v, table, slots, pos, laid = _case([(1, 200)] * 3 + [(70, 64)], 4, 4, 128, 32, BF)
    table[2, :4], table[3, :6], table[4, :2] = table[1, :4], table[1, :6], table[1, :2]
    _check(gpu, (q, k, v, table, slots, pos, laid), 0.1, splits=2)


def test_long(gpu):
    """A long context in many pages, split: counted positions and pages past one load of page numbers."""
    case = _case([(1, 33000), (3, 20011)], 4, 1, 64, 16, BF, seed=9)
    for splits in (1, 64):
        _check(gpu, case, 0.125, splits=splits)
    case = _case([(40, 9000)], 2, 1, 128, 32, FP, seed=10)
    for splits in (1, 9):
        _check(gpu, case, 0.1, splits=splits)


# ---------------------------------------------------------------- writers and reader
def _places(n, slots, cap, seed):
    """n different places, the last one outside by its slot, the one before by its position, one at a released page."""
    g = torch.Generator().manual_seed(seed)
    flat = torch.randperm(slots * cap, generator=g)[:n]
    s, p = flat // cap, (flat % cap).int()
    if n > 3:
        s[-1], p[-2] = slots, cap
        s[-3], p[-3] = 0, -1
    return s, p


@pytest.mark.parametrize("KV,D,page,dtype", [(8, 128, 64, BF), (1, 64, 16, FP), (3, 128, 256, FP), (2, 64, 32, BF)])
@pytest.mark.parametrize("rows", [1, 5, 300])
def test_append_and_read(gpu, KV, D, page, dtype, rows):
    from m3x import ops
    slots, width = 3, 512 // page
    table = torch.randperm(slots * width + 4)[:slots * width].int().view(slots, width)
    table[1, 1] = -1
    cache = ops.PagedKv.empty(slots * width + 4, KV, page, D, table.to(gpu), dtype)
    assert cache.memory_bytes() == 2 * (slots * width + 4) * KV * page * D * 2
    cache.k.fill_(9)
    cache.v.fill_(9)
    s, p = _places(rows, slots, 512, rows)
    x = R.normal(rows, rows, KV + 1, 2 * D).to(dtype).to(gpu)
    k, v = x[:, :KV, :D], x[:, 1:, D:]
    ops.paged_append(k, v, cache, s.to(gpu), p.to(gpu))
    wk, wv = torch.full(cache.k.shape, 9.0, dtype=dtype), torch.full(cache.k.shape, 9.0, dtype=dtype)
    held = torch.zeros(rows, dtype=torch.bool)
    for r in range(rows):
        if 0 <= s[r] < slots and 0 <= p[r] < 512 and table[s[r], p[r] // page] >= 0:
            held[r] = True
            wk[table[s[r], p[r] // page], :, p[r] % page] = k[r].cpu()
            wv[table[s[r], p[r] // page], :, p[r] % page] = v[r].cpu()
    assert torch.equal(cache.k.cpu(), wk) and torch.equal(cache.v.cpu(), wv)
    back = torch.full((2, KV, rows, D), 5.0, dtype=dtype, device=gpu)
    ops.paged_read(cache, s.to(gpu), p.to(gpu), back[0].transpose(0, 1), back[1].transpose(0, 1))
    for b, x in ((back[0], k), (back[1], v)):
        assert torch.equal(b.transpose(0, 1).cpu(), torch.where(held[:, None, None], x.cpu(), torch.zeros_like(x.cpu())))


@pytest.mark.parametrize("H,KV,D,dim,dtype", [(16, 8, 128, 128, BF), (4, 4, 64, 64, FP), (5, 1, 128, 48, FP),
                                              (3, 3, 64, 16, BF), (7, 2, 128, 96, BF)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("rows", [1, 19, 2100])
def test_qk_norm_rope(gpu, H, KV, D, dim, dtype, interleaved, norm, rows):
    """Queries and keys within half a step of the 64-bit result, values as they are, at positions up to 2^30. The fp32
    chain in front of the rounding: a sum of D squares, root, quotient and two products (below D 2^-24 of the value),
    sine and cosine within 4 2^-24 and angles within 2^-31 turns, of both rotated numbers."""
    from m3x import ops
    page, slots = 64, 3
    cap = 1 << 30
    g = torch.Generator().manual_seed(rows)
    pos = torch.randint(0, cap, (rows,), generator=g).int()
    pos[::3] = torch.randint(0, 5000, (len(pos[::3]),), generator=g).int()
    s = torch.arange(rows) % slots
    if rows > 3:
        pos[1], s[2] = -1, slots
    pages = rows + 1
    table = torch.full((slots, cap // page), -1, dtype=torch.int32)
    ok = (pos >= 0) & (s < slots)
    blocks = torch.unique(s[ok] * (cap // page) + pos[ok] // page)
    table.view(-1)[blocks] = torch.randperm(pages, generator=g)[:len(blocks)].int()
    cache = ops.PagedKv.empty(pages, KV, page, D, table.to(gpu), dtype)
    f, factor = ops.rotary_freqs(dim, 1e4, "parts", by=4.0, trained=4096)
    rotary = ops.Rotary(f, interleaved=interleaved, factor=factor, device=gpu)
    x = R.normal(rows + 1, rows, H + 2 * KV, D)
    x[:, H] *= 50
    qkv = torch.zeros(rows, (H + 2 * KV) * D + 8, dtype=dtype)
    qkv[:, :-8] = x.to(dtype).flatten(1)
    x = qkv[:, :-8].reshape(rows, H + 2 * KV, D)
    wq, wk = (torch.exp(R.normal(i, D)).to(dtype) if norm else None for i in (5, 6))
    q = torch.full((rows, H + 1, D), 3.0, dtype=dtype, device=gpu)
    ops.qk_norm_rope_paged(qkv.to(gpu)[:, :-8], q[:, :H], cache, s.to(gpu), pos.to(gpu), rotary,
                           *(w.to(gpu) if norm else None for w in (wq, wk)), 1e-6, H)
    assert (q[:, H] == 3).all()
    u = R.unit(dtype)
    keys, values = (torch.empty(rows, KV, D, dtype=dtype, device=gpu) for _ in "kv")
    ops.paged_read(cache, s.to(gpu), pos.to(gpu), keys, values)
    # two rows at one place leave a mixture: not compared
    place = torch.where(ok, s * cap + pos, -1 - torch.arange(rows))
    _, inverse, counts = torch.unique(place, return_inverse=True, return_counts=True)
    alone = counts[inverse] == 1
    for got, part, w in ((q[:, :H], x[:, :H], wq), (keys, x[:, H:H + KV], wk)):
        want = R.rotate(part, pos, f, interleaved, factor, w, 1e-6)
        size = want.abs() + 0.0
        rot = want[..., :dim].abs()
        if interleaved:
            pair = torch.maximum(rot[..., 0::2], rot[..., 1::2]).repeat_interleave(2, -1)
        else:
            pair = torch.maximum(rot[..., :dim // 2], rot[..., dim // 2:]).repeat(1, 1, 2)
        size[..., :dim] = pair
        tiny = 2.0 ** -25 if dtype == FP else 0.0  # half of fp16's smallest step
        bound = u * want.abs() * (1 + 2 * u) + (D + 24) * 2.0 ** -24 * 1.5 * size + tiny
        if part is not x[:, :H] and got is keys:
            assert (got.cpu()[~ok] == 0).all()
            got, want, bound = got.cpu()[ok & alone], want[ok & alone], bound[ok & alone]
        assert R.within(got, want, bound) <= 1
    assert torch.equal(values.cpu()[ok & alone], x[ok & alone][:, H + KV:])
