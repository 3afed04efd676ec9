"""Ways of calling the paged cache's operators: run together as a step runs them, streams, captured graphs (several
replays with eager work between, one workspace under two graphs, changing layouts), repeated calls."""
import pytest
import torch

import paged_reference as R

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
H, KV, D, PAGE, EPS, SCALE = 8, 2, 128, 32, 1e-6, 0.08


class Step:
    """One layer's step over a cache of `lengths` positions a slot: rows of the runs are written, then attend."""

    def __init__(self, gpu, lengths, runs, window=0, sinks=0, seed=0, cap=640, plan=None):
        from m3x import ops
        self.ops, self.window, self.sinks = ops, window, sinks
        slots, pos, laid = [], [], []
        for s, n in runs:
            laid.append((len(slots), n, lengths[s]))
            slots += [s] * n
            pos += range(lengths[s], lengths[s] + n)
        held = {s: [(0, n + sum(m for t, m in runs if t == s))] for s, n in enumerate(lengths)}
        self.table, pages = R.table_for(held, len(lengths), PAGE, cap // PAGE, seed)
        self.k, self.v = R.pools(self.table, pages, {s: [(0, n)] for s, n in enumerate(lengths)}, KV, PAGE, D, BF, seed + 1)
        self.f, _ = ops.rotary_freqs(D, 1e6)
        self.laid, self.slots, self.pos = laid, torch.tensor(slots), torch.tensor(pos, dtype=torch.int32)
        self.qkv = R.normal(seed + 2, len(slots), (H + 2 * KV) * D).to(BF)
        self.wq, self.wk = (torch.exp(R.normal(seed + i, D) / 4).to(BF) for i in (3, 4))
        self.gpu = {n: getattr(self, n).to(gpu) for n in ("slots", "pos", "qkv", "wq", "wk")}
        self.cache = ops.PagedKv(self.k.to(gpu), self.v.to(gpu), self.table.to(gpu))
        self.rotary = ops.Rotary(self.f, device=gpu)
        self.plan = plan or ops.PagedPlan(laid, H, KV, D, cap, window=window, sinks=sinks, device=gpu)
        self.ws = torch.empty(self.plan.workspace, dtype=torch.uint8, device=gpu) if self.plan.workspace else None
        self.q = torch.empty(len(slots), H, D, dtype=BF, device=gpu)
        self.out = torch.full_like(self.q, 7.0)

    def run(self):
        g, ops = self.gpu, self.ops
        ops.qk_norm_rope_paged(g["qkv"], self.q, self.cache, g["slots"], g["pos"], self.rotary, g["wq"], g["wk"], EPS, H)
        ops.paged_attn(self.q, self.cache, self.out, g["slots"], g["pos"], SCALE, self.plan, self.ws)

    def check(self):
        """Queries, keys and outputs against 64 bits, each from the 16-bit numbers that the one before it wrote."""
        ops = self.ops
        n = len(self.slots)
        keys, values = (torch.empty(n, KV, D, dtype=BF, device=self.q.device) for _ in "kv")
        ops.paged_read(self.cache, self.gpu["slots"], self.gpu["pos"], keys, values)
        x = self.qkv.view(n, H + 2 * KV, D)
        u = R.unit(BF)
        for got, part, w in ((self.q, x[:, :H], self.wq), (keys, x[:, H:H + KV], self.wk)):
            want = R.rotate(part, self.pos, self.f, False, 1.0, w, EPS)
            pair = torch.maximum(want[..., :D // 2].abs(), want[..., D // 2:].abs()).repeat(1, 1, 2)
            # half a step of the result and the chain in fp32 before it, relative to the rotated pair
            assert R.within(got, want, u * want.abs() * (1 + 2 * u) + (D + 24) * 2.0 ** -24 * 1.5 * pair) <= 1
        assert torch.equal(values.cpu(), x[:, H + KV:])
        want, bound = R.attention(self.q.cpu(), self.cache.k.cpu(), self.cache.v.cpu(), self.table, self.slots, self.pos, SCALE,
                                  self.window, self.sinks, self.laid)
        assert R.within(self.out, want, bound) <= 1


LAYOUTS = [([0, 1, 31, 500], [(s, 1) for s in range(4)]), ([10, 0, 300], [(0, 1), (1, 90), (2, 5)]),
           ([400, 64], [(1, 3), (0, 200)])]


@pytest.mark.parametrize("lengths,runs", LAYOUTS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4)])
def test_step(gpu, lengths, runs, window, sinks):
    """Writing and attending in one go: rows see what this call's writer wrote."""
    st = Step(gpu, lengths, runs, window, sinks)
    st.run()
    st.check()


def test_other_stream(gpu):
    """A call works on the current stream: two streams side by side, each with a cache, a plan and a workspace."""
    steps = [Step(gpu, *LAYOUTS[i], seed=i) for i in (0, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(5):
        for s, st in zip(streams, steps):
            with torch.cuda.stream(s):
                st.run()
    torch.cuda.synchronize()
    for st in steps:
        st.check()


@pytest.mark.parametrize("layout", LAYOUTS)
def test_repeated(gpu, layout):
    """The same call gives the same bits, whichever split is done last."""
    from m3x import ops
    st = Step(gpu, *layout, cap=1280)
    st.run()
    first = st.out.clone()
    for splits in (1, 3, 4):
        st.plan.launches = [(*x[:4], splits) for x in st.plan.launches]
        st.plan._finish(torch.device(gpu))
        ws = torch.empty(max(16, st.plan.workspace), dtype=torch.uint8, device=gpu)
        seen = []
        for i in range(6):
            ws.fill_(255 * (i % 2))  # what the workspace holds beforehand does not matter
            ops.paged_attn(st.q, st.cache, st.out, st.gpu["slots"], st.gpu["pos"], SCALE, st.plan, ws)
            seen.append(st.out.clone())
        st.check()
        assert all(torch.equal(seen[0], x) for x in seen)
    assert first.shape == st.out.shape


def _capture(fn):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fn()
    return g


def test_two_graphs_one_workspace(gpu):
    """Two captured steps, replayed in turn with eager calls between them, share a workspace: each replay is the eager
    result, also after positions move."""
    steps = [Step(gpu, *LAYOUTS[0], seed=3), Step(gpu, [300, 444], [(0, 4), (1, 1)], seed=4)]
    for st in steps:
        st.plan.launches = [(*x[:4], 2) for x in st.plan.launches]
        st.plan._finish(torch.device(gpu))
    ws = torch.zeros(max(st.plan.workspace for st in steps), dtype=torch.uint8, device=gpu)
    assert all(st.plan.workspace for st in steps)
    for st in steps:
        st.ws = ws
    graphs = [_capture(st.run) for st in steps]
    for turn in range(4):
        for st, g in zip(steps, graphs):
            st.out.fill_(3.0)
            g.replay()
            got = st.out.clone()
            torch.cuda.synchronize()
            st.check()
            st.run()
            assert torch.equal(got, st.out)
        if turn == 1:
            for st in steps:  # each run one position back
                st.pos = (st.pos - 1).clamp_min(0)
                st.gpu["pos"].copy_(st.pos)
                st.laid = [(a, n, max(0, p - 1)) for a, n, p in st.laid]


@pytest.mark.parametrize("few", [True, False])
def test_reserved_plan(gpu, few, monkeypatch):
    """One captured call over a reserved plan: layouts of its rows change from replay to replay."""
    from m3x import ops
    monkeypatch.setattr(ops.PagedPlan, "_few", lambda *a: few)
    cap, rows = 640, 230
    held = {s: [(0, cap)] for s in range(6)}
    table, pages = R.table_for(held, 6, PAGE, cap // PAGE, 1)
    k, v = R.pools(table, pages, held, KV, PAGE, D, BF, 2)
    q = R.normal(3, rows, H, D).to(BF)
    cache = ops.PagedKv(k.to(gpu), v.to(gpu), table.to(gpu))
    for window, sinks in ((0, 0), (70, 3)):
        plan = ops.PagedPlan.reserve(rows, H, KV, D, cap, window=window, sinks=sinks, device=gpu)
        slots, pos = torch.zeros(rows, dtype=torch.long, device=gpu), torch.zeros(rows, dtype=torch.int32, device=gpu)
        out, x = torch.empty(rows, H, D, dtype=BF, device=gpu), q.to(gpu)
        ws = torch.empty(max(plan.workspace, 16), dtype=torch.uint8, device=gpu)
        g = _capture(lambda: ops.paged_attn(x, cache, out, slots, pos, SCALE, plan, ws))
        for lens in ([1] * 6, [230], [1, 1, 100, 4, 2, 90], [5, 4], [130, 17, 64]):
            laid, at = [], 0
            for s, n in enumerate(lens):
                laid.append((at, n, 37 * s + 5))
                slots[at:at + n] = s
                pos[at:at + n] = torch.arange(n, device=gpu) + 37 * s + 5
                at += n
            for t, new in zip(plan.launches, plan.tiles(laid)):
                t[0].copy_(torch.from_numpy(new))
            out.fill_(7.0)
            g.replay()
            torch.cuda.synchronize()
            want, bound = R.attention(q, k, v, table, slots.cpu(), pos.cpu(), SCALE, window, sinks, laid)
            assert (out[at:] == 7).all() and R.within(out[:at], want[:at], bound[:at]) <= 1


@pytest.mark.parametrize("rows", [20, 40])
def test_plan_of_other_positions(gpu, rows):
    """A plan's positions are a rule's input: rows elsewhere (shorter, longer, past the largest context, none) get theirs."""
    from m3x import ops
    held = {s: [(0, 1280)] for s in range(rows)}
    table, pages = R.table_for(held, rows, PAGE, 1280 // PAGE, 1)
    k, v = R.pools(table, pages, held, KV, PAGE, D, BF, 2)
    q, slots = R.normal(3, rows, H, D).to(BF), torch.arange(rows)
    cache = ops.PagedKv(k.to(gpu), v.to(gpu), table.to(gpu))
    plan = ops.PagedPlan([(r, 1, 20 * (r + 1)) for r in range(rows)], H, KV, D, 20 * rows, device=gpu)
    assert plan.launches[0][0] is not None and plan.launches[0][4] > 1
    ws = torch.empty(plan.workspace, dtype=torch.uint8, device=gpu)
    out = torch.empty(rows, H, D, dtype=BF, device=gpu)
    for at in (lambda r: 20 * (r + 1), lambda r: 1279 - 30 * r, lambda r: r - 3, lambda r: 1279):
        pos = torch.tensor([at(r) for r in range(rows)], dtype=torch.int32)
        out.fill_(7.0)
        ops.paged_attn(q.to(gpu), cache, out, slots.to(gpu), pos.to(gpu), SCALE, plan, ws)
        want, bound = R.attention(q, k, v, table, slots, pos, SCALE)
        assert R.within(out, want, bound) <= 1


def test_no_rows(gpu):
    """Calls without rows, and a plan without runs, do nothing."""
    from m3x import ops
    cache = ops.PagedKv.empty(3, KV, PAGE, D, torch.zeros(1, 4, dtype=torch.int32, device=gpu))
    kv, q = torch.empty(0, KV, D, dtype=BF, device=gpu), torch.empty(0, H, D, dtype=BF, device=gpu)
    at = torch.empty(0, dtype=torch.long, device=gpu), torch.empty(0, dtype=torch.int32, device=gpu)
    ops.paged_append(kv, kv, cache, *at)
    ops.paged_read(cache, *at, kv, kv)
    w = torch.ones(D, dtype=BF, device=gpu)
    ops.qk_norm_rope_paged(torch.empty(0, (H + 2 * KV) * D, dtype=BF, device=gpu), q, cache, *at,
                           ops.Rotary(ops.rotary_freqs(D, 1e4)[0], device=gpu), w, w, EPS, H)
    ops.paged_attn(q, cache, q, *at, 1.0, ops.PagedPlan([], H, KV, D, 64, device=gpu))
    x, at = torch.ones(2, H, D, dtype=BF, device=gpu), (torch.zeros(2, dtype=torch.long, device=gpu),
                                                        torch.zeros(2, dtype=torch.int32, device=gpu))
    out = torch.full_like(x, 7.0)
    ops.paged_attn(x, cache, out, *at, 1.0, ops.PagedPlan([(0, 0, 5)], H, KV, D, 64, device=gpu))
    assert (out == 7).all() and (cache.k == 0).all() and (cache.v == 0).all()


def test_many_tiles(gpu):
    """As many tiles as a call holds, and one more."""
    from m3x import ops
    n = 65535
    table = torch.arange(8, dtype=torch.int32).view(2, 4)
    k, v = R.pools(table, 8, {0: [(0, 64)], 1: [(0, 64)]}, 1, 16, 64, BF, 1)
    cache = ops.PagedKv(k.to(gpu), v.to(gpu), table.to(gpu))
    slots, pos = torch.arange(n) % 2, (torch.arange(n) % 64).int()
    q = R.normal(2, 128, 1, 64).to(BF).repeat(n // 128 + 1, 1, 1)[:n].contiguous()
    out = torch.empty(n, 1, 64, dtype=BF, device=gpu)
    plan = ops.PagedPlan([(r, 1, 0) for r in range(n)], 1, 1, 64, 64, device=gpu)
    ops.paged_attn(q.to(gpu), cache, out, slots.to(gpu), pos.to(gpu), 0.125, plan)
    assert torch.equal(out, out[:128].repeat(n // 128 + 1, 1, 1)[:n])
    want, bound = R.attention(q[:128], k, v, table, slots[:128], pos[:128], 0.125)
    assert R.within(out[:128], want, bound) <= 1
    with pytest.raises(ValueError):
        ops.PagedPlan([(r, 1, 0) for r in range(n + 1)], 1, 1, 64, 64, device=gpu)
