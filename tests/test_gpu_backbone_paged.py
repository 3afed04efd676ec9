"""StaticBackbone(page_size=...) on the GPU against the eager oracle: decode, inline prefill, prefix install, export and
fork, graphs, windows whose pages go back to the pool, the pool's end, and a captured frame step."""
import pytest
import torch

from helpers import convert, floor_check, report
from m3x import synth
from oracle import torch_oracle as O

pytestmark = pytest.mark.gpu

LAYERS, S, CAP, PAGE = 3, 6, 512, 16
PREFIX = [0, 1, 31, 200, 300, 0]


def _oracle(bb_c, slots, kv, cap, D):
    """The 16-bit oracle (16-bit rotation tables) and its evaluation in 32 bits (32-bit tables)."""
    new = lambda dt: [torch.zeros(slots + 1, kv, cap, D, dtype=dt) for _ in bb_c.lm.model.layers]  # noqa: E731
    bf, fp = O.rope_tables(D, 1e6, cap, torch.bfloat16), O.rope_tables(D, 1e6, cap, torch.float32)
    lengths = torch.zeros(slots + 1, dtype=torch.long)
    return ([bb_c, new(torch.bfloat16), new(torch.bfloat16), lengths, *bf],
            [convert(bb_c, torch.float32), new(torch.float32), new(torch.float32), lengths.clone(), *fp])


def _setup(gpu, use_graphs=True, prefix=PREFIX, **kw):
    from m3x.serve.fast_backbone import StaticBackbone
    bb_g = synth.qwen3_backbone(layers=LAYERS, seed=21, device=gpu, affine=synth.AFFINE)
    bb_c = synth.qwen3_backbone(layers=LAYERS, seed=21, device="cpu", affine=synth.AFFINE)
    sb = StaticBackbone(bb_g, S, capacity=CAP, batch_buckets=(1, 2, 4, 8, 64), ctx_buckets=(256, 512),
                        use_graphs=use_graphs, page_size=PAGE, **kw)
    both = _oracle(bb_c, S, 8, CAP, 128)
    g = torch.Generator().manual_seed(22)
    for s, n in enumerate(prefix):
        kv = []
        for i in range(LAYERS):
            k, v = (torch.randn(1, 8, n, 128, generator=g).to(torch.bfloat16) for _ in "kv")
            for o in both:
                o[1][i][s, :, :n], o[2][i][s, :, :n] = k[0], v[0]
            kv.append((k.to(gpu), v.to(gpu)))
        sb.load_prefix(s, kv, n)
        for o in both:
            o[3][s] = n
    return sb, both


def _step(both, slots, x, offset=None, ctx=None):
    slots = torch.tensor(slots)
    return tuple(O.backbone_step(o[0], o[1], o[2], o[3], slots, x.to(o[1][0][:1, :1, :1, :1].dtype), o[4], o[5],
                                 offset=offset, ctx=ctx) for o in both)


def test_install_and_export(gpu):
    """A slot holds what was installed, in as many pages as it needs, and gives them back."""
    sb, both = _setup(gpu)
    assert sb.k == [] and sb.v == [] and len(sb.paged) == LAYERS and sb.pages.pages == S * CAP // PAGE
    assert sb.memory_bytes() == LAYERS * S * CAP * 8 * 128 * 4
    for s, n in enumerate(PREFIX):
        assert sb.pages.held(s) == -(-n // PAGE)
        for i, (k, v) in enumerate(sb.export_prefix(s)):
            assert tuple(k.shape) == (1, 8, n, 128)
            assert torch.equal(k[0].cpu(), both[0][1][i][s, :, :n]) and torch.equal(v[0].cpu(), both[0][2][i][s, :, :n])
    kv = sb.export_prefix(4)
    sb.load_prefix(5, kv, 300)
    for a, b in zip(sb.export_prefix(5), kv):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    free = sb.pages.free_pages
    sb.free(5)
    sb.load_prefix(4, [(k[:, :, :0], v[:, :, :0]) for k, v in kv], 0)
    assert sb.lengths_cpu[4] == 0 and sb.pages.free_pages == free + 2 * 19


def test_step_matches_oracle(gpu):
    """Decode steps of four seats and of one, lengths advanced."""
    sb, both = _setup(gpu)
    g = torch.Generator().manual_seed(23)
    for t, slots in enumerate(([0, 2, 3, 4], [0, 2, 3, 4], [3], [4, 1])):
        x = torch.randn(len(slots), 1024, generator=g).to(torch.bfloat16)
        out = sb.step(slots, x.to(gpu))
        ok, info = floor_check(out, *_step(both, slots, x))
        report(f"paged step {t}", info)
        assert ok, (t, info)
    assert sb.lengths.cpu().tolist() == both[0][3].tolist() == sb.lengths_cpu and not sb._persistent_ok(1)


def test_mixed_and_prefill(gpu):
    """Decoding seats with two inline prefills in one step (twice, with other layouts in the same graph), then a prompt
    in pieces of the largest bucket."""
    sb, both = _setup(gpu)
    g = torch.Generator().manual_seed(24)
    x = torch.randn(2, 1024, generator=g).to(torch.bfloat16)
    p5, p1 = ((torch.randn(n, 1024, generator=g) * 0.5).to(torch.bfloat16) for n in (20, 7))
    dec, last = sb.step_mixed([0, 3], x.to(gpu), [(5, p5.to(gpu)), (1, p1.to(gpu))])
    ref, truth = _step(both, [0, 3] + [5] * 20 + [1] * 7, torch.cat([x, p5, p1]),
                       torch.tensor([0, 0] + list(range(20)) + list(range(7))))
    ok, info = floor_check(torch.cat([dec, torch.stack(last)]), ref[[0, 1, 21, 28]], truth[[0, 1, 21, 28]])
    assert ok, info
    dec, last = sb.step_mixed([3], x[:1].to(gpu), [(4, torch.cat([p1, p5]).to(gpu))])
    ref, truth = _step(both, [3] + [4] * 27, torch.cat([x[:1], p1, p5]), torch.tensor([0] + list(range(27))))
    ok, info = floor_check(torch.cat([dec, torch.stack(last)]), ref[[0, 27]], truth[[0, 27]])
    assert ok, info
    p = (torch.randn(100, 1024, generator=g) * 0.5).to(torch.bfloat16)
    got = sb.prefill(2, p.to(gpu))
    ref, truth = _step(both, [2] * 100, p, torch.arange(100))
    ok, info = floor_check(got[None], ref[-1:], truth[-1:])
    assert ok, info
    assert sb.lengths_cpu[:S] == [1, 8, 131, 202, 327, 20]


def test_graph_replay_equals_eager(gpu):
    a, b = _setup(gpu, use_graphs=True)[0], _setup(gpu, use_graphs=False)[0]
    a.warmup()
    g = torch.Generator().manual_seed(25)
    for slots in ([0, 2, 3, 4], [0, 2, 3, 4], [1], [4, 0], [0, 2, 3, 4]):
        x = torch.randn(len(slots), 1024, generator=g).to(torch.bfloat16).to(gpu)
        assert torch.equal(a.step(slots, x), b.step(slots, x))
        torch.cuda.synchronize()
    for n in (5, 40, 12):
        x, p = (torch.randn(m, 1024, generator=g).to(torch.bfloat16).to(gpu) for m in (2, n))
        (d0, l0), (d1, l1) = (o.step_mixed([2, 0], x, [(1, p), (5, p[:3])]) for o in (a, b))
        assert torch.equal(d0, d1) and all(torch.equal(m, n) for m, n in zip(l0, l1))
    for s in range(S):
        for (k0, v0), (k1, v1) in zip(a.export_prefix(s), b.export_prefix(s)):
            assert torch.equal(k0, k1) and torch.equal(v0, v1)


def test_fork(gpu):
    """A forked slot answers like one with the prefix of its own, in fewer pages; neither writes into the other, and the
    pages outlive the source."""
    sb, _ = _setup(gpu)
    sb.load_prefix(5, sb.export_prefix(4), 300)
    free = sb.pages.free_pages
    sb.fork(0, 4)
    sb.fork(2, 4, 288)
    assert sb.pages.free_pages == free + 2 - 1 and sb.lengths_cpu[0] == 300 and sb.lengths_cpu[2] == 288
    g = torch.Generator().manual_seed(3)
    for t in range(20):
        x = torch.randn(1, 1024, generator=g).to(torch.bfloat16).to(gpu)
        y = torch.randn(1, 1024, generator=g).to(torch.bfloat16).to(gpu)
        out = sb.step([0, 5, 4], torch.cat([x, x, y]))
        assert torch.equal(out[0], out[1]) and not torch.equal(out[0], out[2])
        if t == 10:
            sb.free(4)
            sb.load_prefix(4, [(k[:, :, :40], v[:, :, :40]) for k, v in sb.export_prefix(3)], 40)
    for a, b in zip(sb.export_prefix(0), sb.export_prefix(5)):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for a, b in zip(sb.export_prefix(2), sb.export_prefix(5, 288)):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for s in range(S):
        sb.free(s)
    assert sb.pages.free_pages == sb.pages.pages


def test_window_stream(gpu):
    """A stream under a window with sinks: a prompt and one-row steps against the oracle over the positions each row
    sees, in a pool of no more pages than the window, the sinks and a prompt take."""
    from m3x.serve.fast_backbone import StaticBackbone
    window, sinks, cap = 40, 5, 400
    geo = dict(layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, inter=768, seed=31, affine=synth.AFFINE)
    sb = StaticBackbone(synth.qwen3_backbone(device=gpu, **geo), 2, capacity=cap, batch_buckets=(2, 32), ctx_buckets=(cap,),
                        page_size=PAGE, pages=7, window=window, sinks=sinks)
    both = _oracle(synth.qwen3_backbone(device="cpu", **geo), 2, 2, cap, 64)
    full = [(o[1], o[2]) for o in both]

    class Seen:
        def __init__(self, t):
            self.t = t

        def __setitem__(self, at, x):
            self.t[at] = x

        def __getitem__(self, at):
            return self.t[at] if isinstance(at[2], int) else self.t[:, :, self.keys]
    for o in both:
        o[1], o[2] = [Seen(t) for t in o[1]], [Seen(t) for t in o[2]]

    def oracle(x):
        p = int(both[0][3][1])
        keys = [j for j in range(p + 1) if j > p - window or j < sinks]
        for o in both:
            for c in o[1] + o[2]:
                c.keys = keys
        return tuple(O.backbone_step(o[0], o[1], o[2], o[3], torch.tensor([1]), x.to(o[4].dtype), o[4], o[5], ctx=len(keys))
                     for o in both)
    g = torch.Generator().manual_seed(32)
    for n in (30, 32, 25):
        p = (torch.randn(n, 512, generator=g) * 0.5).to(torch.bfloat16)
        got = sb.prefill(1, p.to(gpu))
        for r in range(n):
            want = oracle(p[r:r + 1])
        ok, info = floor_check(got[None], *want)
        assert ok, (n, info)
    worst = 0
    for t in range(110):
        x = torch.randn(1, 512, generator=g).to(torch.bfloat16)
        out = sb.step([1], x.to(gpu))
        ok, info = floor_check(out, *oracle(x))
        assert ok, (t, info)
        worst = max(worst, sb.pages.held(1))
    assert worst <= 1 + -(-window // PAGE) + 1 and sb.lengths_cpu[1] == 197
    with pytest.raises(ValueError, match="window"):
        sb.export_prefix(1)
    with pytest.raises(ValueError, match="window"):
        sb.fork(0, 1)
    assert len(sb.export_prefix(1, sinks)) == 2 and full[0][0][0].shape[2] == cap


@pytest.mark.parametrize("window", [0, 60])
def test_many_seats(gpu, window):
    """Decode steps of many seats whose contexts are uneven, even, and uneven in another order, in one graph: against the
    oracle (without a window) and the same steps without graphs."""
    from m3x.serve.fast_backbone import StaticBackbone
    seats, cap = 30, 200
    geo = dict(layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, inter=768, seed=31, affine=synth.AFFINE)
    bbs = [StaticBackbone(synth.qwen3_backbone(device=gpu, **geo), seats + 1, capacity=cap, batch_buckets=(32,),
                          ctx_buckets=(cap,), page_size=PAGE, window=window, use_graphs=graphs) for graphs in (True, False)]
    g = torch.Generator().manual_seed(40)
    both = _oracle(synth.qwen3_backbone(device="cpu", **geo), seats + 1, 2, cap, 64)
    orders = set()
    for lengths in ([180 - 6 * s for s in range(seats)], [77] * seats, [0] * 20 + [150 + s for s in range(10)]):
        for s, n in enumerate(lengths):
            kv = [tuple(torch.randn(1, 2, n, 64, generator=g).to(torch.bfloat16) for _ in "kv") for _ in range(2)]
            for i, (k, v) in enumerate(kv):
                for o in both:
                    o[1][i][s, :, :n], o[2][i][s, :, :n] = k[0], v[0]
            for o in both:
                o[3][s] = n
            for sb in bbs:
                sb.load_prefix(s, [(k.to(gpu), v.to(gpu)) for k, v in kv], n)
        for n in (seats, seats, 26):
            x = torch.randn(n, 512, generator=g).to(torch.bfloat16)
            a, b = (sb.step(list(range(n)), x.to(gpu)) for sb in bbs)
            assert torch.equal(a, b)
            torch.cuda.synchronize()
            orders.add(bytes(bbs[0].graphs[(32, cap)].bufs.plan.launches[0][0].cpu().numpy()))
            if not window:
                ok, info = floor_check(a, *_step(both, list(range(n)), x))
                assert ok, (lengths, info)
    assert len(orders) >= (2 if window else 3)


def test_pool_exhausted(gpu):
    """A step that finds no page raises before it changes anything, and goes through once there is one."""
    sb, _ = _setup(gpu, prefix=[0, 16, 0, 0, 0, 0], pages=2)
    x = torch.randn(2, 1024, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(gpu)
    sb.step([0], x[:1])
    before = sb.export_prefix(1)
    with pytest.raises(RuntimeError, match="exhausted"):
        sb.step([0, 1], x)
    with pytest.raises(RuntimeError, match="exhausted"):
        sb.load_prefix(2, before, 16)
    with pytest.raises(RuntimeError, match="exhausted"):
        sb.prefill(3, x)
    with pytest.raises(RuntimeError, match="exhausted"):
        sb.fork(4, 0)  # one position: a page of its own
    sb.fork(5, 1)
    assert sb.lengths_cpu == [1, 16, 0, 0, 0, 16, 0] == sb.lengths.cpu().tolist()
    for a, b in zip(sb.export_prefix(1), before):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    sb.free(0)
    out = sb.step([1], x[1:])
    other, _ = _setup(gpu, prefix=[0, 16, 0, 0, 0, 0])
    assert torch.equal(out, other.step([1], x[1:]))


def test_frame_step(gpu):
    """FrameStep over a paged backbone: replays that cross pages give what the stages give one by one."""
    from m3x.cb0 import Cb0Sampler
    from m3x.frame import FrameStep
    from m3x.serve.fast_depth import FastDepth
    seen = []
    for use_graph in (True, False):
        sb, _ = _setup(gpu)
        bb = sb.backbone
        cb = Cb0Sampler(bb.cb0_head.weight, S, temp=0.9, top_k=50, rep=0.0)
        for s in range(S):
            cb.bind(s, seed=11 + s)
        fd = FastDepth(synth.swiglu_depth(seed=9, device=gpu, affine=synth.AFFINE), S, dtype=torch.bfloat16, temp=0.9,
                       top_k=50, batch_buckets=(4,), fused=True)
        fs = FrameStep(sb, cb, fd, ring_depth=4)
        fs.feedback.copy_(torch.randn(S + 1, 1024, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16))
        gr = fs.capture(4, CAP, use_graph=use_graph)
        fs.set_slots(gr, [2, 0, 3])
        for _ in range(4):
            fs.replay(gr)
            torch.cuda.synchronize()
        assert sb.pages.held(2) == 3
        seen.append((fs.codes(gr)[:3].clone(), gr["bufs"][0].out[:3].clone(), sb.lengths.clone()))
    for a, b in zip(*seen):
        assert torch.equal(a, b)


def test_frame_step_many_seats(gpu):
    """A captured frame step of seats of all ages, whose rows are attended longest first."""
    from m3x.cb0 import Cb0Sampler
    from m3x.frame import FrameStep
    from m3x.serve.fast_backbone import StaticBackbone
    from m3x.serve.fast_depth import FastDepth
    seats, lengths = 26, [(53 * s) % 220 for s in range(30)]
    seen = []
    for use_graph in (True, False):
        bb = synth.qwen3_backbone(layers=2, seed=21, device=gpu, affine=synth.AFFINE)
        sb = StaticBackbone(bb, 30, capacity=256, batch_buckets=(28,), ctx_buckets=(256,), page_size=PAGE)
        g = torch.Generator().manual_seed(50)
        for s, n in enumerate(lengths):
            sb.load_prefix(s, [tuple(torch.randn(1, 8, n, 128, generator=g).to(torch.bfloat16).to(gpu) for _ in "kv")
                               for _ in range(2)], n)
        cb = Cb0Sampler(bb.cb0_head.weight, 30, temp=0.9, top_k=50, rep=0.0)
        for s in range(30):
            cb.bind(s, seed=11 + s)
        fd = FastDepth(synth.swiglu_depth(seed=9, device=gpu, affine=synth.AFFINE), 30, dtype=torch.bfloat16, temp=0.9,
                       top_k=50, batch_buckets=(28,), fused=True)
        fs = FrameStep(sb, cb, fd, ring_depth=4)
        fs.feedback.copy_(torch.randn(31, 1024, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16))
        gr = fs.capture(28, 256, use_graph=use_graph)
        fs.set_slots(gr, list(range(3, 3 + seats)))
        for _ in range(3):
            fs.replay(gr)
            torch.cuda.synchronize()
        order = gr["bufs"][0].plan.launches[0][0][:seats, 0].tolist()
        assert order == sorted(range(seats), key=lambda r: -lengths[3 + r])
        seen.append((fs.codes(gr)[:seats].clone(), gr["bufs"][0].out[:seats].clone(), sb.lengths.clone()))
    for a, b in zip(*seen):
        assert torch.equal(a, b)


def test_refusals(gpu):
    from m3x.serve.fast_backbone import StaticBackbone
    bb = synth.qwen3_backbone(layers=1, device=gpu)
    for kw in (dict(page_size=24), dict(page_size=512), dict(page_size=16, kv_bits=4), dict(pages=4), dict(window=8),
               dict(page_size=16, sinks=4), dict(page_size=16, window=-1), dict(page_size=16, window=4, sinks=-1),
               dict(page_size=16, pages=0)):
        with pytest.raises(ValueError):
            StaticBackbone(bb, 2, **kw)
    sb, _ = _setup(gpu)
    with pytest.raises(ValueError):
        sb.load_prefix(0, [], CAP + 1)
    with pytest.raises(IndexError):
        sb.load_prefix(S, [], 0)
    with pytest.raises(ValueError):
        sb.export_prefix(1, 2)
    with pytest.raises(ValueError):
        sb.fork(0, 1, 2)
    with pytest.raises(IndexError):
        sb.fork(0, S)
    with pytest.raises(IndexError):
        sb.reserve([-1])
    with pytest.raises(ValueError):
        sb.reserve([0], CAP + 1)
    with pytest.raises(ValueError):
        sb.fork(1, 1)
    with pytest.raises(ValueError):
        sb.prefill(5, torch.zeros(CAP + 1, 1024, dtype=torch.bfloat16, device=gpu))
    assert sb.lengths_cpu[:S] == PREFIX
    with pytest.raises(ValueError, match="paged"):
        StaticBackbone(bb, 2, capacity=64, batch_buckets=(1,), ctx_buckets=(64,)).fork(0, 1)
