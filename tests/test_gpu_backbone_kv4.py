"""StaticBackbone(kv_bits=4) on the GPU against the eager oracle whose caches quantise what is written to them: decode,
inline prefill, prefix export and install, graphs, one-row steps, and a captured frame step."""
import pytest
import torch

import fp4_reference as R
from helpers import convert, floor_check, report
from m3x import synth
from oracle import torch_oracle as O

pytestmark = pytest.mark.gpu

LAYERS, S, CAP = 3, 6, 512
PREFIX = [0, 1, 37, 200, 300, 0]


class Q4:
    """A cache tensor of the oracle that holds the 4-bit format's values of what is written to it."""

    def __init__(self, t):
        self.t = t

    def __setitem__(self, at, x):
        self.t[at] = torch.from_numpy(R.quantise(x.double().numpy(), 252)[0]).to(self.t.dtype)

    def __getitem__(self, at):
        return self.t[at]


def _setup(gpu, use_graphs=True, **kw):
    from m3x.serve.fast_backbone import StaticBackbone
    bb_g = synth.qwen3_backbone(layers=LAYERS, seed=21, device=gpu, affine=synth.AFFINE)
    bb_c = synth.qwen3_backbone(layers=LAYERS, seed=21, device="cpu", affine=synth.AFFINE)
    sb = StaticBackbone(bb_g, S, capacity=CAP, batch_buckets=(1, 2, 4, 8, 64), ctx_buckets=(256, 512),
                        use_graphs=use_graphs, kv_bits=4, **kw)
    g = torch.Generator().manual_seed(22)
    kc, vc = ([Q4(torch.zeros(S + 1, 8, CAP, 128, dtype=torch.bfloat16)) for _ in range(LAYERS)] for _ in "kv")
    for s, n in enumerate(PREFIX):
        kv = []
        for i in range(LAYERS):
            k, v = (torch.randn(1, 8, n, 128, generator=g).to(torch.bfloat16) for _ in "kv")
            if n:
                kc[i][s, :, :n], vc[i][s, :, :n] = k[0], v[0]
            kv.append((k.to(gpu), v.to(gpu)))
        sb.load_prefix(s, kv, n)
    lengths = torch.tensor(PREFIX + [0])
    cos, sin = O.rope_tables(128, 1e6, CAP, torch.bfloat16)
    truth = dict(bb=convert(bb_c, torch.float32), kc=[Q4(t.t.float()) for t in kc], vc=[Q4(t.t.float()) for t in vc],
                 lengths=lengths.clone(), cos=cos.float(), sin=sin.float())
    return sb, bb_c, kc, vc, lengths, cos, sin, truth


def _both(setup, slots, x, offset=None):
    sb, bb_c, kc, vc, lengths, cos, sin, T = setup
    slots = torch.tensor(slots)
    return (O.backbone_step(bb_c, kc, vc, lengths, slots, x, cos, sin, offset=offset),
            O.backbone_step(T["bb"], T["kc"], T["vc"], T["lengths"], slots, x.float(), T["cos"], T["sin"],
                            offset=offset))


def test_install_and_export(gpu):
    """What a slot holds is the format's values of what was installed, and an exported prefix installs as itself."""
    sb, _, kc, vc, *_ = _setup(gpu)
    assert sb.k == [] and sb.v == [] and len(sb.kv4) == LAYERS
    assert sb.memory_bytes() == LAYERS * (S + 1) * 8 * CAP * (128 + 8)
    for s, n in enumerate(PREFIX):
        kv = sb.export_prefix(s)
        for i, (k, v) in enumerate(kv):
            assert tuple(k.shape) == (1, 8, n, 128)
            assert torch.equal(k[0].cpu(), kc[i][s, :, :n]) and torch.equal(v[0].cpu(), vc[i][s, :, :n])
    kv = sb.export_prefix(4)
    sb.load_prefix(5, kv, 300)
    for a, b in zip(sb.export_prefix(5), kv):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    y = torch.randn(1, 1024, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(gpu)
    out = sb.step([4, 5], torch.cat([y, y]))
    assert torch.equal(out[0], out[1])
    sb.load_prefix(0, [(k[:, :, :0], v[:, :, :0]) for k, v in kv], 0)
    assert sb.lengths_cpu[0] == 0


def test_step_matches_oracle(gpu):
    """Decode steps of four seats and of one (no persistent run with a 4-bit cache), lengths advanced."""
    st = _setup(gpu)
    sb, lengths = st[0], st[4]
    g = torch.Generator().manual_seed(23)
    for t, slots in enumerate(([0, 2, 3, 4], [0, 2, 3, 4], [3], [4, 1])):
        x = torch.randn(len(slots), 1024, generator=g).to(torch.bfloat16)
        out = sb.step(slots, x.to(gpu))
        ok, info = floor_check(out, *_both(st, slots, x))
        report(f"kv4 step {t}", info)
        assert ok, (t, info)
    assert sb.lengths.cpu().tolist() == lengths.tolist() == sb.lengths_cpu and not sb._persistent_ok(1)


def test_mixed_and_prefill(gpu):
    """Decoding seats with two inline prefills in one step, then a prompt in pieces of the largest bucket."""
    st = _setup(gpu)
    sb = st[0]
    g = torch.Generator().manual_seed(24)
    x = torch.randn(2, 1024, generator=g).to(torch.bfloat16)
    p5, p1 = ((torch.randn(n, 1024, generator=g) * 0.5).to(torch.bfloat16) for n in (20, 7))
    dec, last = sb.step_mixed([0, 3], x.to(gpu), [(5, p5.to(gpu)), (1, p1.to(gpu))])
    ref, truth = _both(st, [0, 3] + [5] * 20 + [1] * 7, torch.cat([x, p5, p1]),
                       torch.tensor([0, 0] + list(range(20)) + list(range(7))))
    ok, info = floor_check(torch.cat([dec, torch.stack(last)]), ref[[0, 1, 21, 28]], truth[[0, 1, 21, 28]])
    assert ok, info
    p = (torch.randn(100, 1024, generator=g) * 0.5).to(torch.bfloat16)
    got = sb.prefill(2, p.to(gpu))
    ref, truth = _both(st, [2] * 100, p, torch.arange(100))
    ok, info = floor_check(got[None], ref[-1:], truth[-1:])
    assert ok, info
    assert sb.lengths_cpu[:S] == [1, 8, 137, 201, 300, 20]
    assert {k for k in sb.graphs} <= {(r, c) for r in (1, 2, 4, 8, 64) for c in (256, 512)}  # one graph a bucket


def test_graph_replay_equals_eager(gpu):
    a, b = _setup(gpu, use_graphs=True)[0], _setup(gpu, use_graphs=False)[0]
    a.warmup()
    g = torch.Generator().manual_seed(25)
    for slots in ([0, 2, 3, 4], [0, 2, 3, 4], [1], [4, 0]):
        x = torch.randn(len(slots), 1024, generator=g).to(torch.bfloat16).to(gpu)
        assert torch.equal(a.step(slots, x), b.step(slots, x))
        torch.cuda.synchronize()
    for s in range(S):
        for (k0, v0), (k1, v1) in zip(a.export_prefix(s), b.export_prefix(s)):
            assert torch.equal(k0, k1) and torch.equal(v0, v1)


def test_frame_step(gpu):
    """FrameStep over a 4-bit backbone: replays give what the stages give one by one."""
    from m3x.cb0 import Cb0Sampler
    from m3x.frame import FrameStep
    from m3x.serve.fast_depth import FastDepth
    seen = []
    for use_graph in (True, False):
        sb = _setup(gpu)[0]
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
        for _ in range(3):
            fs.replay(gr)
            torch.cuda.synchronize()
        seen.append((fs.codes(gr)[:3].clone(), gr["bufs"][0].out[:3].clone(), sb.lengths.clone()))
    for a, b in zip(*seen):
        assert torch.equal(a, b)


def test_refusals(gpu):
    from m3x.serve.fast_backbone import StaticBackbone
    bb = synth.qwen3_backbone(layers=1, device=gpu)
    for bits in (8, 2, None):
        with pytest.raises(ValueError):
            StaticBackbone(bb, 2, kv_bits=bits)
    sb = _setup(gpu)[0]
    with pytest.raises(ValueError):
        sb.load_prefix(0, [], CAP + 1)
    with pytest.raises(IndexError):
        sb.load_prefix(S, [], 0)
    with pytest.raises(ValueError):
        sb.export_prefix(1, 2)
    with pytest.raises(ValueError):
        sb.prefill(5, torch.zeros(CAP + 1, 1024, dtype=torch.bfloat16, device=gpu))


def test_other_geometry(gpu):
    """Eight query heads of 64 over two kv heads at a width without folded norms: decode, prefill and a graph's replay."""
    from m3x.serve.fast_backbone import StaticBackbone
    geo = dict(layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, inter=768, seed=31, affine=synth.AFFINE)
    bb_c = synth.qwen3_backbone(device="cpu", **geo)
    sb = StaticBackbone(synth.qwen3_backbone(device=gpu, **geo), 3, capacity=200, batch_buckets=(2, 32),
                        ctx_buckets=(200,), kv_bits=4)
    assert not sb.fused_norms and sb.kv4[0].cap == 224
    cos, sin = O.rope_tables(64, 1e6, 224, torch.bfloat16)
    new = lambda dt: [Q4(torch.zeros(4, 2, 200, 64, dtype=dt)) for _ in range(2)]  # noqa: E731
    st = (sb, bb_c, new(torch.bfloat16), new(torch.bfloat16), torch.zeros(4, dtype=torch.long), cos, sin,
          dict(bb=convert(bb_c, torch.float32), kc=new(torch.float32), vc=new(torch.float32),
               lengths=torch.zeros(4, dtype=torch.long), cos=cos.float(), sin=sin.float()))
    g = torch.Generator().manual_seed(32)
    p = (torch.randn(30, 512, generator=g) * 0.5).to(torch.bfloat16)
    got = sb.prefill(1, p.to(gpu))
    ref, truth = _both(st, [1] * 30, p, torch.arange(30))
    ok, info = floor_check(got[None], ref[-1:], truth[-1:])
    assert ok, info
    for _ in range(3):
        x = torch.randn(2, 512, generator=g).to(torch.bfloat16)
        ok, info = floor_check(sb.step([1, 2], x.to(gpu)), *_both(st, [1, 2], x))
        assert ok, info
    assert sb.lengths_cpu[:3] == [0, 33, 3]
