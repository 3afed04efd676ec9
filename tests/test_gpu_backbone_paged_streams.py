"""StaticBackbone(page_size=...) on several streams: a call waits for the one before it, whichever slots they are of, since
they share the table, a workspace and pages that go from one slot to another."""
import pytest
import torch

from test_gpu_backbone_paged import PAGE, _setup
from m3x import synth

pytestmark = pytest.mark.gpu


def _x(n, seed):
    return torch.randn(n, 1024, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


@pytest.fixture
def busy(gpu):
    """Some ten milliseconds of work on the current stream."""
    a = torch.randn(8192, 8192, dtype=torch.bfloat16, device=gpu)
    out = torch.empty_like(a)

    def run():
        for _ in range(20):
            torch.mm(a, a, out=out)
    run()
    torch.cuda.synchronize()
    return run


def test_calls_follow_each_other(gpu, busy):
    """Each kind of call behind a step on another stream that has work before it."""
    sb = _setup(gpu, prefix=[40, 33, 200, 10, 0, 0])[0]
    x, p = _x(2, 1).to(gpu), _x(20, 2).to(gpu)
    sb.step([0, 1], x)
    sb.step_mixed([0], x[:1], [(4, p)])
    kv = sb.export_prefix(2)
    torch.cuda.synchronize()
    first, second = torch.cuda.Stream(), torch.cuda.Stream()
    for i, call in enumerate((lambda: sb.step([2, 3], x), lambda: sb.step_mixed([2], x[:1], [(3, p)]), lambda: sb.prefill(3, p),
                 lambda: sb.load_prefix(5, kv, 200), lambda: sb.fork(5, 2), lambda: sb.export_prefix(2), lambda: sb.free(5),
                 lambda: sb.reserve([2]), lambda: sb.make_buffers(4, 512))):
        with torch.cuda.stream(first):
            busy()
            sb.step([0, 1], x)
        with torch.cuda.stream(second):
            call()
        second.synchronize()
        assert first.query(), i
        torch.cuda.synchronize()


def test_pages_change_hands(gpu, busy):
    """Two streams' steps in turn, under a window whose pages go from slot to slot, and of prompts whose splits use the
    workspace: the results of one stream."""
    out = []
    for streams in ([torch.cuda.Stream(), torch.cuda.Stream()], [torch.cuda.current_stream()] * 2):
        sb = _setup(gpu, prefix=[100, 90, 300, 260, 0, 0], window=64, sinks=4, pages=50)[0]
        torch.cuda.synchronize()
        got = []
        for t in range(12):
            for i, s in enumerate(streams):
                with torch.cuda.stream(s):
                    if i == 0 and t % 4 == 0 and len({id(x) for x in streams}) == 2:
                        busy()
                    x = _x(22, 100 * t + i).to(gpu)
                    got.append(sb.step([2 * i, 2 * i + 1], x[:2]))
                    d, last = sb.step_mixed([2 * i], x[:1], [(2 * i + 1, x[2:])])
                    got += [d, last[0]]
        torch.cuda.synchronize()
        out.append(torch.cat([g.view(-1, 1024) for g in got]))
    assert torch.equal(*out)


def test_frame_beside_steps(gpu, busy):
    """A captured frame on one stream, prefills of other slots on another: as on one stream."""
    from m3x.cb0 import Cb0Sampler
    from m3x.frame import FrameStep
    from m3x.serve.fast_depth import FastDepth
    out = []
    for two in (True, False):
        sb = _setup(gpu, prefix=[40, 33, 200, 10, 0, 0])[0]
        cb = Cb0Sampler(sb.backbone.cb0_head.weight, 6, temp=0.9, top_k=50, rep=0.0)
        for s in range(6):
            cb.bind(s, seed=11 + s)
        fd = FastDepth(synth.swiglu_depth(seed=9, device=gpu, affine=synth.AFFINE), 6, dtype=torch.bfloat16, temp=0.9,
                       top_k=50, batch_buckets=(4,), fused=True)
        fs = FrameStep(sb, cb, fd, ring_depth=4)
        fs.feedback.copy_(torch.randn(7, 1024, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16))
        gr = fs.capture(4, 512)
        fs.set_slots(gr, [2, 0, 3])
        sb.prefill(4, _x(5, 3).to(gpu))
        torch.cuda.synchronize()
        frames, prompts = [torch.cuda.Stream() for _ in range(2)] if two else [torch.cuda.current_stream()] * 2
        got = []
        for t in range(6):
            with torch.cuda.stream(frames):
                if two and t % 2 == 0:
                    busy()
                fs.replay(gr)
                got.append(gr["bufs"][0].out[:3].clone())
            with torch.cuda.stream(prompts):
                got.append(sb.prefill(4 + t % 2, _x(3 * PAGE + t, 30 + t).to(gpu))[None])
        torch.cuda.synchronize()
        out.append(torch.cat(got))
    assert torch.equal(*out)
