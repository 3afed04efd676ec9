"""StaticBackbone(page_size=...) on the GPU: calls that find the pool too small leave everything as it was."""
import pytest
import torch

from test_gpu_backbone_paged import S, _setup

pytestmark = pytest.mark.gpu


def _state(sb):
    p = sb.pages
    return list(sb.lengths_cpu), sb.lengths.tolist(), p._host.tolist(), p._uses.tolist(), sorted(p._free)


def _same(a, b):
    assert len(a) == len(b)
    for (k0, v0), (k1, v1) in zip(a, b):
        assert torch.equal(k0, k1) and torch.equal(v0, v1)


def _x(n, seed):
    return torch.randn(n, 1024, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)


@pytest.mark.parametrize("call", ["load_prefix", "fork"])
def test_target_keeps_its_prefix(gpu, call):
    """A prefix or a fork that the pool has no pages for is refused, and the slot it was for holds what it held."""
    prefix = [40, 16, 33, 0, 0, 0]
    sb, other = _setup(gpu, prefix=prefix, pages=7)[0], _setup(gpu, prefix=prefix)[0]
    for o in (sb, other):
        o.fork(3, 1)
    before, held = _state(sb), [sb.export_prefix(s) for s in range(S)]
    assert sb.pages.free_pages == 0
    for _ in range(2):
        with pytest.raises(RuntimeError, match="exhausted"):
            if call == "fork":
                sb.fork(3, 0)  # two shared pages and one of its own
            else:
                sb.load_prefix(1, held[0], 40)
        assert _state(sb) == before
        for s in range(S):
            _same(sb.export_prefix(s), held[s])
    sb.free(2)
    other.free(2)
    x = _x(3, 5).to(gpu)
    assert torch.equal(sb.step([0, 1, 3], x), other.step([0, 1, 3], x))
    for o in (sb, other):
        o.free(1)
        o.free(3)  # four pages: the sequence in slot 0 holds three of the seven
        if call == "fork":
            o.fork(3, 0)
        else:
            o.load_prefix(1, held[0], 40)
    _same(sb.export_prefix(3 if call == "fork" else 1), other.export_prefix(3 if call == "fork" else 1))
    assert torch.equal(sb.pages.table.cpu(), torch.from_numpy(sb.pages._host))


def test_step_lets_go_of_nothing(gpu):
    """A step under a window that finds too few pages, even with those behind the windows, keeps those too."""
    sb = _setup(gpu, prefix=[100, 0, 0, 0, 0, 0], pages=8, window=40)[0]
    before, held = _state(sb), sb.export_prefix(0)
    for call in (lambda: sb.step(list(range(S)), _x(S, 6).to(gpu)), lambda: sb.reserve(list(range(S)))):
        with pytest.raises(RuntimeError, match="exhausted"):
            call()
        assert _state(sb) == before
        _same(sb.export_prefix(0), held)
    out = sb.step(list(range(5)), _x(5, 7).to(gpu))
    assert torch.equal(out, _setup(gpu, prefix=[100, 0, 0, 0, 0, 0], window=40)[0].step(list(range(5)), _x(5, 7).to(gpu)))
