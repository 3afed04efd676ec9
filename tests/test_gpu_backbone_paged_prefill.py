"""StaticBackbone.prefill over a paged cache under a window: all of a long prompt or nothing of it."""
import pytest
import torch

from test_gpu_backbone_paged import _setup

pytestmark = pytest.mark.gpu


def test_windowed_prompt_in_pieces(gpu):
    """A prompt of three pieces whose second one the pool has no pages for: refused before the first, and right once a slot
    is freed."""
    x = (torch.randn(150, 1024, generator=torch.Generator().manual_seed(8)) * 0.5).to(torch.bfloat16).to(gpu)
    prefix = [0, 16, 0, 0, 0, 0]
    sb, other = (_setup(gpu, prefix=prefix, window=40, **kw)[0] for kw in (dict(pages=7), {}))
    for _ in range(2):
        with pytest.raises(RuntimeError, match="exhausted"):
            sb.prefill(3, x)
        assert sb.lengths_cpu == [0, 16, 0, 0, 0, 0, 0] == sb.lengths.tolist() and sb.pages.held(3) == 0
        assert sb.pages.free_pages == 6
    sb.free(1)
    other.free(1)
    assert torch.equal(sb.prefill(3, x), other.prefill(3, x)) and sb.lengths_cpu[3] == 150
    y = x[:1] * 2
    assert torch.equal(sb.step([3], y), other.step([3], y)) and sb.pages.held(3) == other.pages.held(3)
