"""What a paged StaticBackbone holds besides its pages."""
import pytest
import torch

from m3x import synth

pytestmark = pytest.mark.gpu


def test_nothing_by_capacity(gpu):
    """Positions cost a table entry a page and slot: no table of angles (a million of them would be 512 MB here)."""
    from m3x.serve.fast_backbone import StaticBackbone
    bb = synth.qwen3_backbone(device=gpu, layers=1, hidden=512, heads=4, kv_heads=1, head_dim=128, inter=768, seed=31,
                              affine=synth.AFFINE)
    held = []
    for cap in (1 << 10, 1 << 20):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        sb = StaticBackbone(bb, 2, capacity=cap, batch_buckets=(2,), ctx_buckets=(512,), page_size=256, pages=4,
                            use_graphs=False)
        held.append((torch.cuda.memory_allocated() - before, torch.cuda.max_memory_allocated() - before))
        x = torch.randn(2, 512, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(gpu)
        out = sb.step([0, 1], x)
        assert torch.isfinite(out).all() and sb.lengths_cpu == [1, 1, 0]
        del sb, out
    entries = 3 * (1 << 20) // 256 * 4  # the table's
    assert all(b - a <= entries + (1 << 16) for a, b in zip(*held)), held
