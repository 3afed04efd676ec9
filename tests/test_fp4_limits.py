"""Arguments at the ends of what the 4-bit entry points take, on the CPU: refused before a launch, or computed on the
host."""
import ctypes
import math

import pytest
import torch

P = ctypes.c_void_p(4096)  # never read: every call below is refused


def _cache(cap=64, D=128):
    from m3x import ops
    return ops.Kv4Cache.empty(2, 2, cap, D, "cpu")


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 2.0 ** 127 * 1.0001, -3e38, 1e300])
def test_attn_scale_refused(scale):
    """A scale whose factor of the exponents is not finite."""
    from m3x import ops
    from m3x._lib import lib
    c = _cache()
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    at = torch.zeros(3, dtype=torch.long), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="scale"):
        ops.kv4_attn(q, c, q, *at, scale, 64, 128, None)
    a = ops.Kv4CacheArgs(4096, 4096, 4096, 4096, 1, 2, 128, 64)
    assert lib().m3x_kv4_attn(ctypes.addressof(a), P, 512, 128, P, 512, 128, P, P, scale, 1, 4, 64, 128, None, 0, 0,
                              None) == -1


@pytest.mark.parametrize("rows,heads,kv_heads,max_ctx", [(65536, 16, 8, 1 << 20), (100000, 16, 8, 1 << 20),
                                                         (1 << 20, 64, 64, 1 << 30), (224, 16, 8, 2049), (1, 16, 8, 1 << 30)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attn_chunk_within_the_context(rows, heads, kv_heads, max_ctx, dim):
    """The split rule stays within the context (and so within an int) at any count that attention takes, and the
    workspace of its splits is what they need."""
    from m3x import ops
    chunk = ops.kv4_attn_chunk(rows, heads, kv_heads, max_ctx, dim)
    assert 128 <= chunk < max_ctx + 128 and chunk % 128 == 0
    splits = -(-max_ctx // chunk)
    want = rows * heads * splits * (dim + 2) * 4 if splits > 1 else 0
    assert ops.kv4_attn_workspace(rows, heads, dim, max_ctx, chunk) == want


def test_attn_chunk_past_an_int():
    """A chunk that an int does not hold is refused, not wrapped."""
    from m3x import ops
    c = _cache()
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    at = torch.zeros(3, dtype=torch.long), torch.zeros(3, dtype=torch.int32)
    for chunk in (1 << 31, 1 << 32, (1 << 32) + 128):
        with pytest.raises(ValueError, match="chunk"):
            ops.kv4_attn(q, c, q, *at, 1.0, 64, chunk, None)
        with pytest.raises(ValueError):
            ops.kv4_attn_workspace(3, 4, 128, 1 << 20, chunk)


def test_pack_sizes_refused():
    from m3x import ops
    from m3x._lib import lib
    for N, K in ((1 << 30, 32), (1 << 26, 2048), ((1 << 20) - 15, 128 << 10)):
        assert lib().m3x_pack_weight4(P, 32, N, K, P, P, 0, None) == -1
        with pytest.raises(ValueError, match="fewer than"):
            ops.pack_weight4(torch.zeros(1, K, dtype=torch.bfloat16).expand(N, K))
