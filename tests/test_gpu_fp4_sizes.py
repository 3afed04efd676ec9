"""The 4-bit weights at many rows and inputs."""
import numpy as np
import pytest
import torch

import fp4_reference as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,K", [(1048592, 32), (1100003, 64), (3, 262176)])
def test_pack_and_multiply_many(gpu, N, K):
    """Past 65535 tiles of rows, or 2048 steps: packed bytes and products at both ends, and at the tiles around 65535."""
    from m3x import ops
    g = torch.Generator().manual_seed(N % 1000)
    w = torch.randn(N, K, generator=g).bfloat16()
    p = ops.pack_weight4(w.to(gpu))
    x = torch.randn(2, K, generator=g).bfloat16()
    y = ops.linear4(x.to(gpu), p).cpu().double().numpy()
    for a in sorted({0, max(0, min(65535 * 16 - 32, N - 64) // 16 * 16), max(0, N - 40) // 16 * 16}):
        b = min(N, a + 64)
        t = slice(a // 16, -(-b // 16))
        got = R.weight_values(p.codes[t], p.scales[t], b - a, K)
        assert np.array_equal(got, R.quantise(w[a:b].double().numpy(), 252)[0])
        want = x.double().numpy() @ got.T
        off = (K + 8) * 2.0 ** -24 * (np.abs(x.double().numpy()) @ np.abs(got).T)  # K products summed in fp32, any order
        assert (np.abs(y[:, a:b] - want) <= off + 2.0 ** -8 * (np.abs(want) + off)).all(), a
