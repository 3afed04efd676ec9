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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,K", [(70, 160), (5000, 160), (4200, 1056), (9000, 1056)])
def test_rows_of_one_block(gpu, dtype, N, K):
    """1 to 16 rows through one, two and four tiles a workgroup: a row's bits do not depend on how many there are (so not
    on how x is read), and they are right."""
    from m3x import ops
    g = torch.Generator().manual_seed(N)
    x = torch.randn(16, K, generator=g).to(dtype).to(gpu)
    pg, pu = (ops.pack_weight4((torch.randn(N, K, generator=g) * K ** -0.5).to(dtype).to(gpu)) for _ in "gu")
    y, act = ops.linear4(x, pg), ops.linear4_act(x, pg, pu, ops.ACT_SWIGLU)
    for M in (1, 4, 5, 11, 12, 13, 15):
        assert torch.equal(ops.linear4(x[:M], pg), y[:M]) and torch.equal(
            ops.linear4_act(x[:M], pg, pu, ops.ACT_SWIGLU), act[:M]), M
    x64, h, tiny = x.cpu().double().numpy(), torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0
    a, b = (x64 @ R.weight_values(p.codes, p.scales, N, K).T for p in (pg, pu))
    da, db = ((K + 8) * 2.0 ** -24 * (np.abs(x64) @ np.abs(R.weight_values(p.codes, p.scales, N, K)).T) for p in (pg, pu))
    assert (np.abs(y.cpu().double().numpy() - a) <= da + h * (np.abs(a) + da) + tiny).all()
    silu = a / (1 + np.exp(-a))  # its slope is at most 1.13; the activation is within 2^-20 of its value
    off = 1.13 * da * (np.abs(b) + db) + np.abs(silu) * db + 2.0 ** -20 * np.abs(silu * b)
    assert (np.abs(act.cpu().double().numpy() - silu * b) <= off + h * (np.abs(silu * b) + off) + tiny).all()
