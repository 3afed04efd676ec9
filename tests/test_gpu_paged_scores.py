"""Scores of any finite size over the paged cache: the weights go by differences of scores, so that rows whose scores are
large come out as rows of small ones do, in either kernel, split or not."""
import pytest
import torch

import paged_reference as R
from test_gpu_paged import BF, FP, _case, _run

pytestmark = pytest.mark.gpu


def _one_hot(v, dtype):
    """How far a mean of values may be from v where all of the weight lies on keys of one score: their weights are one power
    of two, exact in the sums, so that half a step of the type is left, and the fp32 chain."""
    return (R.unit(dtype) + 2.0 ** -20) * v.abs() + 2.0 ** -24


def _put(pool, table, slot, page, j, x):
    pool[table[slot, j // page].long(), :, j % page] = x


SIZES = [(FP, 128, 2000.0, 2000.0), (FP, 128, 8000.0, 8000.0), (FP, 128, 30000.0, 22496.0), (FP, 64, 65504.0, 65504.0),
         (BF, 64, 33024.0, 33024.0), (BF, 128, 1e9, 3e7), (BF, 128, 2.0 ** 60, 2.0 ** 60), (BF, 64, 300.0, 250.0)]


@pytest.mark.parametrize("dtype,D,q0,k0", SIZES)
@pytest.mark.parametrize("n", [1, 3, 70])
@pytest.mark.parametrize("splits", [1, 3])
def test_large_scores(gpu, dtype, D, q0, k0, n, splits):
    """All of the weight on the best key, wherever it lies, and shared evenly by keys of the same score in several waves,
    groups of waves and splits; the other keys' scores small, or larger ones of the other sign."""
    page, p0 = 32, 600
    q, k, v, table, slots, pos, laid = _case([(n, p0)], 4, 2, D, page, dtype, seed=12)
    q[:] = q0
    for best in ([3], [599], [200], [10, 170, 171, 290, 598]):
        for others, at in ((None, k0), (-k0, k0 / 2), (-k0, -k0 / 2)):
            k1 = k.clone()
            if others is not None:
                k1 = torch.where(torch.isfinite(k1), torch.full_like(k1, others), k1)
            for j in best:
                _put(k1, table, 1, page, j, at)
            want = R.rows_of(v, table, 1, torch.tensor(best), page).mean(0).repeat_interleave(2, 0).expand(n, 4, D)
            size = R.rows_of(v.abs(), table, 1, torch.tensor(best), page).mean(0).repeat_interleave(2, 0).expand(n, 4, D)
            for cut in (True, False):
                got = _run(gpu, q, k1, v, table, slots, pos, laid, D ** -0.5, splits=splits, cut=cut)
                worst = R.within(got, want, _one_hot(size, dtype))
                assert worst <= 1, (best, others, cut, worst)
                got = _run(gpu, -q, k1, v, table, slots, pos, laid, -D ** -0.5, splits=splits, cut=cut)
                assert R.within(got, want, _one_hot(size, dtype)) <= 1


@pytest.mark.parametrize("dtype,D", [(FP, 128), (BF, 128), (FP, 64), (BF, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (64, 8)])
@pytest.mark.parametrize("best", [5, 205, 250])
@pytest.mark.parametrize("splits", [1, 2])
def test_large_beside_small(gpu, dtype, D, window, sinks, best, splits):
    """Heads of large scores beside heads of ordinary ones in the same tiles, rows that do not see the best key, and rows
    that see nothing: each row is right by itself."""
    page, runs = 32, [(1, 300), (3, 297), (70, 250), (40, -3), (1, -1), (130, 180)]
    q, k, v, table, slots, pos, laid = _case(runs, 8, 2, D, page, dtype, window, sinks, seed=13)
    q0, k0 = (65504.0, 60000.0) if dtype == FP else (3e6, 1e9)
    q[:, :, 0] = 0
    q[:, 1::3] = 0
    q[:, 1::3, 0] = q0
    for s, (n, p) in enumerate(runs):
        if best < p + n and (not window or table[s + 1, best // page] >= 0):
            _put(k, table, s + 1, page, best, k[table[s + 1, best // page].long(), :, best % page].clone())
            k[table[s + 1, best // page].long(), :, best % page, 0] = k0
    want, bound = R.attention(q, k, v, table, slots, pos, 0.1, window, sinks, laid)
    for a, n, p in laid:
        for r in range(n):
            if best in R.see(p + r, window, sinks):
                bound[a + r, 1::3] = _one_hot(want[a + r, 1::3], dtype)
    assert torch.isfinite(bound).all()
    for cut in (True, False):
        got = _run(gpu, q, k, v, table, slots, pos, laid, 0.1, window, sinks, splits=splits, cut=cut)
        worst = R.within(got, want, bound)
        assert worst <= 1, (cut, worst)


@pytest.mark.parametrize("scale", [2.0 ** -120, -2.0 ** -125, 2.0 ** -128, -2.0 ** -131, 1e-45, 0.0])
@pytest.mark.parametrize("n", [1, 3, 70])
def test_small_scales(gpu, scale, n):
    """Scores up to 2^126 under scales down to fp32's smallest."""
    q, k, v, table, slots, pos, laid = _case([(n, 400)], 4, 2, 128, 32, BF, seed=14)
    q[:] = 2.0 ** 59
    k = k.clamp(-2, 2) / 2 * 2.0 ** 59  # (NaN where nothing is held)
    k[..., 8:] = k[..., :1]
    want, bound = R.attention(q, k, v, table, slots, pos, scale, runs=laid)
    for cut in (True, False):
        worst = R.within(_run(gpu, q, k, v, table, slots, pos, laid, scale, splits=2, cut=cut), want, bound)
        assert worst <= 1, (cut, worst)


@pytest.mark.parametrize("dtype,D", [(FP, 128), (BF, 64)])
@pytest.mark.parametrize("splits", [1, 4])
def test_many_workgroups(gpu, dtype, D, splits):
    """The same in a prompt of more workgroups than there are CUs, whose keys one group of waves has to itself: sums whose
    references differ from split to split, by more and less than what one multiply-add a weight bears."""
    page, n, p0 = 64, 320, 400
    q0, k0 = (60000.0, 50000.0) if dtype == FP else (3e6, 1e9)
    q, k, v, table, slots, pos, laid = _case([(n, p0)], 32, 8, D, page, dtype, seed=15)
    q[:, :, 0] = 0
    q[:, 1::3] = 0
    q[:, 1::3, 0] = q0
    q[:, 2::3] *= 40  # scores of some hundreds
    for best in ([7], [395], [7, 200, 395]):
        k1 = k.clone()
        for j in best:
            k1[table[1, j // page].long(), :, j % page, 0] = k0
        want, bound = R.attention(q, k1, v, table, slots, pos, 0.1, runs=laid)
        size = R.rows_of(v.abs(), table, 1, torch.tensor(best), page).mean(0).repeat_interleave(4, 0)
        bound[:, 1::3] = _one_hot(size, dtype)[None, 1::3].expand(n, -1, -1)
        got = _run(gpu, q, k1, v, table, slots, pos, laid, 0.1, splits=splits, cut=False)
        worst = R.within(got, want, bound)
        assert worst <= 1, (best, worst)
