"""Rows at positions past the table's end, under a window: they see those of the first tokens and of their window that
exist, in either kernel, split or not."""
import pytest
import torch

import paged_reference as R
from test_gpu_paged import BF, FP, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,width,window,sinks,n,p0", [
    (64, 16, 512, 16, 68, 1981), (16, 4, 20, 5, 80, 140), (16, 64, 16, 100, 90, 5000), (64, 16, 512, 300, 300, 1400),
    (32, 8, 64, 40, 200, 226), (16, 16, 100, 1, 90, 270), (16, 16, 100, 256, 90, 270), (16, 8, 50, 1000, 70, 700),
    (16, 4, 20, 5, 1, 140), (16, 4, 20, 5, 3, 82), (16, 4, 20, 0, 80, 140), (32, 8, 0, 0, 90, 400)])
@pytest.mark.parametrize("D,dtype", [(128, BF), (64, FP)])
def test_past_the_end(gpu, page, width, window, sinks, n, p0, D, dtype):
    cap = page * width
    held = {1: [(0, cap)]}
    table, pages = R.table_for(held, 3, page, width, 3)
    k, v = R.pools(table, pages, held, 2, page, D, dtype, 4)
    q = R.normal(5, n, 8, D).to(dtype)
    slots, pos = torch.ones(n, dtype=torch.long), torch.arange(p0, p0 + n, dtype=torch.int32)
    laid = [(0, n, p0)]
    want, bound = R.attention(q, k, v, table, slots, pos, 0.1, window, sinks, laid)
    assert window == 0 or (want[-1] == 0).all() == (sinks == 0)
    for cut in (True, False):
        for splits in (1, 2, 5):
            got = _run(gpu, q, k, v, table, slots, pos, laid, 0.1, window, sinks, splits=splits, cut=cut)
            worst = R.within(got, want, bound)
            assert worst <= 1, (cut, splits, worst)
