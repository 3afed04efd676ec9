"""The paged cache's operators in 64 bits, and inputs for their tests."""
import math

import torch


def unit(dtype):
    """Half a step of a type, relative to the value."""
    return torch.finfo(dtype).eps / 2


def see(p, window, sinks):
    """Positions that a row at position p sees."""
    return [j for j in range(p + 1) if not window or j > p - window or j < sinks]


def rows_of(pool, table, slot, positions, page):
    """[n, kv, D] double numbers of a slot's positions (CPU tensors)."""
    ids = table[slot, positions // page].long()
    return pool[ids, :, positions % page].double()


def attention(q, k, v, table, slots, pos, scale, window=0, sinks=0, runs=None):
    """(out, bound) in 64 bits for CPU tensors: the result of every row of `runs` (all by default; NaN elsewhere), and
    how far a kernel may be from it. With u half a step of the type and A = sum w |v| / sum w: weights rounded once (u A
    in the numerator and in the sum each, a factor of 1 + 2 u for what both leave out), fp32 sums of n products (n 2^-24
    A), scores of D products off by D 2^-24 sum |q k| and their exponents by 2^-24 of themselves (weights by e - 1 of
    that, twice), fp16 weights below 2^-39 of the largest in all n lost, one rounding of the output."""
    rows, H, D = q.shape
    N, KV, P, _ = k.shape
    G, cap, u = H // KV, table.shape[1] * P, unit(q.dtype)
    out = torch.full((rows, H, D), float("nan"), dtype=torch.float64)
    bound = torch.zeros_like(out)
    for first, n, _ in runs if runs is not None else [(r, 1, 0) for r in range(rows)]:
        for r in range(first, first + n):
            slot, p = int(slots[first]), int(pos[first]) + r - first
            keys = torch.tensor([j for j in see(p, window, sinks) if j < cap], dtype=torch.long)
            if 0 <= slot < table.shape[0] and len(keys):
                ids = table[slot, keys // P]
                keys = keys[(ids >= 0) & (ids < N)]
            if not 0 <= slot < table.shape[0] or not len(keys):
                out[r] = 0
                continue
            kk, vv = (rows_of(x, table, slot, keys, P).repeat_interleave(G, 1) for x in (k, v))  # [n, H, D]
            x = q[r].double()
            s = torch.einsum("hd,nhd->hn", x, kk) * scale
            size = (torch.einsum("hd,nhd->hn", x.abs(), kk.abs()) * abs(scale)).amax(-1)
            w = torch.softmax(s, -1)
            out[r] = torch.einsum("hn,nhd->hd", w, vv)
            A = torch.einsum("hn,nhd->hd", w, vv.abs())
            score = torch.expm1((D + 8) * 2.0 ** -24 * size)[:, None]
            bound[r] = (2 * u * (1 + 4 * u) + 2 * len(keys) * 2.0 ** -24 + 4 * score + 2.0 ** -20) * A \
                + len(keys) * 2.0 ** -38 * vv.abs().amax(0) + u * out[r].abs() * (1 + 4 * u) + 2.0 ** -24
    return out, bound


def rotate(x, pos, inv_freq, interleaved, factor, w, eps):
    """[rows, heads, D] double: normed by w (None: not), rotated."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    angle = torch.outer(pos.clamp_min(0).double(), inv_freq.double())
    c, s = (t[:, None] * factor for t in (angle.cos(), angle.sin()))
    n = 2 * inv_freq.numel()
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., :n // 2], x[..., n // 2:n])
    y = x.clone()
    ra, rb = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:n:2], y[..., 1:n:2] = ra, rb
    else:
        y[..., :n // 2], y[..., n // 2:n] = ra, rb
    return y


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def table_for(held, slots, page, width, seed, spare=3):
    """(table, pages) where slot s holds the positions of the spans held[s], pages in no order, -1 elsewhere."""
    table = torch.full((slots, width), -1, dtype=torch.int32)
    n = 0
    for s, spans in held.items():
        for first, end in spans:
            for b in range(first // page, -(-end // page)):
                if table[s, b] < 0:
                    table[s, b] = n
                    n += 1
    order = torch.randperm(n + spare, generator=torch.Generator().manual_seed(seed)).int()
    return torch.where(table >= 0, order[table.clamp_min(0).long()], table), n + spare


def pools(table, pages, held, KV, page, D, dtype, seed, stale=float("nan")):
    """Pools that hold numbers at the held positions and `stale` everywhere else."""
    k, v = (torch.full((pages, KV, page, D), stale, dtype=dtype) for _ in "kv")
    for s, spans in held.items():
        for i, (first, end) in enumerate(spans):
            at = torch.arange(first, end)
            for x, y in ((k, 2 * s + 1000 * i), (v, 2 * s + 1 + 1000 * i)):
                x[table[s, at // page].long(), :, at % page] = normal(seed * 77 + y, end - first, KV, D).to(dtype)
    return k, v


def within(got, want, bound):
    """Largest error over its bound (NaN where the result is no number counts as infinite)."""
    got = got.detach().cpu().double()
    off = (got - want).abs()
    ok = torch.isfinite(got) | ~torch.isfinite(want)
    if not ok.all():
        return math.inf
    return (off / bound.clamp_min(1e-300)).nan_to_num(0.0, 0.0).max().item() if off.numel() else 0.0
