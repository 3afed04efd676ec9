"""Tensor-level wrappers over the m3x C ABI (include/m3x.h).

Each wrapper checks devices, dtypes and shapes (ValueError, like the reference surfaces), passes raw pointers,
element strides and torch's current HIP stream, and raises RuntimeError on a non-zero status. Nothing here
allocates on the device except where a function documents that it returns a new tensor; graph-captured code
passes preallocated outputs and workspaces.
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

import torch

from ._lib import check, lib

NORM_LAYER, NORM_RMS = 0, 1
ACT_NONE, ACT_SWIGLU, ACT_GELU = -1, 0, 1
_DT = {torch.bfloat16: 0, torch.float16: 1}
_DT_ANY = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _dt(t: torch.Tensor) -> int:
    if t.dtype not in _DT:
        raise ValueError(f"m3x kernels take bfloat16 or float16 tensors, got {t.dtype}")
    return _DT[t.dtype]


def _dt3(t: torch.Tensor) -> int:
    """dtype code for the entry points that also have an fp32 instance (projections, depth norms / attention /
    sampler / feedback, and the codec's kernels)."""
    if t.dtype not in _DT_ANY:
        raise ValueError(f"m3x kernels take bfloat16, float16 or float32 tensors, got {t.dtype}")
    return _DT_ANY[t.dtype]


def _dev(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("m3x kernels take device tensors")


def _rows2d(t: torch.Tensor, name: str):
    if t.dim() != 2 or t.stride(-1) != 1:
        raise ValueError(f"{name} must be a 2-D tensor with a contiguous last dimension, got {tuple(t.shape)}")


def _need(t: torch.Tensor, dtype, name: str):
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")


def _index(slots=None, pos=None):
    """The ABI's index types: slot tensors are int64, position tensors int32 (a wrong width would be read as
    out-of-range indices on the device)."""
    if slots is not None:
        _need(slots, torch.long, "slots")
    if pos is not None:
        _need(pos, torch.int32, "pos")


# ---------------------------------------------------------------- backbone step
def positions(lengths, slots, offset, pos):
    _dev(lengths, slots, offset, pos)
    _need(lengths, torch.long, "lengths")
    _need(slots, torch.long, "slots")
    _need(pos, torch.int32, "pos")
    if offset is not None:
        _need(offset, torch.long, "offset")
    check(lib().m3x_positions(_p(lengths), _p(slots), _p(offset), _p(pos), slots.numel(), _stream()), "positions")


def lengths_add(lengths, slots, real):
    _dev(lengths, slots, real)
    _index(slots=slots)
    check(lib().m3x_lengths_add(_p(lengths), _p(slots), _p(real), slots.numel(), _stream()), "lengths_add")


def add_rms(h, a, w, eps, h_out=None, y=None):
    """h_out = bf16(h + a); y = RMSNorm(h_out) (a None: y = RMSNorm(h), h_out unused). Returns (h_out, y)."""
    _dev(h, a, w, h_out, y)
    _rows2d(h, "h")
    if h.dtype != torch.bfloat16:
        raise ValueError("fused add+norm kernel is bf16-only")
    rows, n = h.shape
    if y is None:
        y = torch.empty_like(h)
    if a is not None:
        _rows2d(a, "a")
        if a.shape != h.shape:
            raise ValueError(f"add_rms: a {tuple(a.shape)} != h {tuple(h.shape)}")
        if h_out is None:
            h_out = torch.empty_like(h)
    check(lib().m3x_add_rms(_p(h), h.stride(0), _p(a), 0 if a is None else a.stride(0), _p(h_out),
                            0 if h_out is None else h_out.stride(0), _p(y), y.stride(0), _p(w), float(eps), rows, n,
                            _stream()), "add_rms")
    return h_out, y


def qk_norm_rope_cache(qkv, q_out, k_cache, v_cache, slots, pos, cos, sin, wq, wk, eps, heads, kv_heads):
    _dev(qkv, q_out, k_cache, v_cache, slots, pos, cos, sin, wq, wk)
    _index(slots=slots, pos=pos)
    D = k_cache.shape[-1]
    rows = qkv.shape[0]
    if qkv.shape[1] != (heads + 2 * kv_heads) * D:
        raise ValueError(f"qkv width {qkv.shape[1]} != (heads + 2*kv_heads)*head_dim")
    check(lib().m3x_qk_norm_rope_cache(
        _p(qkv), qkv.stride(0), _p(q_out), q_out.stride(0), q_out.stride(1), _p(k_cache), _p(v_cache),
        k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), _p(slots), _p(pos), _p(cos), _p(sin), cos.stride(0),
        _p(wq), _p(wk), float(eps), rows, heads, kv_heads, D, k_cache.shape[2], _stream()), "qk_norm_rope_cache")


def linear_qk_rope(x, w, qkv, q_out, k_cache, v_cache, slots, pos, cos, sin, wq, wk, eps, heads, kv_heads,
                   part=None, eps_in=0.0):
    """The q|k|v projection (x @ W.T, or with part given linear_normed's RMSNorm-folded product, W from fold_norm)
    followed by qk_norm_rope_cache on its output, in one launch when the row count's plan holds whole heads per
    workgroup (above 192 rows at N = 4096), else two through qkv. qkv holds the projection afterwards at up to 192 and at
    257..512 rows. Same bits as linear / linear_normed + qk_norm_rope_cache."""
    M, K, qkv = _lin_args(x, w, qkv, w.N)
    _dev(q_out, k_cache, v_cache, slots, pos, cos, sin, wq, wk, part)
    _index(slots=slots, pos=pos)
    D = k_cache.shape[-1]
    if w.N != (heads + 2 * kv_heads) * D:
        raise ValueError(f"linear_qk_rope: weight rows {w.N} != (heads + 2*kv_heads)*head_dim")
    if x.dtype != torch.bfloat16:
        raise ValueError("linear_qk_rope: bf16 only")
    if part is not None and (part.dtype != torch.float32 or not part.is_contiguous()
                             or part.numel() < tile_stats_elems(M, K)):
        raise ValueError("linear_qk_rope: part must hold the tile statistics of x")
    check(lib().m3x_linear_qk_rope(
        _p(x), x.stride(0), _p(part), float(eps_in), _p(w.data), _p(qkv), qkv.stride(0), _p(q_out), q_out.stride(0),
        q_out.stride(1), _p(k_cache), _p(v_cache), k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), _p(slots),
        _p(pos), _p(cos), _p(sin), cos.stride(0), _p(wq), _p(wk), float(eps), M, K, heads, kv_heads, D,
        k_cache.shape[2], _stream()), "linear_qk_rope")


def decode_attn_workspace(rows, kv_heads, max_ctx, chunk) -> int:
    return int(lib().m3x_decode_attn_workspace(rows, kv_heads, max_ctx, chunk))


def decode_attn(q, k_cache, v_cache, out, slots, pos, scale, max_ctx, chunk, workspace, heads, kv_heads,
                items=None):
    """q, out: [rows, heads, D] (any row/head strides, contiguous D); caches [slots, kv_heads, cap, D].
    items (int32, optional): the step's work items (attn_items with attn_item_bins bins); the rows of an inline
    prefill then share one pass over their slot's keys per min(16, 2 * (16 // (heads // kv_heads))) rows."""
    _dev(q, k_cache, v_cache, out, slots, pos, workspace, items)
    _index(slots=slots, pos=pos)
    rows = q.shape[0]
    if items is not None:
        bins = attn_item_bins(rows, kv_heads, max_ctx, chunk)
        if items.dtype != torch.int32 or not items.is_contiguous() or items.numel() < 2 + bins:
            raise ValueError(f"decode_attn: items must be contiguous int32 with {bins} bins (attn_items)")
    ws = 0 if workspace is None else workspace.numel() * workspace.element_size()
    check(lib().m3x_decode_attn(
        _p(q), q.stride(0), q.stride(1), _p(k_cache), _p(v_cache), k_cache.stride(0), k_cache.stride(1),
        k_cache.stride(2), k_cache.shape[2], _p(out), out.stride(0), out.stride(1), _p(slots), _p(pos), _p(items),
        float(scale), rows, heads, kv_heads, k_cache.shape[-1], int(max_ctx), int(chunk), _p(workspace), ws,
        _stream()), "decode_attn")


def attn_item_bins(rows, kv_heads, max_ctx, chunk) -> int:
    return int(lib().m3x_decode_attn_item_bins(rows, kv_heads, max_ctx, chunk))


def attn_items(runs, heads, kv_heads, bins, chunk):
    """Work items of decode_attn for rows laid out as runs: (first row, rows, first position) per run, a decode
    row being a run of one row and an inline prefill of T tokens a run of T rows at consecutive positions of one
    slot. Each run is cut into blocks of up to min(16, 2 * (16 // (heads // kv_heads))) rows and each block's keys into splits of
    `chunk` keys; an item is one split of one block. The items are dealt into `bins` bins (attn_item_bins) longest
    processing time first: each goes to the least loaded bin, its cost its keys plus a fixed 64. Returns int32
    [bins, start[0..bins], codes bin by bin], code = 2048 * first_row + 32 * split + rows. Built on the host by the
    library (m3x_decode_attn_items)."""
    r = np.ascontiguousarray(np.asarray(runs, dtype=np.int32).reshape(-1, 3))
    qb = max(1, 16 // (heads // kv_heads))
    n, p0 = r[:, 1].astype(np.int64), r[:, 2].astype(np.int64)
    bound = int((-(-n // qb) * (-(-(p0 + n) // chunk))).sum())  # blocks x the run's most splits
    out = np.empty(2 + bins + bound, dtype=np.int32)
    cnt = lib().m3x_decode_attn_items(r.ctypes.data, r.shape[0], heads, kv_heads, bins, chunk, out.ctypes.data,
                                      out.size)
    if cnt < 0:
        raise ValueError(f"attn_items: m3x_decode_attn_items returned {cnt}")
    return out[:cnt]


class PackedWeight:
    """An [N, K] weight (bf16, fp16 or fp32) in MFMA fragment order (see m3x_pack_weight): `data` holds
    ceil(N/16)*16*K elements."""
    __slots__ = ("data", "N", "K")

    def __init__(self, data, N, K):
        self.data, self.N, self.K = data, N, K

    @property
    def dtype(self):
        return self.data.dtype

    @property
    def device(self):
        return self.data.device

    def rows(self, start, stop):
        """Rows [start, stop) as their own packed weight (start % 16 == 0); shares storage."""
        if start % 16 or not 0 <= start < stop <= self.N:
            raise ValueError(f"rows({start}, {stop}) of a packed [{self.N}, {self.K}] weight")
        return PackedWeight(self.data[start * self.K:-(-stop // 16) * 16 * self.K], stop - start, self.K)


def pack_weight(w):
    """Pack w [N, K] (row stride % 8 == 0, K % 32 == 0) into fragment order; one launch on the current stream."""
    _dev(w)
    _rows2d(w, "w")
    N, K = w.shape
    n = int(lib().m3x_packed_weight_elems(N, K))
    if n < 0:
        raise ValueError(f"pack_weight: K={K} must be a multiple of 32")
    out = torch.empty(n, dtype=w.dtype, device=w.device)
    check(lib().m3x_pack_weight(_p(w), w.stride(0), N, K, _p(out), _dt3(w), _stream()), "pack_weight")
    return PackedWeight(out, N, K)


def _lin_args(x, w, y, N):
    if not isinstance(w, PackedWeight):
        raise TypeError("linear: the weight must be packed with ops.pack_weight")
    _dev(x, w.data, y)
    _rows2d(x, "x")
    M, K = x.shape
    if w.K != K or w.dtype != x.dtype:
        raise ValueError(f"linear: x {tuple(x.shape)} {x.dtype} vs packed w [{w.N}, {w.K}] {w.dtype}")
    if y is None:
        y = torch.empty(M, N, dtype=x.dtype, device=x.device)
    _rows2d(y, "y")
    if y.shape != (M, N) or y.dtype != x.dtype:
        raise ValueError(f"linear: y {tuple(y.shape)} {y.dtype}, expected {(M, N)} {x.dtype}")
    return M, K, y


def linear(x, w, y=None):
    """y = x @ W.T with x [M, K] and W [N, K] packed by pack_weight (same dtype); returns y [M, N]."""
    M, K, y = _lin_args(x, w, y, w.N)
    check(lib().m3x_linear(_p(x), x.stride(0), _p(w.data), _p(y), y.stride(0), M, w.N, K, _dt3(x), _stream()),
          "linear")
    return y


def linear_act(x, w_gate, w_up, kind, y=None):
    """SWIGLU: y = bf16(silu(x @ Wg.T)) * (x @ Wu.T); GELU: y = gelu(x @ Wg.T) (w_up None); weights packed."""
    I = w_gate.N
    M, K, y = _lin_args(x, w_gate, y, I)
    if kind == ACT_SWIGLU:
        if not isinstance(w_up, PackedWeight) or (w_up.N, w_up.K) != (w_gate.N, w_gate.K):
            raise ValueError("linear_act: w_up must be a packed weight of w_gate's shape")
        _dev(w_up.data)
    check(lib().m3x_linear_act(_p(x), x.stride(0), _p(w_gate.data), _p(w_up.data if kind == ACT_SWIGLU else None),
                               _p(y), y.stride(0), M, I, K, kind, _dt3(x), _stream()), "linear_act")
    return y


def tile_stats_elems(rows, n):
    """float32 elements of the tile statistics linear_resid writes for `rows` rows of width n (2 per 16 columns)."""
    return rows * (n // 16) * 2


def linear_resid(x, w, h, h_out, part, kind, c=None, tc=1):
    """h_out = dt(h + dt(x @ W.T)) [then dt(h_out + c[m // tc])], and the 16-column tile statistics of h_out into
    `part` (float32, >= tile_stats_elems(M, N)) for a following norm of `kind` (NORM_RMS or NORM_LAYER).
    h may be a strided row view (row stride h.stride(0)); h_out may be h."""
    M, K, h_out = _lin_args(x, w, h_out, w.N)
    _dev(h, c, part)
    for t, name in ((h, "h"), (c, "c")):
        if t is not None and (t.dim() != 2 or t.stride(-1) != 1 or t.dtype != x.dtype or t.shape[1] < w.N):
            raise ValueError(f"linear_resid: {name} must be a row-strided [rows, >= {w.N}] {x.dtype} view")
    if h.shape[0] < M or (c is not None and c.shape[0] * tc < M):
        raise ValueError("linear_resid: h / c have too few rows")
    if part.dtype != torch.float32 or not part.is_contiguous() or part.numel() < tile_stats_elems(M, w.N):
        raise ValueError("linear_resid: part must be a contiguous float32 buffer of tile_stats_elems(M, N)")
    check(lib().m3x_linear_resid(_p(x), x.stride(0), _p(w.data), _p(h), h.stride(0), _p(c),
                                 0 if c is None else c.stride(0), tc, _p(h_out), h_out.stride(0), _p(part), M, w.N, K,
                                 kind, _dt(x), _stream()), "linear_resid")
    return h_out


def fold_norm(w, nw, nb=None):
    """Load-time preparation of a projection w [N, K] that consumes normed rows (linear_normed): the norm's weight
    nw [K] (and LayerNorm bias nb [K]) folded in. Returns (packed dt(w * nw), u, v): for LayerNorm the fp32 column
    vectors u[n] = sum_k dt(w * nw)[n, k] and v[n] = sum_k nb[k] w[n, k]; None for RMSNorm. A joined gate|up weight
    [2I, K] gives u, v in the same [gate | up] order that linear_normed takes with ACT_SWIGLU."""
    _dev(w, nw, nb)
    if w.dim() != 2 or nw.numel() != w.shape[1] or (nb is not None and nb.numel() != w.shape[1]):
        raise ValueError("fold_norm: w [N, K] with nw (and nb) of K elements")
    wf = (w.float() * nw.float()[None]).to(w.dtype).contiguous()
    packed = pack_weight(wf)
    if nb is None:
        return packed, None, None
    return packed, wf.float().sum(1).contiguous(), (w.float() @ nb.float()).contiguous()


def linear_normed(x, part, eps, kind, w_gate, w_up=None, act_kind=ACT_NONE, u=None, v=None, y=None):
    """y = act(norm(x) @ W.T) for rows x of width 1024 whose tile statistics linear_resid left in `part`, with the
    weights prepared by fold_norm (u, v: its column vectors, LayerNorm only; [2N] for ACT_SWIGLU). act_kind
    ACT_NONE (w_up None), ACT_SWIGLU (w_up) or ACT_GELU."""
    M, K, y = _lin_args(x, w_gate, y, w_gate.N)
    _dev(part, u, v)
    if act_kind == ACT_SWIGLU and (not isinstance(w_up, PackedWeight) or (w_up.N, w_up.K) != (w_gate.N, w_gate.K)):
        raise ValueError("linear_normed: w_up must be a packed weight of w_gate's shape")
    if part.dtype != torch.float32 or not part.is_contiguous() or part.numel() < tile_stats_elems(M, K):
        raise ValueError("linear_normed: part must hold the tile statistics of x")
    ncol = w_gate.N * (2 if act_kind == ACT_SWIGLU else 1)
    if kind == NORM_LAYER:
        for t, name in ((u, "u"), (v, "v")):
            if t is None or t.dtype != torch.float32 or not t.is_contiguous() or t.numel() != ncol:
                raise ValueError(f"linear_normed: LayerNorm needs fold_norm's {name} ({ncol} float32)")
    check(lib().m3x_linear_normed(_p(x), x.stride(0), _p(part), _p(u), _p(v), eps, kind, _p(w_gate.data),
                                  _p(w_up.data if act_kind == ACT_SWIGLU else None), _p(y), y.stride(0), M,
                                  w_gate.N, K, act_kind, _dt(x), _stream()), "linear_normed")
    return y


def act(inp, out, kind):
    """SWIGLU: out[:, :I] = bf16(silu(g))*u for inp = [g | u]; GELU: out = gelu(inp[:, :I])."""
    _dev(inp, out)
    _rows2d(inp, "inp")
    _rows2d(out, "out")
    check(lib().m3x_act(_p(inp), inp.stride(0), _p(out), out.stride(0), inp.shape[0], out.shape[1], kind, _dt(inp),
                        _stream()), "act")
    return out


# ---------------------------------------------------------------- depth step
def _bt_strides(t, T):
    """(row-of-b stride, row-of-t stride) of a [B, T, N] view or a contiguous [B*T, N] tensor."""
    if t.dim() == 3:
        if t.stride(-1) != 1:
            raise ValueError("last dimension must be contiguous")
        return t.stride(0), t.stride(1)
    _rows2d(t, "x")
    return T * t.stride(0), t.stride(0)


def add_norm(x, a, c, x_out, y, w, b, eps, T, kind):
    """x, a: [B, T, N] views or [B*T, N]; c: [B, N] (row stride may be 0) or None; x_out/y contiguous [B*T, N]."""
    _dev(x, a, c, x_out, y, w, b)
    n = x.shape[-1]
    rows = y.shape[0]
    sxb, sxt = _bt_strides(x, T)
    sab, sat = _bt_strides(a, T) if a is not None else (0, 0)
    check(lib().m3x_add_norm(_p(x), sxb, sxt, _p(a), sab, sat, _p(c), 0 if c is None else c.stride(0), _p(x_out),
                             _p(y), _p(w), _p(b), float(eps), rows, T, n, kind, _dt3(y), _stream()), "add_norm")


def add_rows(x, bias, out):
    """out = x + bias (bias [N] broadcast, or [rows, N])."""
    _dev(x, bias, out)
    ldb = 0 if bias.dim() == 1 else bias.stride(0)
    check(lib().m3x_add_rows(_p(x), x.stride(0), _p(bias), ldb, _p(out), out.stride(0), x.shape[0], x.shape[-1],
                             _dt3(x), _stream()), "add_rows")


def depth_attn(qkv, kd, vd, out, B, T, p0, tq0, heads, head_dim, scale, write_kv=True):
    _dev(qkv, kd, vd, out)
    sqb, sqt = _bt_strides(qkv, T)
    sob, sot = _bt_strides(out, T - tq0)
    check(lib().m3x_depth_attn(_p(qkv), sqb, sqt, _p(kd), _p(vd), _p(out), sob, sot, B, T, p0, tq0, heads, head_dim,
                               kd.shape[2], float(scale), int(write_kv), _dt3(qkv), _stream()), "depth_attn")


def topk_sample(logits, u, inv_temp, top_k, greedy, out, out_i64=False):
    """logits [B, V] 16-bit; u [B] view (any stride) or None for greedy; out [B] view (int32/int64)."""
    _dev(logits, u, out)
    _rows2d(logits, "logits")
    B, V = logits.shape
    check(lib().m3x_topk_sample(_p(logits), logits.stride(0), V, _p(u), 0 if u is None else u.stride(0),
                                float(inv_temp), int(top_k), int(greedy), _p(out), out.stride(0), int(out_i64), B,
                                _dt3(logits), _stream()), "topk_sample")


def topk_sample_embed(logits, u, inv_temp, top_k, greedy, out, table, prefix, x_out=None, y=None, w=None, b=None,
                      eps=0.0, kind=NORM_RMS, out_i64=False):
    """topk_sample, then prefix[r] = table[code_r]; with y given also x_out[r] = table[code_r] and
    y[r] = norm(table[code_r]) (the add_norm arithmetic with no addend). prefix: [B, n] view (any row stride);
    x_out, y: contiguous [B, n]."""
    _dev(logits, u, out, table, prefix, x_out, y, w, b)
    _rows2d(logits, "logits")
    _rows2d(table, "table")
    B, V = logits.shape
    n = table.shape[-1]
    if prefix.shape[-1] != n or prefix.shape[0] != B:
        raise ValueError("topk_sample_embed: prefix must be [B, n]")
    if table.shape[0] < V:
        raise ValueError(f"topk_sample_embed: table has {table.shape[0]} rows for {V} codes")
    if any(t is not None and t.dtype != logits.dtype for t in (table, prefix, x_out, y, w, b)):
        raise ValueError("topk_sample_embed: logits, table, prefix, x_out, y, w and b share one dtype")
    for t, name in ((x_out, "x_out"), (y, "y")):
        if t is not None and (not t.is_contiguous() or tuple(t.shape) != (B, n)):
            raise ValueError(f"topk_sample_embed: {name} must be contiguous [B, n]")
    check(lib().m3x_topk_sample_embed(
        _p(logits), logits.stride(0), V, _p(u), 0 if u is None else u.stride(0), float(inv_temp), int(top_k),
        int(greedy), _p(out), out.stride(0), int(out_i64), B, _p(table), table.stride(0), table.shape[0], _p(prefix),
        prefix.stride(0), _p(x_out), _p(y), _p(w), _p(b), float(eps), int(kind), n, _dt3(logits), _stream()),
        "topk_sample_embed")


def cb0_sample(logits, aeos, slots, u, temp_t=None, temp=1.0, topk_t=None, top_k=50, aeos_bias=None, rep_t=None,
               hist_t=None, frames_t=None, min_t=None, hazard_t=None, ctr_t=None, cb0_out=None, cb0_i32=None,
               stop_out=None, topp_t=None, top_p=1.0):
    _dev(logits, slots, u, temp_t, topk_t, aeos_bias, rep_t, hist_t, frames_t, min_t, hazard_t, ctr_t, cb0_out,
         cb0_i32, stop_out, topp_t)
    _index(slots=slots)
    if topp_t is not None and topp_t.dtype != torch.float32:
        raise ValueError("topp_t must be float32")
    _rows2d(logits, "logits")
    if logits.dtype != torch.bfloat16:
        raise ValueError("cb0 logits must be bfloat16")
    B, V = logits.shape
    check(lib().m3x_cb0_sample(
        _p(logits), logits.stride(0), V, int(aeos), _p(slots), _p(u), u.stride(0), _p(temp_t), float(temp),
        _p(topk_t), int(top_k), _p(topp_t), float(top_p), _p(aeos_bias), _p(rep_t), _p(hist_t), 0 if hist_t is None else hist_t.shape[1],
        _p(frames_t), _p(min_t), _p(hazard_t), _p(ctr_t), _p(cb0_out), _p(cb0_i32),
        0 if cb0_i32 is None else cb0_i32.stride(0), _p(stop_out), B, _stream()), "cb0_sample")


def philox_uniforms(seeds, ctrs, slots, out, level0):
    """out [B, nlevels] (row stride free) = Philox uniforms for levels level0.. of each slot's stream."""
    _dev(seeds, ctrs, slots, out)
    _index(slots=slots)
    _need(seeds, torch.int32, "seeds")
    _need(ctrs, torch.int32, "ctrs")
    _need(out, torch.float32, "out")
    check(lib().m3x_philox_uniforms(_p(seeds), _p(ctrs), _p(slots), _p(out), out.stride(0), int(level0),
                                    out.shape[1], slots.numel(), _stream()), "philox_uniforms")


def philox_exponential(seeds, ctrs, out, level):
    """out [B, V] = Exp(1) noise of each row's (seed, counter) stream at `level`."""
    _dev(seeds, ctrs, out)
    _need(seeds, torch.int32, "seeds")
    _need(ctrs, torch.int32, "ctrs")
    _need(out, torch.float32, "out")
    check(lib().m3x_philox_exponential(_p(seeds), _p(ctrs), _p(out), out.stride(0), int(level), out.shape[1],
                                       out.shape[0], _stream()), "philox_exponential")


def philox_block(counter, key, out):
    check(lib().m3x_philox_block(_p(counter), _p(key), _p(out), _stream()), "philox_block")


def ctr_add(ctr, slots):
    _dev(ctr, slots)
    _index(slots=slots)
    check(lib().m3x_ctr_add(_p(ctr), _p(slots), slots.numel(), _stream()), "ctr_add")


def feedback(table, codes, out, w, eps, scale, n_q, n_codes):
    _dev(table, codes, out, w)
    _need(codes, torch.int32, "codes")
    check(lib().m3x_feedback(_p(table), _p(codes), codes.stride(0), _p(out), out.stride(0), _p(w), float(eps),
                             float(scale), out.shape[0], out.shape[1], int(n_q), int(n_codes), _dt3(table),
                             _stream()), "feedback")


def copy_rows(src, dst, src_idx=None, src_off=0, dst_idx=None, rows=None):
    """dst[dst_idx[r] or r] = src[src_idx[r] + src_off or r] for r < rows (rows of 16-bit elements with
    width % 8 == 0, or of fp32 elements with width % 4 == 0, moved as pairs of 16-bit halves)."""
    _dev(src, dst, src_idx, dst_idx)
    if src.dtype != dst.dtype or src.element_size() not in (2, 4):
        raise ValueError(f"copy_rows: {src.dtype} -> {dst.dtype}")
    w = src.element_size() // 2  # 16-bit units per element
    n = src.shape[-1] * w
    if dst.shape[-1] * w != n:
        raise ValueError("copy_rows: row widths differ")
    if rows is None:
        rows = src_idx.numel() if src_idx is not None else (dst_idx.numel() if dst_idx is not None else src.shape[0])
    idx_i32 = 0
    ld_idx = 1
    if src_idx is not None:
        if src_idx.dtype == torch.int32:
            idx_i32 = 1
        elif src_idx.dtype != torch.long:
            raise ValueError("indices must be int32 or int64")
        ld_idx = src_idx.stride(0)
    if dst_idx is not None:
        _need(dst_idx, torch.long, "dst_idx")
    check(lib().m3x_copy_rows(_p(src), src.stride(-2) * w, _p(src_idx), int(src_off), src.shape[-2], _p(dst),
                              dst.stride(-2) * w, _p(dst_idx), int(rows), n, idx_i32, ld_idx, _stream()), "copy_rows")


def cast_rows(src, dst):
    """dst = src converted to dst's dtype (bf16 / fp16 / fp32 rows with a contiguous last dimension)."""
    _dev(src, dst)
    _rows2d(src, "src")
    _rows2d(dst, "dst")
    if src.shape != dst.shape or src.dtype not in _DT_ANY or dst.dtype not in _DT_ANY:
        raise ValueError(f"cast_rows: {tuple(src.shape)} {src.dtype} -> {tuple(dst.shape)} {dst.dtype}")
    check(lib().m3x_cast_rows(_p(src), src.stride(0), _DT_ANY[src.dtype], _p(dst), dst.stride(0),
                              _DT_ANY[dst.dtype], src.shape[0], src.shape[1], _stream()), "cast_rows")
    return dst


def code_ring_write(codes, ring, head, B):
    _dev(codes, ring, head)
    check(lib().m3x_code_ring_write(_p(codes), codes.stride(0), _p(ring), _p(head), ring.shape[0], ring.shape[1],
                                    ring.shape[2], int(B), _stream()), "code_ring_write")


# ---------------------------------------------------------------- the depth frame as one persistent run
class DepthRunArgs(ctypes.Structure):
    """Mirror of M3xDepthRun (include/m3x.h); its size is checked against the library's."""
    _P4 = ctypes.c_void_p * 4
    _fields_ = [(n, ctypes.c_int) for n in ("B", "L0", "L1", "layers", "H", "hd", "F", "V", "act", "norm_kind",
                                            "dtype", "nwg")] + [
        ("inv_temp", ctypes.c_float), ("top_k", ctypes.c_int), ("greedy", ctypes.c_int),
        ("eps1", ctypes.c_float * 4), ("eps2", ctypes.c_float * 4), ("eps_f", ctypes.c_float),
        ("n1w", _P4), ("n1b", _P4), ("n2w", _P4), ("n2b", _P4), ("fw", ctypes.c_void_p), ("fb", ctypes.c_void_p),
        ("wqkv", _P4), ("wo", _P4), ("wg", _P4), ("wu", _P4), ("wd", _P4), ("heads", ctypes.c_void_p * 31),
        ("embed", ctypes.c_void_p), ("cross", ctypes.c_void_p), ("ld_cross", ctypes.c_long),
        ("prefix", ctypes.c_void_p), ("ld_prefix", ctypes.c_long), ("codes", ctypes.c_void_p),
        ("ld_codes", ctypes.c_long), ("u", ctypes.c_void_p), ("ld_u", ctypes.c_long), ("kd", _P4), ("vd", _P4),
        ("kv_sb", ctypes.c_long), ("kv_sh", ctypes.c_long), ("xchg", ctypes.c_void_p), ("sync", ctypes.c_void_p),
        ("logits_out", ctypes.c_void_p), ("prof", ctypes.c_void_p), ("probe", ctypes.c_int),
        ("spin_limit", ctypes.c_uint)]


def depth_run_xchg_bytes() -> int:
    return int(lib().m3x_depth_run_xchg_bytes())


def depth_run(args: DepthRunArgs):
    """Launch a persistent depth run on the current stream (args built by FastDepth)."""
    if ctypes.sizeof(DepthRunArgs) != int(lib().m3x_depth_run_args_bytes()):
        raise RuntimeError("DepthRunArgs does not match the library's M3xDepthRun: rebuild the library")
    check(lib().m3x_depth_run(ctypes.byref(args), _stream()), "depth_run")


def depth_run_void(sync, codes, B, L0, L1):
    """After a run (stream order): codes[:B, L0:L1] = -1 when the run's error word sync[2] is set."""
    _dev(sync, codes)
    check(lib().m3x_depth_run_void(_p(sync), _p(codes), codes.stride(0), B, L0, L1, _stream()), "depth_run_void")


# ---------------------------------------------------------------- one-row backbone run (serve/fast_backbone.py)
class BackboneLayer(ctypes.Structure):
    """Mirror of M3xBackboneLayer (include/m3x.h); rows of a device table, one per layer."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("wqkv", "wo", "wg", "wu", "wd", "wq", "wk", "kc", "vc")]


class BackboneRunArgs(ctypes.Structure):
    """Mirror of M3xBackboneRun (include/m3x.h); its size is checked against the library's."""
    _fields_ = [("layer", ctypes.c_void_p)] + [(n, ctypes.c_int) for n in ("layers", "cap", "nwg", "probe")] + [
        ("spin_limit", ctypes.c_uint), ("eps", ctypes.c_float), ("scale", ctypes.c_float),
        ("x", ctypes.c_void_p), ("h_out", ctypes.c_void_p), ("slots", ctypes.c_void_p), ("pos", ctypes.c_void_p),
        ("cos", ctypes.c_void_p), ("sin", ctypes.c_void_p), ("s_cos", ctypes.c_long), ("w_in0", ctypes.c_void_p),
        ("sk_s", ctypes.c_long), ("sk_h", ctypes.c_long), ("sk_t", ctypes.c_long), ("xchg", ctypes.c_void_p),
        ("sync", ctypes.c_void_p), ("prof", ctypes.c_void_p), ("w_fin", ctypes.c_void_p), ("y_out", ctypes.c_void_p),
        ("lengths", ctypes.c_void_p), ("real", ctypes.c_void_p)]


def backbone_run_xchg_bytes() -> int:
    return int(lib().m3x_backbone_run_xchg_bytes())


def backbone_layer_table(layers, device):
    """The device table of M3xBackboneLayer rows for `layers` (lists of BackboneLayer)."""
    if ctypes.sizeof(BackboneLayer) != int(lib().m3x_backbone_run_layer_bytes()):
        raise RuntimeError("BackboneLayer does not match the library's M3xBackboneLayer: rebuild the library")
    raw = (BackboneLayer * len(layers))(*layers)
    host = torch.frombuffer(bytearray(bytes(raw)), dtype=torch.int64).clone()
    return host.to(device)


def backbone_run(args: BackboneRunArgs):
    """Launch a one-row backbone run on the current stream (args built by StaticBackbone)."""
    if ctypes.sizeof(BackboneRunArgs) != int(lib().m3x_backbone_run_args_bytes()):
        raise RuntimeError("BackboneRunArgs does not match the library's M3xBackboneRun: rebuild the library")
    check(lib().m3x_backbone_run(ctypes.byref(args), _stream()), "backbone_run")


# ---------------------------------------------------------------- 4-bit cache and weights
_raw_stream = torch._C._cuda_getCurrentRawStream  # a device's current stream as torch.cuda.current_stream, ~2 us cheaper
_current_device = torch._C._cuda_getDevice  # as torch.cuda.current_device of an initialised process, ~0.2 us cheaper


def _launch(dev, fn, *args):
    """A launching entry point on device `dev` (an index) and its current stream, whichever device is current."""
    if dev == _current_device():
        rc = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _raw_stream(dev))
    if rc:
        check(rc, fn.__name__)


class Kv4CacheArgs(ctypes.Structure):
    """Mirror of M3xKv4 (include/m3x.h)."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "ks", "v", "vs")] + [
        (n, ctypes.c_int) for n in ("slots", "kv_heads", "head_dim", "cap")]


class Kv4Cache:
    """A layer's KV cache in 4 bits (format and layout: include/m3x.h): uint8 tensors
    k [slots, kv_heads, cap, head_dim / 2], ks [slots, kv_heads, cap, head_dim / 32],
    v [slots, kv_heads, cap / 4, 16, 4, head_dim / 32], vs [slots, kv_heads, cap / 4, head_dim / 32, 4].
    head_dim 64 or 128, cap a multiple of 32. The tensors are the handle's for its life: their storage is not resized
    or replaced."""
    __slots__ = ("k", "ks", "v", "vs", "slots", "kv_heads", "cap", "head_dim", "device", "_index", "_args", "_ref")

    def __init__(self, k, ks, v, vs):
        if k.dim() != 4:
            raise ValueError(f"Kv4Cache: k must be [slots, kv_heads, cap, head_dim / 2], got {tuple(k.shape)}")
        S, KV, cap, half = k.shape
        D = 2 * half
        if D not in (64, 128) or cap % 32 or cap > 1 << 30 or min(S, KV, cap) < 1:
            raise ValueError(f"Kv4Cache: head_dim {D} must be 64 or 128 and cap {cap} a multiple of 32 up to 2^30")
        for t, shape, name in ((k, (S, KV, cap, D // 2), "k"), (ks, (S, KV, cap, D // 32), "ks"),
                               (v, (S, KV, cap // 4, 16, 4, D // 32), "v"), (vs, (S, KV, cap // 4, D // 32, 4), "vs")):
            if t.dtype != torch.uint8 or tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"Kv4Cache: {name} must be contiguous uint8 {shape}, got {t.dtype} {tuple(t.shape)}")
            if t.device != k.device or t.data_ptr() % 16:
                raise ValueError(f"Kv4Cache: {name} must be 16-byte aligned on {k.device}")
        self.k, self.ks, self.v, self.vs = k, ks, v, vs
        self.slots, self.kv_heads, self.cap, self.head_dim, self.device = S, KV, cap, D, k.device
        self._index = k.get_device()
        self._args = Kv4CacheArgs(k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr(), S, KV, D, cap)
        self._ref = ctypes.addressof(self._args)

    @classmethod
    def empty(cls, slots, kv_heads, cap, head_dim, device):
        """A new cache (all zeros)."""
        if head_dim not in (64, 128):
            raise ValueError(f"Kv4Cache: head_dim {head_dim} must be 64 or 128")

        def z(*shape):
            return torch.zeros(*shape, dtype=torch.uint8, device=device)
        D = head_dim
        return cls(z(slots, kv_heads, cap, D // 2), z(slots, kv_heads, cap, D // 32),
                   z(slots, kv_heads, cap // 4, 16, 4, D // 32), z(slots, kv_heads, cap // 4, D // 32, 4))

    def memory_bytes(self):
        return sum(t.numel() for t in (self.k, self.ks, self.v, self.vs))


def _kv4_rows(name, cache, slots, pos):
    """(rows, slots pointer, pos pointer) of a call's rows."""
    if not isinstance(cache, Kv4Cache):
        raise TypeError(f"{name}: the cache must be an ops.Kv4Cache")
    if slots.dtype != torch.int64 or pos.dtype != torch.int32:
        raise ValueError(f"{name}: slots must be int64 and pos int32, got {slots.dtype}, {pos.dtype}")
    shape = slots.shape
    if len(shape) != 1 or pos.shape != shape or not slots.is_contiguous() or not pos.is_contiguous():
        raise ValueError(f"{name}: slots and pos must be contiguous [rows], got {tuple(shape)}, {tuple(pos.shape)}")
    if slots.get_device() != cache._index or pos.get_device() != cache._index:
        raise ValueError(f"{name}: slots on {slots.device}, pos on {pos.device}, the cache on {cache.device}")
    return shape[0], slots.data_ptr(), pos.data_ptr()


def _kv4_heads(name, what, t, cache, rows, heads, dtype=None):
    """(pointer, row stride, head stride) of rows [rows, heads, head_dim]."""
    if t.shape != (rows, heads, cache.head_dim):
        raise ValueError(f"{name}: {what} must be {(rows, heads, cache.head_dim)}, got {tuple(t.shape)}")
    if t.dtype not in _DT if dtype is None else t.dtype != dtype:
        raise ValueError(f"{name}: {what} must be {'bfloat16 or float16' if dtype is None else dtype}, got {t.dtype}")
    if t.get_device() != cache._index:
        raise ValueError(f"{name}: {what} on {t.device}, the cache on {cache.device}")
    sr, sh, sd = t.stride()
    ptr = t.data_ptr()
    if (sr | sh | ptr >> 1) & 7 or (sd != 1 and rows):
        raise ValueError(f"{name}: {what} needs a contiguous last dimension and 16-byte aligned rows (strides {t.stride()})")
    return ptr, sr, sh


def _on_gpu(name, cache):
    if cache._index < 0:
        raise ValueError(f"{name}: m3x kernels take device tensors")


def kv4_append(k, v, cache, slots, pos):
    """K and V rows [rows, kv_heads, head_dim] (bf16 or fp16, any row and head strides) quantised to position pos[r]
    (int32) of slot slots[r] (int64). A row whose slot or position is outside the cache is not written; rows at one
    place leave a mixture there."""
    rows, sp, pp = _kv4_rows("kv4_append", cache, slots, pos)
    ka = _kv4_heads("kv4_append", "k", k, cache, rows, cache.kv_heads)
    va = _kv4_heads("kv4_append", "v", v, cache, rows, cache.kv_heads, k.dtype)
    _on_gpu("kv4_append", cache)
    _launch(cache._index, lib().m3x_kv4_append, cache._ref, *ka, *va, sp, pp, rows, _DT[k.dtype])


def qk_norm_rope_kv4(qkv, q_out, cache, slots, pos, cos, sin, wq, wk, eps, heads):
    """qk_norm_rope_cache over a Kv4Cache: q_out's bits are its, and the rotated keys (bf16) and the values are
    quantised as kv4_append does. bf16; cos, sin [>= cache.cap, head_dim]."""
    name = "qk_norm_rope_kv4"
    rows, sp, pp = _kv4_rows(name, cache, slots, pos)
    D, KV = cache.head_dim, cache.kv_heads
    _rows2d(qkv, "qkv")
    if qkv.shape != (rows, (heads + 2 * KV) * D):
        raise ValueError(f"{name}: qkv must be [{rows}, {(heads + 2 * KV) * D}], got {tuple(qkv.shape)}")
    qa = _kv4_heads(name, "q_out", q_out, cache, rows, heads, torch.bfloat16)
    for t, what in ((cos, "cos"), (sin, "sin")):
        if t.dim() != 2 or t.shape[0] < cache.cap or t.shape[1] != D or t.stride(1) != 1:
            raise ValueError(f"{name}: {what} must be [>= {cache.cap}, {D}], got {tuple(t.shape)}")
    if cos.stride(0) != sin.stride(0):
        raise ValueError(f"{name}: cos and sin share one row stride")
    if wq.numel() != D or wk.numel() != D or not wq.is_contiguous() or not wk.is_contiguous():
        raise ValueError(f"{name}: wq and wk have {D} elements")
    for t in (qkv, cos, sin, wq, wk):
        if t.dtype != torch.bfloat16 or t.get_device() != cache._index:
            raise ValueError(f"{name}: bfloat16 tensors on {cache.device}, got {t.dtype} on {t.device}")
    _on_gpu(name, cache)
    _launch(cache._index, lib().m3x_qk_norm_rope_kv4, cache._ref, qkv.data_ptr(), qkv.stride(0), *qa, sp, pp,
            cos.data_ptr(), sin.data_ptr(), cos.stride(0), wq.data_ptr(), wk.data_ptr(), float(eps), rows, heads)


def kv4_read(cache, slots, pos, k, v):
    """k, v [rows, kv_heads, head_dim] (bf16 or fp16, any row and head strides) = the numbers at position pos[r] of
    slot slots[r]; zeros for a row outside the cache."""
    rows, sp, pp = _kv4_rows("kv4_read", cache, slots, pos)
    ka = _kv4_heads("kv4_read", "k", k, cache, rows, cache.kv_heads)
    va = _kv4_heads("kv4_read", "v", v, cache, rows, cache.kv_heads, k.dtype)
    _on_gpu("kv4_read", cache)
    _launch(cache._index, lib().m3x_kv4_read, cache._ref, sp, pp, *ka, *va, rows, _DT[k.dtype])


def kv4_attn_chunk(rows, heads, kv_heads, max_ctx, head_dim=128) -> int:
    """Keys per split of kv4_attn for `rows` rows of up to max_ctx keys: a workgroup (a row, a kv head, a split) per CU
    at head_dim 128, two at 64 (whose arithmetic is the larger share), at least 128 keys each and no more than there are
    (rounded up to 128); up to 1024 keys whole (no join of splits behind). Rows known to be a prompt's count as one per
    16 // (heads // kv_heads), the rows that share a pass: 64 of them at 4000 keys 13.4 us instead of 22.5.

    Measured on MI355X (graph-timed, us, 16/8 heads of 128, combine included): one row at 1024 keys 7.2 whole (128 keys
    a split: 6.4), 32 rows 8.8 (512: 12.5); one row at 2048 7.0 (128; 512: 8.2, 2048: 11.0), 32 rows 14.4 whole (1024:
    18.2); one row at 32000 11.5 (1024; 256: 15.3, 4096: 21.8), 4 rows 27.7 (4096; 1024: 27.9, 8192: 37.9); 224 rows at
    2048 77 whole. 32/4 heads of 64: 2 rows at 120000 19.2 (1920; 1024: 22.5, 8192: 31.9), 16 rows at 32000 30.9 (4096;
    512: 40.0)."""
    if max_ctx <= 1024:
        return 1024
    blocks = rows * kv_heads * -(-heads // (16 * kv_heads))
    tiles = -(-max_ctx // 128)
    return 128 * min(tiles, max(1, -(-blocks * max_ctx // (128 * (256 if head_dim == 128 else 512)))))


def kv4_attn_workspace(rows, heads, head_dim, max_ctx, chunk) -> int:
    """Bytes of workspace for kv4_attn (0: none)."""
    if max(rows, heads, head_dim, max_ctx, chunk) >= 1 << 31:
        raise ValueError(f"kv4_attn_workspace: counts below 2^31, got {(rows, heads, head_dim, max_ctx, chunk)}")
    return int(lib().m3x_kv4_attn_workspace(rows, heads, head_dim, max_ctx, chunk))


def kv4_attn(q, cache, out, slots, pos, scale, max_ctx, chunk, workspace):
    """out[r, h] = softmax(scale q[r, h] . K^T) V over positions 0 .. pos[r] of slot slots[r]; q, out
    [rows, heads, head_dim] (bf16 or fp16, any row and head strides). A row with pos[r] < 0 or a slot outside the
    cache gets zeros. max_ctx: at least every pos[r] + 1; chunk: keys per split (kv4_attn_chunk); workspace: a tensor of
    kv4_attn_workspace bytes, or None when that is 0 (calls that may run at the same time need one each). Rows of one
    slot at consecutive positions (a prompt's) that stand next to each other share one pass over the keys. |scale| is at
    most 2^127."""
    rows, sp, pp = _kv4_rows("kv4_attn", cache, slots, pos)
    heads = q.shape[1] if q.dim() == 3 else 0
    if heads == 0 or heads % cache.kv_heads:
        raise ValueError(f"kv4_attn: {heads} query heads over {cache.kv_heads} kv heads")
    qa = _kv4_heads("kv4_attn", "q", q, cache, rows, heads)
    oa = _kv4_heads("kv4_attn", "out", out, cache, rows, heads, q.dtype)
    if not 1 <= max_ctx <= cache.cap or not 128 <= chunk < 1 << 31 or chunk % 128:
        raise ValueError(f"kv4_attn: max_ctx {max_ctx} must be in [1, {cache.cap}] and chunk {chunk} a multiple of 128 "
                         "below 2^31")
    if not abs(scale) <= 2.0 ** 127:
        raise ValueError(f"kv4_attn: |scale| must be at most 2^127, got {scale}")
    ws, ws_bytes = 0, 0
    if max_ctx > chunk:
        need = kv4_attn_workspace(rows, heads, cache.head_dim, max_ctx, chunk)
        if workspace is not None:
            ws, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        if ws_bytes < need:
            raise ValueError(f"kv4_attn: a workspace of {need} bytes is needed, got {ws_bytes}")
        if ws_bytes and (not workspace.is_contiguous() or ws % 16 or workspace.get_device() != cache._index):
            raise ValueError(f"kv4_attn: the workspace must be contiguous, 16-byte aligned and on {cache.device}")
    _on_gpu("kv4_attn", cache)
    _launch(cache._index, lib().m3x_kv4_attn, cache._ref, *qa, *oa, sp, pp, scale, rows, heads, max_ctx, chunk, ws,
            ws_bytes, _DT[q.dtype])


class PackedWeight4:
    """An [N, K] weight in 4 bits (format and layout: include/m3x.h): uint8 codes [tiles, steps, 64, 16] and scales
    [tiles, ceil(steps / 4), 64, 4], tiles of 16 rows and steps of 128 inputs."""
    __slots__ = ("codes", "scales", "N", "K")

    def __init__(self, codes, scales, N, K):
        if N < 1 or K < 32 or K % 32:
            raise ValueError(f"PackedWeight4: K={K} must be a multiple of 32")
        tiles, steps = -(-N // 16), -(-K // 128)
        for t, shape, name in ((codes, (tiles, steps, 64, 16), "codes"), (scales, (tiles, -(-steps // 4), 64, 4), "scales")):
            if t.dtype != torch.uint8 or tuple(t.shape) != shape or not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"PackedWeight4: {name} must be contiguous, aligned uint8 {shape}, got {t.dtype} "
                                 f"{tuple(t.shape)}")
        if codes.device != scales.device:
            raise ValueError(f"PackedWeight4: codes on {codes.device}, scales on {scales.device}")
        self.codes, self.scales, self.N, self.K = codes, scales, N, K

    @property
    def device(self):
        return self.codes.device

    def rows(self, start, stop):
        """Rows [start, stop) as their own packed weight (start % 16 == 0); shares storage. A stop inside a tile leaves
        the tile's other rows in place, unused."""
        if start % 16 or not 0 <= start < stop <= self.N:
            raise ValueError(f"rows({start}, {stop}) of a packed [{self.N}, {self.K}] weight")
        a, b = start // 16, -(-stop // 16)
        return PackedWeight4(self.codes[a:b], self.scales[a:b], stop - start, self.K)

    def memory_bytes(self):
        return self.codes.numel() + self.scales.numel()


def pack_weight4(w):
    """w [N, K] (bf16, fp16 or fp32; row stride % 8 == 0, K % 32 == 0, fewer than 2^26 tiles of 16 rows x 128 inputs) in 4 bits;
    one launch on the current stream."""
    _rows2d(w, "w")
    N, K = w.shape
    if N < 1 or K < 32 or K % 32:
        raise ValueError(f"pack_weight4: K={K} must be a multiple of 32")
    if -(-N // 16) * -(-K // 128) >= 1 << 26:
        raise ValueError(f"pack_weight4: fewer than 2^26 tiles of 16 x 128, got {N} x {K}")
    if w.stride(0) % 8 or w.data_ptr() % 16:
        raise ValueError(f"pack_weight4: w needs 16-byte aligned rows (stride {w.stride(0)})")
    dt = _dt3(w)
    _dev(w)
    tiles, steps = -(-N // 16), -(-K // 128)
    codes = torch.empty(tiles, steps, 64, 16, dtype=torch.uint8, device=w.device)
    scales = torch.empty(tiles, -(-steps // 4), 64, 4, dtype=torch.uint8, device=w.device)
    _launch(w.get_device(), lib().m3x_pack_weight4, w.data_ptr(), w.stride(0), N, K, codes.data_ptr(),
            scales.data_ptr(), dt)
    return PackedWeight4(codes, scales, N, K)


def _lin4_args(name, x, w, y):
    """(y, device index, x's pointer and row stride, y's pointer and row stride, rows)."""
    if not isinstance(w, PackedWeight4):
        raise TypeError(f"{name}: the weight must be packed with ops.pack_weight4")
    shape = x.shape
    if len(shape) != 2 or shape[1] != w.K or x.dtype not in _DT:
        raise ValueError(f"{name}: x must be bfloat16 or float16 [rows, {w.K}], got {x.dtype} {tuple(shape)}")
    M = shape[0]
    sr, sk = x.stride()
    xp = x.data_ptr()
    if (sr | xp >> 1) & 7 or (sk != 1 and M):
        raise ValueError(f"{name}: x needs a contiguous last dimension and 16-byte aligned rows (strides {x.stride()})")
    if y is None:
        y = x.new_empty((M, w.N))
        ldy = w.N
    else:
        if y.shape != (M, w.N) or y.dtype != x.dtype or (M and w.N > 1 and y.stride(1) != 1):
            raise ValueError(f"{name}: y must be {x.dtype} {(M, w.N)} with a contiguous last dimension, got {y.dtype} "
                             f"{tuple(y.shape)}")
        ldy = y.stride(0)
    dev = x.get_device()
    if dev < 0:
        raise ValueError(f"{name}: m3x kernels take device tensors")
    if w.codes.get_device() != dev or y.get_device() != dev:
        raise ValueError(f"{name}: x on {x.device}, the weight on {w.device}, y on {y.device}")
    return y, dev, xp, sr, y.data_ptr(), ldy, M


def linear4(x, w, y=None):
    """y = x @ W.T for rows x [M, K] (bf16 or fp16) and a weight packed by pack_weight4; the 4-bit form of `linear`
    for few rows. Returns y [M, N] (new unless given)."""
    y, dev, xp, ldx, yp, ldy, M = _lin4_args("linear4", x, w, y)
    _launch(dev, lib().m3x_linear4, xp, ldx, w.codes.data_ptr(), w.scales.data_ptr(), yp, ldy, M, w.N, w.K, _DT[x.dtype])
    return y


def linear4_act(x, w_gate, w_up, kind, y=None):
    """SWIGLU: y = silu(x @ Wg.T) * (x @ Wu.T); GELU: y = gelu(x @ Wg.T) (w_up None); the 4-bit form of `linear_act`,
    rounded once."""
    if kind not in (ACT_SWIGLU, ACT_GELU):
        raise ValueError("linear4_act: kind must be ACT_SWIGLU or ACT_GELU")
    u = (0, 0)
    if kind == ACT_SWIGLU:
        if not isinstance(w_up, PackedWeight4) or not isinstance(w_gate, PackedWeight4) or \
                (w_up.N, w_up.K) != (w_gate.N, w_gate.K) or w_up.device != w_gate.device:
            raise ValueError("linear4_act: w_up must be a packed weight of w_gate's shape, on its device")
        u = (w_up.codes.data_ptr(), w_up.scales.data_ptr())
    y, dev, xp, ldx, yp, ldy, M = _lin4_args("linear4_act", x, w_gate, y)
    _launch(dev, lib().m3x_linear4_act, xp, ldx, w_gate.codes.data_ptr(), w_gate.scales.data_ptr(), *u, yp, ldy, M,
            w_gate.N, w_gate.K, kind, _DT[x.dtype])
    return y


# ---------------------------------------------------------------- paged 16-bit cache
class PagedKvArgs(ctypes.Structure):
    """Mirror of M3xPagedKv (include/m3x.h)."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "table")] + [("page_stride", ctypes.c_long)] + [
        (n, ctypes.c_int) for n in ("pages", "page_size", "kv_heads", "head_dim", "slots", "width", "dtype")]


class PagedKv:
    """A layer's KV cache in pages (include/m3x.h): pools k, v [pages, kv_heads, page_size, head_dim] (bf16 or fp16; one
    page stride, the rest contiguous) and the table [slots, width] (int32, contiguous) that names the page of every
    page_size positions of a slot. Layers may share a table, slots a page; an entry outside the pool (-1) is no page.
    head_dim 64 or 128, page_size 16, 32, 64, 128 or 256, up to 2^30 positions a slot (`cap`). The tensors are the
    handle's for its life: their storage is not resized or replaced; the table's entries may change between calls."""
    __slots__ = ("k", "v", "table", "pages", "page_size", "kv_heads", "head_dim", "slots", "cap", "dtype", "device",
                 "_index", "_args", "_ref")

    def __init__(self, k, v, table):
        if k.dim() != 4:
            raise ValueError(f"PagedKv: k must be [pages, kv_heads, page_size, head_dim], got {tuple(k.shape)}")
        N, KV, P, D = k.shape
        if D not in (64, 128) or P not in (16, 32, 64, 128, 256) or min(N, KV) < 1 or k.dtype not in _DT:
            raise ValueError(f"PagedKv: head_dim {D} must be 64 or 128, page_size {P} a power of two from 16 to 256 and "
                             f"the type bfloat16 or float16, got {k.dtype}")
        for t, name in ((k, "k"), (v, "v")):
            if t.shape != k.shape or t.dtype != k.dtype or t.device != k.device or t.stride() != k.stride():
                raise ValueError(f"PagedKv: {name} must be {k.dtype} {tuple(k.shape)} with strides {k.stride()} on "
                                 f"{k.device}")
            if t.stride()[1:] != (P * D, D, 1) or t.stride(0) % 8 or t.stride(0) < KV * P * D or t.data_ptr() % 16:
                raise ValueError(f"PagedKv: {name}'s pages must be contiguous and 16-byte aligned (strides {t.stride()})")
        if table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous() or table.device != k.device:
            raise ValueError(f"PagedKv: table must be contiguous int32 [slots, width] on {k.device}")
        S, W = table.shape
        if min(S, W) < 1 or W * P > 1 << 30:
            raise ValueError(f"PagedKv: a table of {S} x {W} pages of {P}: at least one slot, at most 2^30 positions")
        self.k, self.v, self.table = k, v, table
        self.pages, self.page_size, self.kv_heads, self.head_dim, self.slots = N, P, KV, D, S
        self.cap, self.dtype, self.device, self._index = W * P, k.dtype, k.device, k.get_device()
        self._args = PagedKvArgs(k.data_ptr(), v.data_ptr(), table.data_ptr(), k.stride(0), N, P, KV, D, S, W,
                                 _DT[k.dtype])
        self._ref = ctypes.addressof(self._args)

    @classmethod
    def empty(cls, pages, kv_heads, page_size, head_dim, table, dtype=torch.bfloat16):
        """New pools (zeros) under `table`."""
        return cls(*(torch.zeros(pages, kv_heads, page_size, head_dim, dtype=dtype, device=table.device) for _ in "kv"),
                   table)

    def memory_bytes(self):
        """Bytes of the pools."""
        return 2 * self.k.numel() * self.k.element_size()


class RotaryArgs(ctypes.Structure):
    """Mirror of M3xRotary (include/m3x.h)."""
    _fields_ = [("freq", ctypes.c_void_p), ("dim", ctypes.c_int), ("interleaved", ctypes.c_int),
                ("factor", ctypes.c_float)]


def _turns(inv_freq):
    """round(f / (2 pi) * 2^64) mod 2^64 of each (finite) f, exact, as int64 words. 2 pi by Machin's formula,
    pi / 4 = 4 arctan(1/5) - arctan(1/239), in integers of 256 bits."""
    one = 1 << 256

    def arctan_inverse(n):
        total = term = one // n
        k = 1
        while term:
            term //= -n * n
            k += 2
            total += term // k
        return total
    two_pi = 8 * (4 * arctan_inverse(5) - arctan_inverse(239))
    out = []
    for f in inv_freq:
        num, den = float(f).as_integer_ratio()
        scaled = num * (one << 64)
        whole = (2 * scaled + den * two_pi) // (2 * den * two_pi) & ((1 << 64) - 1)
        out.append(whole - (1 << 64) if whole >> 63 else whole)
    return out


class Rotary:
    """A rotation of the first 2 * len(inv_freq) dims of each head by position: inv_freq in radians a position (a tensor
    or floats, taken as they are in 64 bits; 8 to 64 of them, a multiple of 8), pairs (i, i + dim / 2), or (2i, 2i + 1)
    when interleaved; factor multiplies the rotated values. Angles are exact at any position. See rotary_freqs."""
    __slots__ = ("freq", "dim", "interleaved", "factor", "_index", "_args", "_ref")

    def __init__(self, inv_freq, interleaved=False, factor=1.0, device="cuda"):
        f = torch.as_tensor(inv_freq, dtype=torch.float64).detach().cpu()
        if f.dim() != 1 or f.numel() % 8 or not 8 <= f.numel() <= 64 or not torch.isfinite(f).all():
            raise ValueError(f"Rotary: 8 to 64 finite frequencies, a multiple of 8, got {tuple(f.shape)}")
        if not abs(float(factor)) < 3.4e38:
            raise ValueError(f"Rotary: factor {factor}")
        self.freq = torch.tensor(_turns(f.tolist()), dtype=torch.int64).to(device)
        self.dim, self.interleaved, self.factor = 2 * f.numel(), bool(interleaved), float(factor)
        self._index = self.freq.get_device()
        self._args = RotaryArgs(self.freq.data_ptr(), self.dim, int(self.interleaved), self.factor)
        self._ref = ctypes.addressof(self._args)


def rotary_freqs(dim, theta, kind="plain", by=1.0, trained=None, fast=32.0, slow=1.0):
    """(inv_freq float64 [dim / 2], factor) for Rotary, inv_freq_i = theta^(-2i / dim), for contexts `by` times as long
    as the model was trained for. kind:
      plain   as they are
      linear  positions interpolated: inv_freq / by
      base    theta * by^(dim / (dim - 2)): the slowest pair interpolated, the fastest as it is
      parts   by each pair's turns r over the `trained` length: as they are from `fast` turns on, interpolated up to
              `slow`, in between by (r - slow) / (fast - slow); factor 0.1 ln(by) + 1"""
    if kind not in ("plain", "linear", "base", "parts"):
        raise ValueError(f"rotary_freqs: kind {kind!r}")
    if dim < 4 or dim % 2 or not theta > 0 or not by >= 1 or (kind == "parts" and (not trained or not fast > slow)):
        raise ValueError(f"rotary_freqs: dim {dim}, theta {theta}, by {by}, trained {trained}, turns {slow} to {fast}")
    if kind == "base":
        theta = theta * by ** (dim / (dim - 2))
    f = float(theta) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if kind == "linear":
        return f / by, 1.0
    if kind == "parts":
        keep = ((trained * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        return f * keep + f / by * (1 - keep), 0.1 * math.log(by) + 1
    return f, 1.0


def _paged_rows(name, cache, slots, pos):
    """(rows, slots pointer, pos pointer) of a call's rows."""
    if not isinstance(cache, PagedKv):
        raise TypeError(f"{name}: the cache must be an ops.PagedKv")
    shape, dev = slots.shape, cache._index
    if slots.dtype != torch.int64 or pos.dtype != torch.int32 or len(shape) != 1 or pos.shape != shape or \
            not slots.is_contiguous() or not pos.is_contiguous():
        raise ValueError(f"{name}: slots and pos must be contiguous int64 and int32 [rows], got {slots.dtype} {tuple(shape)}, "
                         f"{pos.dtype} {tuple(pos.shape)}")
    if slots.get_device() != dev or pos.get_device() != dev:
        raise ValueError(f"{name}: slots on {slots.device}, pos on {pos.device}, the cache on {cache.device}")
    return shape[0], slots.data_ptr(), pos.data_ptr()


def _paged_heads(name, what, t, cache, shape):
    """(pointer, row stride, head stride) of rows of this shape [rows, heads, head_dim]."""
    if t.shape != shape or t.dtype != cache.dtype:
        raise ValueError(f"{name}: {what} must be {cache.dtype} {shape}, got {t.dtype} {tuple(t.shape)}")
    if t.get_device() != cache._index:
        raise ValueError(f"{name}: {what} on {t.device}, the cache on {cache.device}")
    sr, sh, sd = t.stride()
    ptr = t.data_ptr()
    if (sr | sh | ptr >> 1) & 7 or (sd != 1 and shape[0]):
        raise ValueError(f"{name}: {what} needs a contiguous last dimension and 16-byte aligned rows (strides {t.stride()})")
    return ptr, sr, sh


def _paged_elsewhere(cache, fn, *args):
    """A call whose cache is not on the current device: made there."""
    _on_gpu(fn.__name__, cache)
    with torch.cuda.device(cache._index):
        return fn(*args)


def paged_append(k, v, cache, slots, pos):
    """K and V rows [rows, kv_heads, head_dim] (the cache's type, any row and head strides) to position pos[r] (int32) of
    slot slots[r] (int64). A row whose slot, position or page is outside the cache is not written; rows at one place leave
    a mixture there."""
    rows, sp, pp = _paged_rows("paged_append", cache, slots, pos)
    shape = rows, cache.kv_heads, cache.head_dim
    kp, kr, kh = _paged_heads("paged_append", "k", k, cache, shape)
    vp, vr, vh = _paged_heads("paged_append", "v", v, cache, shape)
    dev = cache._index
    if dev < 0 or dev != _current_device():
        return _paged_elsewhere(cache, paged_append, k, v, cache, slots, pos)
    rc = lib().m3x_paged_append(cache._ref, kp, kr, kh, vp, vr, vh, sp, pp, rows, _raw_stream(dev))
    if rc:
        check(rc, "paged_append")


def qk_norm_rope_paged(qkv, q_out, cache, slots, pos, rotary, wq, wk, eps, heads):
    """q|k|v rows [rows, (heads + 2 kv_heads) * head_dim] of a step: each head of q and k RMS-normed with wq, wk
    [head_dim] (both None: not normed) and rotated at its row's position, queries to q_out [rows, heads, head_dim], keys
    and values into the cache as paged_append does. Everything in the cache's type; fp32 arithmetic, rounded once.
    q_out does not overlap qkv."""
    name = "qk_norm_rope_paged"
    rows, sp, pp = _paged_rows(name, cache, slots, pos)
    D, width = cache.head_dim, (heads + 2 * cache.kv_heads) * cache.head_dim
    if qkv.shape != (rows, width) or heads < 1:
        raise ValueError(f"{name}: qkv must be [{rows}, {width}], got {tuple(qkv.shape)}")
    if not isinstance(rotary, Rotary) or rotary.dim > D:
        raise ValueError(f"{name}: rotary must be an ops.Rotary of at most {D} dims")
    op, orow, oh = _paged_heads(name, "q_out", q_out, cache, (rows, heads, D))
    qp, (s_qkv, s_one) = qkv.data_ptr(), qkv.stride()
    if qkv.dtype != cache.dtype or qkv.get_device() != cache._index or rotary._index != cache._index:
        raise ValueError(f"{name}: qkv must be {cache.dtype} on {cache.device}, as the rotation, got {qkv.dtype} on "
                         f"{qkv.device}")
    if (s_qkv | qp >> 1) & 7 or (s_one != 1 and rows):
        raise ValueError(f"{name}: qkv needs a contiguous last dimension and 16-byte aligned rows (strides {qkv.stride()})")
    wqp = wkp = 0
    if wq is not None or wk is not None:
        if wq is None or wk is None or wq.numel() != D or wk.numel() != D:
            raise ValueError(f"{name}: wq and wk are two vectors of {D}, or both None")
        wqp, wkp = wq.data_ptr(), wk.data_ptr()
        if (wqp | wkp) & 15 or wq.dtype != cache.dtype or wk.dtype != cache.dtype or not wq.is_contiguous() or \
                not wk.is_contiguous() or wq.get_device() != cache._index or wk.get_device() != cache._index:
            raise ValueError(f"{name}: wq and wk must be contiguous, 16-byte aligned {cache.dtype} on {cache.device}")
    dev = cache._index
    if dev < 0 or dev != _current_device():
        return _paged_elsewhere(cache, qk_norm_rope_paged, qkv, q_out, cache, slots, pos, rotary, wq, wk, eps, heads)
    rc = lib().m3x_qk_norm_rope_paged(cache._ref, qp, s_qkv, op, orow, oh, sp, pp, rotary._ref, wqp, wkp, eps, rows, heads,
                                      _raw_stream(dev))
    if rc:
        check(rc, name)


def paged_read(cache, slots, pos, k, v):
    """k, v [rows, kv_heads, head_dim] (the cache's type, any row and head strides) = position pos[r] of slot slots[r];
    zeros where there is none."""
    rows, sp, pp = _paged_rows("paged_read", cache, slots, pos)
    shape = rows, cache.kv_heads, cache.head_dim
    kp, kr, kh = _paged_heads("paged_read", "k", k, cache, shape)
    vp, vr, vh = _paged_heads("paged_read", "v", v, cache, shape)
    dev = cache._index
    if dev < 0 or dev != _current_device():
        return _paged_elsewhere(cache, paged_read, cache, slots, pos, k, v)
    rc = lib().m3x_paged_read(cache._ref, sp, pp, kp, kr, kh, vp, vr, vh, rows, _raw_stream(dev))
    if rc:
        check(rc, "paged_read")


NARROW_COLS, WIDE_COLS = 32, 128  # columns (rows x query heads of a kv head) that a workgroup of either kernel takes


def paged_tiles(runs, heads, kv_heads, narrow_cols=NARROW_COLS, cut=0):
    """The tiles of paged_attn for rows laid out as runs, (first row, rows, first position) each, of one slot at
    consecutive positions: (narrow, wide), int32 [n, 2] of (first row, rows). A run of up to narrow_cols columns is one narrow
    tile, a longer one wide tiles of up to 128 columns and about the same size; with cut > 0 narrow tiles of up to `cut`
    columns instead, a run's one behind the other (they read the same keys at about the same time: 32 runs of 32 rows onto
    500 keys 19.7 us, dealt by their keys alone 22.8). Those with the most keys come first, so that the last ones to finish
    are short (61 rows of up to 4000 keys 93 us, in no order 102 to 112; 30 x 5 of up to 3001 20.0, 21.4)."""
    G = heads // kv_heads
    r = np.asarray(runs, dtype=np.int64).reshape(-1, 3)
    r = r[r[:, 1] > 0]
    r = r[np.argsort(-(r[:, 2] + r[:, 1]), kind="stable")]
    few = (r[:, 1] * G <= narrow_cols) | (r[:, 1] == 1)
    most = max(1, (cut or WIDE_COLS) // G)
    long = r if cut else r[~few]
    n = np.where(few, 1, -(-r[:, 1] // most)) if cut else -(-long[:, 1] // most)
    of = np.repeat(np.arange(len(long)), n)
    at = np.arange(len(of)) - np.repeat(np.cumsum(n) - n, n)
    a, b = at * long[of, 1] // n[of], (at + 1) * long[of, 1] // n[of]
    order = np.lexsort((-at, of)) if cut else np.argsort(-(long[of, 2] + b), kind="stable")
    tiles = np.stack([long[of, 0] + a, b - a], 1)[order].astype(np.int32)
    return (tiles, tiles[:0]) if cut else (r[few, :2].astype(np.int32), tiles)


def _narrow_cols(head_dim):
    """Columns of the largest narrow tile: three 16 x 16 blocks fit two workgroups a CU with heads of 64 (measured on
    MI355X, 40 columns, us against 32 and 128: 30 tiles of up to 3001 keys 22 / 25 / 28, 100 of 2048 40 / 72 / 50)."""
    return 48 if head_dim == 64 else NARROW_COLS


class PagedPlan:
    """How paged_attn runs a step's rows, for all its layers and for every step of the same row layout: runs as in
    paged_tiles (rows in none are left as they are), the heads, the largest context that the rows will see (a rule's
    input, no limit), window and sinks (see paged_attn). `workspace`: bytes that a call needs. The plan holds counters that
    a call leaves as it found them: calls that may run at the same time need a plan and a workspace each."""
    __slots__ = ("rows", "heads", "kv_heads", "head_dim", "window", "sinks", "launches", "workspace", "_index", "_calls",
                 "_arrived", "_apart")

    def __init__(self, runs, heads, kv_heads, head_dim, max_ctx, window=0, sinks=0, device="cuda"):
        if kv_heads < 1 or heads < 1 or heads % kv_heads:
            raise ValueError(f"PagedPlan: {heads} query heads over {kv_heads} kv heads")
        r = self._runs(runs)
        if not 0 <= window < 1 << 31 or not 0 <= sinks < 1 << 31:
            raise ValueError(f"PagedPlan: window {window}, sinks {sinks}")
        self._begin(int((r[:, 0] + r[:, 1]).max()) if len(r) else 0, heads, kv_heads, head_dim, window, sinks)
        for i, (x, of, wide) in enumerate(self._deal(r, _narrow_cols(head_dim))):
            if not len(x):
                continue
            # the runs' own contexts, where they are what the plan is made for and not placeholders
            ends = (of[:, 2] + of[:, 1]).clip(0)
            mean = int(ends.mean()) if wide or 2 * ends.max() >= max_ctx else None
            every = len(x) == self.rows and (x[:, 1] == 1).all() and (x[:, 0] == np.arange(self.rows)).all()
            most, caps = int(x[:, 1].max()), None if i else self._caps(of)
            if caps is not None:
                x, every = np.stack([x[:, 0], x[:, 1] | caps << 16], 1), False
            tiles = None if every else torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(device)
            self._add(tiles, len(x), most, max_ctx, wide, mean)
            if caps is not None:
                self.launches[-1] = (*self.launches[-1][:4], int(caps.max()))
        self._finish(torch.device(device))

    @staticmethod
    def _runs(runs):
        r = np.asarray(runs, dtype=np.int64).reshape(-1, 3)
        r = r[r[:, 1] != 0]
        if (r[:, :2] < 0).any() or (r[:, 0] + r[:, 1] >= 1 << 31).any():
            raise ValueError("PagedPlan: runs are (first row, rows, first position)")
        o = r[np.argsort(r[:, 0], kind="stable")]
        if (o[1:, 0] < o[:-1, 0] + o[:-1, 1]).any():
            raise ValueError("PagedPlan: a row is in two runs")
        return r

    def _deal(self, r, narrow_cols, room=65535, long_cols=0, together=False):
        """What each launch gets of the runs: (tiles, the runs that they are of, whether wide) of the single rows, of the
        narrow tiles and of the wide ones. Runs of up to narrow_cols columns are one narrow tile; longer ones are cut into
        narrow tiles where _few says so or they have no more than long_cols columns. Single rows go along with up to `room`
        narrow tiles where they are up to a workgroup a CU, or if `together`.

        Measured on MI355X (16/8 heads of 128, us): 8 rows of 2048 keys beside a prompt of 56 20 together, 33 apart; 24
        beside one of 488 onto 1000 keys 40, 50, beside one of 1000 42, 64; 64 beside one of 192 97, 90; 224 beside one of
        288 317, 286: a kernel for more columns reads many single rows' keys more slowly, 64 rows of 2048 95 us against
        80."""
        G = self.heads // self.kv_heads
        single, rest = r[r[:, 1] == 1], r[r[:, 1] > 1]
        none = np.empty((0, 2), dtype=np.int32)
        cut = paged_tiles(rest, self.heads, self.kv_heads, narrow_cols, cut=NARROW_COLS)[0]
        short, wide = rest, none
        if len(rest) and (rest[:, 1] * G > narrow_cols).any():
            ends = (rest[:, 2] + rest[:, 1]).clip(0)
            if not self._few(len(cut) * self._blocks(cut, NARROW_COLS), int(ends.mean())):
                long = rest[:, 1] * G > max(narrow_cols, long_cols)
                short = rest[~long]
                cut = paged_tiles(short, self.heads, self.kv_heads, narrow_cols, cut=NARROW_COLS)[0]
                wide = paged_tiles(rest[long], self.heads, self.kv_heads, narrow_cols)[1]
        live = int((single[:, 2] >= 0).sum())
        if together or (len(single) and len(cut) and len(single) + len(cut) <= room and
                        live * self._blocks(single, NARROW_COLS) <= 256):
            short, single = np.concatenate([single, short]), single[:0]
            cut = paged_tiles(short, self.heads, self.kv_heads, narrow_cols, cut=NARROW_COLS)[0]
        elif self.uneven(single):
            single = single[np.argsort(-single[:, 2], kind="stable")]
        if live == 0 and len(single) and len(wide) and room == 65535:  # for their zeros, instead of a launch of their own
            wide, single = np.concatenate([wide, single[:, :2]]), single[:0]
        return (single[:, :2], single, False), (cut, short, False), (wide, rest, True)

    def _ends(self, runs):
        """Keys that the runs' last rows see, about."""
        return (runs[:, 2] + runs[:, 1]).clip(0, self.window + self.sinks + 1 if self.window else None)

    def _caps(self, runs):
        """Splits a tile for single rows of uneven contexts: chunks of 256 to 800 keys that come to two to three workgroups a
        CU; none beyond two a CU without. Measured on MI355X (16/8 heads of 128, rows of up to 4000 keys, us: none, chunks of
        400 / 600 / 800 / 1000 / 1600 keys): 32 rows 67, 56.5 / 56.0 / 53.8 / 55.1 / 65.6; 64 rows 93.8, 97 / 97 / 91.8 / 97 /
        95; 128 rows 168, 177 to 194. The rule was made at heads of 128; at heads of 64 (16/8): 32 rows 32.7, 31.6 / 32.1 /
        37.4 / 36.9 / 36.0, the rule 37.9; 64 rows 54.3, 54.5 / 52.4 / 51.3 / 52.0 / 57.4, the rule 51.2; 128 rows 96.7, 97 to
        106."""
        ends = self._ends(runs)
        one = self._blocks(runs, 16)
        if not self.uneven(runs) or len(runs) * one > 512:
            return None
        return (-(-ends // min(800, max(256, int(ends.sum()) * one // 640)))).clip(1, 16)

    def uneven(self, runs):
        """Whether the longest of the runs has more than 4/3 of their mean's keys."""
        ends = self._ends(np.asarray(runs))
        return len(ends) > 0 and 3 * int(ends.max()) > 4 * ends.mean()

    def _blocks(self, tiles, cols):
        """Workgroups a tile (and split)."""
        return self.kv_heads * -(-int(tiles[:, 1].max(initial=0)) * (self.heads // self.kv_heads) // cols)

    def _few(self, blocks, keys):
        """Whether prompts go through narrow tiles, cut to 32 columns: `blocks` workgroups of about `keys` keys each.

        Each reads its keys by itself, where the wide kernel's 128 columns share them, and starts sooner. Measured on
        MI355X (16/8 heads of 128; blocks, us cut / wide): 32 rows onto 300 keys (16) 9.8 / 15.3, 64 onto 4000 (32) 17.3 /
        22.2, 200 onto 2000 (104) 21.1 / 23.0, 512 onto 2048 (256) 25.8 / 28.8, 32 x 32 onto 500 (512) 19.5 / 22.6, 16 x 64
        onto 1000 (512) 27.7 / 30.5; on the other side 256 rows onto 6000 (128) 39.5 / 34.1, 64 onto 32000 (32) 48 / 41, 512
        onto 6000 (256) 59 / 47, 5 x 200 onto 1000 (520) 34.8 / 28.7, 40 x 32 onto 500 (640) 26.0 / 25.0. Heads of 64 take
        the same side (16/8 heads): 7.7 / 12.4, 13.1 / 15.6, 16.1 / 16.2, 21.3 / 21.2, 13.8 / 16.8, 19.7 / 24.4; 28.1 / 23.4,
        35.3 / 31.8, 44.2 / 35.1, 24.8 / 23.6, and, where cut would be faster, 17.7 / 19.2."""
        keys = min(keys, self.window + self.sinks + NARROW_COLS) if self.window else keys
        return blocks <= 512 and blocks * keys <= 600_000

    @classmethod
    def reserve(cls, rows, heads, kv_heads, head_dim, max_ctx, window=0, sinks=0, device="cuda", single=False):
        """A plan for any layout of up to `rows` rows (single: in runs of one row), what a captured graph launches: before a
        call, `tiles` of its runs go into the tensors of its `launches`: single rows (up to two workgroups a CU together with
        the next), narrow tiles and, for more rows than _few takes if all are one prompt, wide ones. A launch that gets no
        tile costs 1 to 3 us."""
        if kv_heads < 1 or heads < 1 or heads % kv_heads or rows < 1:
            raise ValueError(f"PagedPlan: {rows} rows, {heads} query heads over {kv_heads} kv heads")
        self = cls([], heads, kv_heads, head_dim, max_ctx, window, sinks, device)
        G = heads // kv_heads
        few, most = max(1, NARROW_COLS // G), max(1, WIDE_COLS // G)
        self.rows = rows
        one = self._blocks(np.array([[0, 1]]), NARROW_COLS)
        self._apart = single or rows * one > 512  # single rows have a launch of their own
        if single:  # as many splits as even rows take, and room for uneven ones'
            self._reserve(rows, 1, False, device)
            most = paged_attn_splits(rows * one, max_ctx, self.launches[0][3], head_dim=head_dim)
            self.launches[0] = (*self.launches[0][:4], max(most, min(8, 1536 // (rows * one), -(-max_ctx // 800))))
            self._finish(torch.device(device))
            return self
        if self._apart:
            self._reserve(rows, 1, False, device)
        # runs of two rows and more: a tile's part of them is the largest where one row more makes two tiles
        n = rows if not self._apart else -(-rows * 2 // (few + 1)) if few < 3 else rows // 2
        self._reserve(n, min(few, rows), False, device)
        if not self._few(-(-rows * G // NARROW_COLS) * kv_heads, max_ctx):
            self._reserve(2 * rows // most + 1, min(most, rows), True, device)
        self._finish(torch.device(device))
        return self

    def _reserve(self, n, tile_rows, wide, device):
        """A launch of up to n tiles, with splits for few of them: up to 2048 workgroups, most of which have nothing to do (64
        rows, all of a prompt onto 3900 keys 40 us unsplit, 31 so; onto 16 keys 7.9 and 8.1)."""
        tiles = torch.zeros(n, 2, dtype=torch.int32).to(device)
        self._add(tiles, n, tile_rows, 0, wide)
        cols = self.launches[-1][3]
        blocks = n * self._blocks(np.array([[0, tile_rows]]), cols)
        self.launches[-1] = (*self.launches[-1][:4], 1 if tile_rows == 1 < self.rows else max(1, min(16, 2048 // blocks)))

    def tiles(self, runs):
        """A reserved plan's tiles for these runs, one array of its tensor's size for each launch, rows as they come with
        the splits that their number and keys ask for."""
        r = self._runs(runs)
        if len(r) and (r[:, 0] + r[:, 1]).max() > self.rows:
            raise ValueError(f"PagedPlan: runs past the {self.rows} rows that the plan is for")
        if len(self.launches) == self._apart and (r[:, 1] > 1).any():
            raise ValueError(f"PagedPlan: a run of {r[:, 1].max()} rows, reserved for single ones")
        wide = self.launches[-1][3] == WIDE_COLS
        lists = self._deal(r, 0, self.launches[-1 - wide][1], WIDE_COLS // 2 if wide else 1 << 31, not self._apart)
        lists = lists[not self._apart:]
        out = []
        for i, ((x, of, _), (_, n, tile_rows, cols, splits)) in enumerate(zip(lists, self.launches)):
            if len(x) > n:
                raise ValueError(f"PagedPlan: {len(x)} tiles, reserved for {n}")
            full = np.zeros((n, 2), dtype=np.int32)
            full[:len(x)] = x[:, :2]
            caps = self._caps(of) if self._apart and i == 0 else None
            if caps is not None:
                full[:len(x), 1] |= np.minimum(caps, splits).astype(np.int32) << 16
            elif splits > 1 and len(x):
                seen = self.window + self.sinks + tile_rows if self.window else 1 << 30
                ends = (of[:, 2] + of[:, 1]).clip(0, seen)
                blocks = len(x) * self._blocks(x, cols)
                s = paged_attn_splits(blocks, int(ends.max()), cols, int(ends.mean()), blocks * cols, self.head_dim)
                full[:len(x), 1] |= min(s, splits) << 16
            out.append(full)
        return out

    def _begin(self, rows, heads, kv_heads, head_dim, window, sinks):
        self.rows, self.heads, self.kv_heads, self.head_dim = rows, heads, kv_heads, head_dim
        self.window, self.sinks, self.launches, self._apart = int(window), int(sinks), [], False

    def _add(self, tiles, n, tile_rows, max_ctx, wide=False, mean_ctx=None):
        if n > 65535:
            raise ValueError(f"PagedPlan: {n} tiles, a call holds 65535")
        G = self.heads // self.kv_heads
        cols = WIDE_COLS if wide else 16 if tile_rows * G <= 16 else NARROW_COLS
        if cols == NARROW_COLS < tile_rows * G <= _narrow_cols(self.head_dim):
            cols = _narrow_cols(self.head_dim)
        blocks = n * self.kv_heads * -(-tile_rows * G // cols)
        seen = self.window + self.sinks + tile_rows if self.window else max_ctx
        keys, mean = min(max_ctx, seen), min(max_ctx if mean_ctx is None else mean_ctx, seen)
        columns = blocks * min(cols, tile_rows * G)
        self.launches.append((tiles, n, tile_rows, cols,
                              paged_attn_splits(blocks, keys, cols, mean, columns, self.head_dim)))

    def _finish(self, device):
        self.workspace = max([0] + [int(lib().m3x_paged_attn_workspace(n, self.kv_heads, self.heads, tr, cols,
                                                                       self.head_dim, splits))
                                    for _, n, tr, cols, splits in self.launches])
        if device.type == "cuda":
            self._index = torch.cuda.current_device() if device.index is None else device.index
        else:
            self._index = -1
        G, split = self.heads // self.kv_heads, [x for x in self.launches if x[4] > 1 and x[3] != WIDE_COLS]
        need = max([0] + [n * self.kv_heads * -(-tr * G // cols) for _, n, tr, cols, _ in split])
        # (copied, not filled on the device: in place for every stream)
        self._arrived = torch.zeros(need, dtype=torch.int32).to(device) if need else None
        at = self._arrived.data_ptr() if need else 0
        self._calls = [(0 if t is None else t.data_ptr(), n, tr, cols, s, at) for t, n, tr, cols, s in self.launches]


def paged_attn_splits(blocks, keys, cols, mean_keys=None, columns=0, head_dim=128) -> int:
    """Workgroups that share a tile's keys, for `blocks` (tiles x kv heads x blocks of `cols` columns) of up to `keys` keys
    each.

    Few columns: up to half a workgroup a CU without splits, as many as make one a CU of the mean's keys. At least 128 keys each
    for one row's heads (16 columns) up to 8 splits (the join is 1 us of 6 to 8: one row at 250 keys 5.8 whole, 6.4 split, at
    700 keys 9.8 / 8.4 / 7.1 / 6.6 at 1 / 2 / 4 / 8, at 1500 16.5 / 11.7 / 8.6 / 7.5), else 256, and three times as many to
    begin with (the join is 3 to 5: 64 rows onto 500 keys 12.4 whole, 13.6 to 17 split). More single rows: as many of up to
    four as even out what the CUs get. Measured on MI355X (graph-timed, us, 16/8 heads of 128, 1 / 2 / 3 / 4 splits): 20 rows
    of 2048 keys 40.4 / 38.5 / 30.8 / 32.9, 28 38.1 / 41.6 / 43.0 / 43.0, 34 67.5 / 57.2 / 53.8 / 52.2, 48 71.8 / 64.5 / 69.3
    / 66.5, 64 80 / 85 / - / 87, 100 144.5 / 137.4 / 136.7 / 136.3, 224 277 / 293; 40 of 1000 35.7 / 32.4 / 31.1 / 30.7; 48
    of a 1024-key window 40.0 / 37.1 / 39.4 / 42.4. One row of 2048 21.3 / 14.5 / - / 9.8, 8.0 at 8, 8.2 at 16; 16 rows 34.2 /
    24.4 / 28.8 / 24.9. 32 columns: 64 rows onto 4000 keys 40.7 / 28.8 / 20.5 / 17.3 / 21.5 at 1 / 2 / 4 / 8 / 16; 512 onto
    2048 25.8 / 32.1. 32/4 heads of 64: 2 rows at 120000 keys 73 / 44 / 48 / 56 at 16 / 32 / 64 / 128; 30 x 5 rows over up to
    3001 29.8 / 25.2 / 22.5 / 21.1 / 25.0 at 1 / 2 / 3 / 4 / 5.

    Prompts: the least of what the tiles' turns of 32 keys take (1.05 us for one of two groups of waves that share a
    workgroup's keys, which they do up to a workgroup a CU; 0.52 for each of more workgroups that share a CU; the longest
    tile alone 0.75) and, from two on, the join's launch and partial results (3 us, 3 TB/s). Measured: 512 rows over 2048
    keys 43.9 / 33.5 / 27.1 / 32.5 at 1 / 2 / 4 / 8; 64 rows over 32000 77 / 49 / 40 at 8 / 16 / 32; 8 x 200 rows
    over 500 21.0 / 31.0 at 1 / 2. Heads of 64, whose turns are shorter, go by the same figures (16/8 heads, chosen first):
    512 rows over 2048 20.5 at 4, 34.2 / 25.3 / 19.4 at 1 / 2 / 8; 64 over 32000 31.9 at 32, 64 / 41 at 8 / 16; 8 x 200 over
    500 15.1 at 1, 21.6 at 2; 1024 onto 8000 73 at 2, 64 at 4; 4096 onto 4000 161 to 170 at 1, 150 / 146 at 2 / 4."""
    blocks, mean_keys = max(blocks, 1), keys if mean_keys is None else max(mean_keys, 1)
    if cols != WIDE_COLS:
        if blocks > 128 and cols == 16:
            def cost(s):  # the CU with the most workgroups sets the time; from two on the join
                return 0.0195 * head_dim / 128 * -(-blocks * s // 256) * mean_keys / s + (2.5 + 0.5 * s if s > 1 else 0)
            best = min((s for s in (1, 2, 3, 4) if s == 1 or s * 256 <= keys), key=cost)
            return best if cost(best) < 0.97 * cost(1) else 1
        if keys < (384 if cols == 16 else 768):
            return 1
        most = min(max(8, keys // 256), keys // 128, 64) if cols == 16 else min(keys // 256, 64)
        return max(1, min(256 * keys // max(1, blocks * mean_keys), most))

    def time(s):
        work = blocks * s
        if work <= 256:
            turns = 1.05 * keys / (64 * s)
        else:
            turns = max(0.52 * -(-work // 256) * mean_keys / (32 * s), 0.75 * keys / (32 * s))
        return turns + (3 + s * columns * head_dim * 8 / 3e6 if s > 1 else 0)
    return min((s for s in (1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64) if s == 1 or s * 128 <= keys), key=time)


def paged_attn(q, cache, out, slots, pos, scale, plan, workspace=None):
    """out[r, h] = softmax(scale q[r, h] . K^T) V over the positions j of slot slots[r] that row r at position p = pos[r]
    sees: j <= p and, with a window (plan.window > 0), j > p - window or j < plan.sinks. q, out [rows, heads, head_dim]
    (the cache's type, any row and head strides). A row that sees nothing gets zeros (pos[r] < 0, a slot outside the
    cache, positions in no page); a row in none of the plan's runs is left as it is. The rows of a run are of one slot at
    consecutive positions: its first row's are read. workspace: a tensor of plan.workspace bytes, or None when that is 0.
    Scores q . k are below 2^127 in size, |scale| is at most 2^126."""
    rows, sp, pp = _paged_rows("paged_attn", cache, slots, pos)
    if not isinstance(plan, PagedPlan):
        raise TypeError("paged_attn: the plan must be an ops.PagedPlan")
    heads = plan.heads
    if plan.kv_heads != cache.kv_heads or plan.head_dim != cache.head_dim or plan.rows > rows or plan._index != cache._index:
        raise ValueError(f"paged_attn: a plan of {plan.rows} rows, {heads} / {plan.kv_heads} heads of {plan.head_dim} for "
                         f"{rows} rows over {cache.kv_heads} kv heads of {cache.head_dim} on {cache.device}")
    shape = rows, heads, plan.head_dim
    qp, qr, qh = _paged_heads("paged_attn", "q", q, cache, shape)
    op, orow, oh = _paged_heads("paged_attn", "out", out, cache, shape)
    if not abs(scale) <= 2.0 ** 126:
        raise ValueError(f"paged_attn: |scale| must be at most 2^126, got {scale}")
    ws, ws_bytes = 0, 0
    if plan.workspace:
        if workspace is not None:
            ws, ws_bytes = workspace.data_ptr(), workspace.numel() * workspace.element_size()
        if ws_bytes < plan.workspace:
            raise ValueError(f"paged_attn: a workspace of {plan.workspace} bytes is needed, got {ws_bytes}")
        if not workspace.is_contiguous() or ws % 16 or workspace.get_device() != cache._index:
            raise ValueError(f"paged_attn: the workspace must be contiguous, 16-byte aligned and on {cache.device}")
    dev = cache._index
    if dev < 0 or dev != _current_device():
        return _paged_elsewhere(cache, paged_attn, q, cache, out, slots, pos, scale, plan, workspace)
    fn, stream = lib().m3x_paged_attn, _raw_stream(dev)
    for tiles, n, tile_rows, cols, splits, arrived in plan._calls:
        rc = fn(cache._ref, qp, qr, qh, op, orow, oh, sp, pp, tiles, n, tile_rows, cols, scale, rows, heads, plan.window,
                plan.sinks, splits, ws, ws_bytes, arrived, stream)
        if rc:
            check(rc, "paged_attn")


# ---------------------------------------------------------------- Mimi decode (serve/fast_codec.py)
def rvq_decode(codes, tables, out):
    """out[b] = [table_0[codes[b, 0]] | sum over q >= 1 of table_q[codes[b, q]]]; tables [nq, n_codes, dim]."""
    _dev(codes, tables, out)
    nq, n_codes, dim = tables.shape
    check(lib().m3x_rvq_decode(_p(codes), codes.stride(0), _p(tables), _p(out), out.stride(0), codes.shape[0], nq,
                               n_codes, dim, _dt3(tables), _stream()), "rvq_decode")


def dwconvt(x, w, tail, slots, out, k, s):
    """Depthwise transposed conv of one frame per seat with per-slot overlap tails; out [B * s, C]."""
    _dev(x, w, tail, slots, out)
    _index(slots=slots)
    check(lib().m3x_dwconvt(_p(x), x.stride(0), _p(w), _p(tail), tail.stride(0), _p(slots), _p(out), x.shape[0],
                            x.shape[1], k, s, _dt3(x), _stream()), "dwconvt")


def conv_gather(x, state, slots, cols, B, T, C, k, dil, use_elu, chunk):
    """GEMM rows of a causal conv with per-slot input history (state [slots, pad * C] or None when pad = 0);
    cols None only advances the history."""
    _dev(x, state, slots, cols)
    _index(slots=slots)
    check(lib().m3x_conv_gather(_p(x), x.stride(0), _p(state), 0 if state is None else state.stride(0), _p(slots),
                                _p(cols), 0 if cols is None else cols.stride(0), B, T, C, k, dil, int(use_elu), chunk,
                                _dt3(x), _stream()),
          "conv_gather")


def rows_op(g, out, bias=None, scale=None, res=None, use_elu=False):
    """out = act(res + scale * (g + bias)), act = ELU when use_elu; rows of g and out [rows, C]."""
    _dev(g, out, bias, scale, res)
    check(lib().m3x_rows_op(_p(g), g.stride(0), _p(bias), _p(scale), _p(res), 0 if res is None else res.stride(0),
                            _p(out), out.stride(0), out.shape[0], out.shape[1], int(use_elu), _dt3(g), _stream()),
          "rows_op")


def conv_gemm(x, w, y, bias=None, res=None, use_elu=False, gather=None):
    """y = act(res + (x @ W.T + bias)) for a packed W with N in {16, 32, 64, 128}; act = ELU when use_elu.
    gather = (state, slots, T, C, dil, pre_elu): x is the conv's input [B * T, C] and the product reads
    m3x_conv_gather's rows in place (the history is not advanced here)."""
    if not isinstance(w, PackedWeight):
        raise TypeError("conv_gemm: the weight must be packed with ops.pack_weight")
    st, slots, T, C, dil, pre = gather if gather is not None else (None, None, 0, 0, 1, False)
    _dev(x, w.data, y, bias, res, st, slots)
    _index(slots=slots)
    check(lib().m3x_conv_gemm(_p(x), x.stride(0), _p(w.data), _p(bias), _p(res), 0 if res is None else res.stride(0),
                              _p(y), y.stride(0), y.shape[0], w.N, w.K, int(use_elu), _p(st),
                              0 if st is None else st.stride(0), _p(slots), T, C, dil, int(pre), _dt3(x), _stream()),
          "conv_gemm")
    return y


def resid_ln(h, a, scale, w, b, eps, y):
    """h = h + scale * a in place (16-bit rounding once), then y = LayerNorm(h) with (w, b, eps); rows of 512."""
    _dev(h, a, scale, w, b, y)
    check(lib().m3x_resid_ln(_p(h), h.stride(0), _p(a), a.stride(0), _p(scale), _p(w), _p(b), _p(y), y.stride(0),
                             float(eps), h.shape[0], h.shape[1], _dt3(h), _stream()), "resid_ln")


def convt_overlap(cols, tail, slots, bias, out, B, Tin, C, k, s, chunk):
    """Overlap-add of a transposed conv's GEMM columns with per-slot tails; out [B * Tin * s, C]."""
    _dev(cols, tail, slots, bias, out)
    _index(slots=slots)
    check(lib().m3x_convt_overlap(_p(cols), cols.stride(0), _p(tail), tail.stride(0), _p(slots), _p(bias), _p(out),
                                  out.stride(0), B, Tin, C, k, s, chunk, _dt3(cols), _stream()), "convt_overlap")


def ring_attn(qkv, kring, vring, key_pos, tokens, slots, inv_freq, rope_scale, out, B, T, H, ring, window):
    """Sliding-window attention of T new tokens per seat over per-slot rings of post-RoPE keys."""
    _dev(qkv, kring, vring, key_pos, tokens, slots, inv_freq, out)
    _index(slots=slots)
    check(lib().m3x_ring_attn(_p(qkv), qkv.stride(0), _p(kring), _p(vring), _p(key_pos), _p(tokens), _p(slots),
                              _p(inv_freq), float(rope_scale), _p(out), out.stride(0), B, T, H, 64, ring, window,
                              _dt3(qkv), _stream()), "ring_attn")


def advance_tokens(tokens, slots, B, T, dummy):
    _dev(tokens, slots)
    _index(slots=slots)
    check(lib().m3x_advance_tokens(_p(tokens), _p(slots), B, T, dummy, _stream()), "advance_tokens")


def final_conv(x, state, slots, w, bias, pcm, B, T, C, k, chunk):
    """fp32 PCM of the last causal conv (C -> 1 channel) with per-slot history; pcm [B, >= T] float32."""
    _dev(x, state, slots, w, pcm)
    _index(slots=slots)
    check(lib().m3x_final_conv(_p(x), x.stride(0), _p(state), 0 if state is None else state.stride(0), _p(slots),
                               _p(w), float(bias), _p(pcm), pcm.stride(0), B, T, C, k, chunk, _dt3(x), _stream()),
          "final_conv")
