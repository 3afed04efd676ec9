// Writers and reader of the paged KV cache (layout: m3x_paged.h). The attention over it: paged_attn.hip.
#include "m3x_paged.h"

// mirror of M3xRotary (include/m3x.h)
struct M3xRotary {
  const uint64_t* freq;
  int dim, interleaved;
  float factor;
};

namespace {
// cos and sin of p * f turns times `factor`. f is a 64-bit binary fraction of a turn: the upper half of p f mod 2^64 is
// the turn's fraction within 2^-32 and p 2^-64 at any position, with two integer products. v_sin_f32 and v_cos_f32 take
// turns; measured over 2^20 fractions they are within 3.2 * 2^-24.
struct CosSin {
  float c, s;
};
__device__ __forceinline__ CosSin turn(uint32_t p, uint64_t f, float factor) {
  const int32_t part = (int32_t)(__umulhi(p, (uint32_t)f) + p * (uint32_t)(f >> 32));
  const float t = (float)part * 0x1p-32f;
  return {__builtin_amdgcn_cosf(t) * factor, __builtin_amdgcn_sinf(t) * factor};
}
__device__ __forceinline__ void st16_nt(uint16_t* p, const u16x8& x) {
  typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store(__builtin_bit_cast(u32x4_t, x), reinterpret_cast<u32x4_t*>(p));
}
}  // namespace

// q|k|v rows: every head of q and k normed (weights given) and rotated at the row's position, queries to q_out, keys and
// values into their pages. Arithmetic in fp32, one rounding at the end:
//   x' = x / sqrt(mean(x^2) + eps) * w;  (a, b) -> (a cos - b sin, b cos + a sin) for the pairs of the first `dim` dims,
//   (i, i + dim / 2) or (2i, 2i + 1).
// D / 8 threads a head, HB heads of one row one after another with the same angles. In the first layout a thread also
// loads its partner dims (from the cache the neighbour's load fills) instead of exchanging them.
// Bound by the launch and one memory round trip up to some hundred rows (16/8 heads of 128: 1 row 2.9 us, 224 rows 4.1, 512
// 4.6), then by bytes: 2048 rows of 32/8 heads of 128, half of each rotated, 50 MB in 11.1 us, 4.5 TB/s (a large copy: 4.9).
template <int DT, int D, int HB>
__global__ __launch_bounds__(256) void qk_norm_rope_paged_kernel(
    const uint16_t* __restrict__ qkv, long s_qkv, uint16_t* __restrict__ qo, long s_qo_b, long s_qo_h, Paged c,
    const int64_t* __restrict__ slots, const int32_t* __restrict__ pos, M3xRotary rot, const uint16_t* __restrict__ wq,
    const uint16_t* __restrict__ wk, float eps, int rows, int H) {
  constexpr int TPI = D / 8;
  const int t = threadIdx.x % TPI, d0 = 8 * t;
  const long item = (long)blockIdx.x * (256 / TPI) + threadIdx.x / TPI;
  const int KV = c.kv_heads, NH = H + KV, blocks = (NH + HB - 1) / HB;
  const long row = item / blocks;
  const int j0 = (int)(item % blocks) * HB;
  const bool active = row < rows;  // spare threads compute on row 0 and store nothing (heads reduce over lanes)
  const long r = active ? row : 0;
  const int half = rot.dim / 2;
  // the thread's partner dims: another thread's in the first layout, its own in the second
  const bool turned = d0 < rot.dim;
  const bool first = d0 < half;
  const int dp = turned && !rot.interleaved ? (first ? d0 + half : d0 - half) : d0;
  const uint16_t* src = qkv + r * s_qkv;
  const int p = pos[r];
  const long slot = slots[r];
  u16x8 xv[HB], pv[HB], vv[HB];
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    const long at = (long)min(j0 + i, NH - 1) * D;
    xv[i] = ld16(src + at + d0);
    pv[i] = ld16(src + at + dp);
  }
  // the rows' last loads beside the first: values (of key heads) and their place, asked for before the arithmetic
  const bool keys = j0 + HB > H;
  long at = -1;
  if (keys) {
#pragma unroll
    for (int i = 0; i < HB; ++i) vv[i] = ld16(src + (long)(min(max(j0 + i, H), NH - 1) + KV) * D + d0);
    at = c.at<D>(slot, 0, p);
  }
  float cs[8], sn[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) cs[e] = 1.f, sn[e] = 0.f;
  if (turned) {
    const uint32_t ps = (uint32_t)max(p, 0);
    if (rot.interleaved) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const CosSin a = turn(ps, rot.freq[(d0 + e) / 2], rot.factor);
        cs[e] = cs[e + 1] = a.c;
        sn[e] = -a.s, sn[e + 1] = a.s;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const CosSin a = turn(ps, rot.freq[(first ? d0 : d0 - half) + e], rot.factor);
        cs[e] = a.c;
        sn[e] = first ? -a.s : a.s;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < HB; ++i) {
    const int j = j0 + i;
    float x[8], y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = E<DT>::to_f(xv[i].v[e]);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = rot.interleaved ? x[e ^ 1] : E<DT>::to_f(pv[i].v[e]);
    if (wq) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
      const float inv = 1.f / sqrtf(group_sum<TPI>(ss) * (1.f / D) + eps);
      const uint16_t* w = j < H ? wq : wk;
      const u16x8 wx = ld16(w + d0), wy = ld16(w + dp);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] *= inv * E<DT>::to_f(wx.v[e]);
        y[e] *= inv * E<DT>::to_f(rot.interleaved ? wx.v[e ^ 1] : wy.v[e]);
      }
    }
    if (!active || j >= NH) continue;
    u16x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o.v[e] = E<DT>::from_f(turned ? fmaf(y[e], sn[e], x[e] * cs[e]) : x[e]);
    if (j < H) {
      st16(qo + row * s_qo_b + (long)j * s_qo_h + d0, o);
    } else {
      const long to = at + ((long)(j - H) << c.shift) * D + d0;
      if (at >= 0) {
        st16(c.k + to, o);
        st16(c.v + to, vv[i]);
      }
    }
  }
}

// K and V rows into their pages, D / 8 threads per (row, kv head): a copy, bound by the launch (8 heads of 128: 1 row 2.3
// us, 300 rows 2.9), then by bytes: 16384 rows, 134 MB in 22 us, 6.0 TB/s (what it writes stays in the memory-side cache).
template <int D>
__global__ __launch_bounds__(256) void paged_append_kernel(const uint16_t* __restrict__ k, long sk_r, long sk_h,
                                                           const uint16_t* __restrict__ v, long sv_r, long sv_h, Paged c,
                                                           const int64_t* __restrict__ slots,
                                                           const int32_t* __restrict__ pos, int rows) {
  constexpr int TPI = D / 8;
  const int d0 = 8 * (threadIdx.x % TPI);
  const long item = (long)blockIdx.x * (256 / TPI) + threadIdx.x / TPI;
  const long row = item / c.kv_heads;
  const int kh = (int)(item % c.kv_heads);
  if (row >= rows) return;
  const u16x8 kx = ld16(k + row * sk_r + kh * sk_h + d0);
  const u16x8 vx = ld16(v + row * sv_r + kh * sv_h + d0);
  const long at = c.at<D>(slots[row], kh, pos[row]);
  if (at < 0) return;
  st16(c.k + at + d0, kx);
  st16(c.v + at + d0, vx);
}

// Positions as rows, zeros where there is none; stored with the non-temporal hint (read once by their taker). Bound by the
// launch (300 positions of 8 heads of 128 2.7 us), then bytes: 65520 positions of 8 heads of 64, 268 MB in 41 us, 6.5 TB/s.
template <int D>
__global__ __launch_bounds__(256) void paged_read_kernel(Paged c, const int64_t* __restrict__ slots,
                                                         const int32_t* __restrict__ pos, uint16_t* __restrict__ k,
                                                         long sk_r, long sk_h, uint16_t* __restrict__ v, long sv_r,
                                                         long sv_h, int rows) {
  constexpr int TPI = D / 8;
  const int d0 = 8 * (threadIdx.x % TPI);
  const long item = (long)blockIdx.x * (256 / TPI) + threadIdx.x / TPI;
  const long row = item / c.kv_heads;
  const int kh = (int)(item % c.kv_heads);
  if (row >= rows) return;
  const long at = c.at<D>(slots[row], kh, pos[row]);
  u16x8 kx = zero_v8<M3X_BF16>(), vx = kx;
  if (at >= 0) {
    kx = ld16(c.k + at + d0);
    vx = ld16(c.v + at + d0);
  }
  st16_nt(k + row * sk_r + kh * sk_h + d0, kx);
  st16_nt(v + row * sv_r + kh * sv_h + d0, vx);
}

// ---------------------------------------------------------------------------------------------------------
namespace {
// whether D / 8 threads for each of `items` fit a launch (fewer than 2^32 threads)
bool paged_fits(long items, int head_dim) { return items * (head_dim / 8) < (1L << 32) - 256; }
int paged_rows_ok(const void* k, long sk_r, long sk_h, const void* v, long sv_r, long sv_h) {
  return !(((sk_r | sk_h | sv_r | sv_h) & 7) || !m3x_aligned16(k) || !m3x_aligned16(v));
}
}  // namespace

M3X_API int m3x_paged_append(const M3xPagedKv* cache, const void* k, long sk_r, long sk_h, const void* v, long sv_r,
                             long sv_h, const int64_t* slots, const int32_t* pos, int rows, void* stream) {
  Paged c;
  if (const int st = paged_take(cache, c)) return st;
  if (rows < 0) return M3X_EINVAL;
  if (rows == 0) return M3X_OK;
  if (!k || !v || !slots || !pos) return M3X_ENULL;
  const long items = (long)rows * c.kv_heads;
  if (!paged_rows_ok(k, sk_r, sk_h, v, sv_r, sv_h) || !paged_fits(items, cache->head_dim)) return M3X_EINVAL;
  const dim3 grid(m3x_ceil_div(items, 2048 / cache->head_dim));
#define M3X_PAGED_APPEND(DD)                                                                                          \
  hipLaunchKernelGGL(paged_append_kernel<DD>, grid, dim3(256), 0, (hipStream_t)stream, (const uint16_t*)k, sk_r, sk_h, \
                     (const uint16_t*)v, sv_r, sv_h, c, slots, pos, rows)
  if (cache->head_dim == 128) M3X_PAGED_APPEND(128);
  else M3X_PAGED_APPEND(64);
#undef M3X_PAGED_APPEND
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}

M3X_API int m3x_paged_read(const M3xPagedKv* cache, const int64_t* slots, const int32_t* pos, void* k, long sk_r,
                           long sk_h, void* v, long sv_r, long sv_h, int rows, void* stream) {
  Paged c;
  if (const int st = paged_take(cache, c)) return st;
  if (rows < 0) return M3X_EINVAL;
  if (rows == 0) return M3X_OK;
  if (!k || !v || !slots || !pos) return M3X_ENULL;
  const long items = (long)rows * c.kv_heads;
  if (!paged_rows_ok(k, sk_r, sk_h, v, sv_r, sv_h) || !paged_fits(items, cache->head_dim)) return M3X_EINVAL;
  const dim3 grid(m3x_ceil_div(items, 2048 / cache->head_dim));
#define M3X_PAGED_READ(DD)                                                                                     \
  hipLaunchKernelGGL(paged_read_kernel<DD>, grid, dim3(256), 0, (hipStream_t)stream, c, slots, pos, (uint16_t*)k, \
                     sk_r, sk_h, (uint16_t*)v, sv_r, sv_h, rows)
  if (cache->head_dim == 128) M3X_PAGED_READ(128);
  else M3X_PAGED_READ(64);
#undef M3X_PAGED_READ
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}

M3X_API int m3x_qk_norm_rope_paged(const M3xPagedKv* cache, const void* qkv, long s_qkv, void* q_out, long s_qo_b,
                                   long s_qo_h, const int64_t* slots, const int32_t* pos, const M3xRotary* rotary,
                                   const void* wq, const void* wk, float eps, int rows, int heads, void* stream) {
  Paged c;
  if (const int st = paged_take(cache, c)) return st;
  if (!rotary) return M3X_ENULL;
  const int D = cache->head_dim;
  if (rows < 0 || heads <= 0 || rotary->dim < 16 || rotary->dim > D || rotary->dim % 16) return M3X_EINVAL;
  if (rows == 0) return M3X_OK;
  if (!qkv || !q_out || !slots || !pos || !rotary->freq || !wq != !wk) return M3X_ENULL;
  if (((s_qkv | s_qo_b | s_qo_h) & 7) || !m3x_aligned16(qkv) || !m3x_aligned16(q_out) || !m3x_aligned16(wq) ||
      !m3x_aligned16(wk) || ((uintptr_t)rotary->freq & 7u))
    return M3X_EINVAL;
  const long nh = (long)heads + c.kv_heads;
  // q_out apart from qkv: a thread also reads dims of its head that another thread writes
  const uintptr_t i0 = (uintptr_t)qkv, i1 = i0 + 2 * ((rows - 1) * s_qkv + (nh + c.kv_heads) * D);
  const uintptr_t o0 = (uintptr_t)q_out, o1 = o0 + 2 * ((rows - 1) * s_qo_b + (heads - 1L) * s_qo_h + D);
  if (o0 < i1 && i0 < o1) return M3X_EINVAL;
  if (heads > 65535 || !paged_fits(rows * nh, D)) return M3X_EINVAL;
  // four heads a thread share the angles once that leaves two waves a SIMD (16/8 heads of 128, us with four, with one: 1
  // row 4.4, 3.0, 1024 rows 7.6, 6.8, 2048 rows 10.5, 11.5)
  const int hb = rows * nh * (D / 8) >= 4L * 64 * 2048 ? 4 : 1;
  const dim3 grid(m3x_ceil_div(rows * ((nh + hb - 1) / hb), 2048 / D));
#define M3X_QKN(DT, DD, HB)                                                                                        \
  hipLaunchKernelGGL((qk_norm_rope_paged_kernel<DT, DD, HB>), grid, dim3(256), 0, (hipStream_t)stream,             \
                     (const uint16_t*)qkv, s_qkv, (uint16_t*)q_out, s_qo_b, s_qo_h, c, slots, pos, *rotary,        \
                     (const uint16_t*)wq, (const uint16_t*)wk, eps, rows, heads)
#define M3X_QKN_HB(DT, DD)      \
  if (hb == 4) M3X_QKN(DT, DD, 4); \
  else M3X_QKN(DT, DD, 1)
  if (cache->dtype == M3X_BF16) {
    if (D == 128) { M3X_QKN_HB(M3X_BF16, 128); }
    else { M3X_QKN_HB(M3X_BF16, 64); }
  } else {
    if (D == 128) { M3X_QKN_HB(M3X_F16, 128); }
    else { M3X_QKN_HB(M3X_F16, 64); }
  }
#undef M3X_QKN_HB
#undef M3X_QKN
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}
