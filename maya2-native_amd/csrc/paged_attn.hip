// Attention over the paged KV cache (layout: m3x_paged.h): chunks of new tokens and single tokens, with a window.
//
// out[r, h, :] = sum_j w_j v_j / sum_j w_j, w_j = exp(scale q[r, h] . k_j), over the positions j that row r at position p
// sees: j <= p and, with a window, j > p - window or j < sinks.
//
// The work comes as tiles (first row, rows): rows of one slot at consecutive positions. A tile's columns are its rows'
// query heads of one kv head, column c standing for row c / G, head c % G. Keys are the rows of the score product:
//   S^T = K . Q^T (MFMA 16x16x32)   lane (column li = l % 16, group lg = l / 16) holds keys 4 lg .. 4 lg + 3 of 16
//   softmax                         running maximum and sum in fp32, exp2; a lane keeps its own column's
//   O^T += V^T . P                  S^T's accumulators of two 16-key groups are the P operand as they stand
// A tile's keys are counted in steps of KT positions, first those of the sinks, then those from the window's begin on,
// and divided evenly among the splits; the splits' partial results are joined by a second launch.
#include <algorithm>
#include <cstring>

#include "m3x_paged.h"

namespace {
typedef uint32_t pg_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t pg_u2 __attribute__((ext_vector_type(2)));
typedef __bf16 pg_bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 pg_h2 __attribute__((ext_vector_type(2)));
typedef float pg_f2 __attribute__((ext_vector_type(2)));

// Weights stand at 2^up of their size: fp16's would lose precision below 2^-14, and a sum of bf16 ones times values near
// the format's largest would overflow where their mean does not.
template <int DT> constexpr float pg_up = DT == M3X_F16 ? 15.f : -24.f;

struct PagedAttn {
  const uint16_t* q;
  long sq_b, sq_h;
  uint16_t* out;
  long so_b, so_h;
  const int64_t* slots;
  const int32_t* pos;
  const int32_t* tiles;  // (first row, rows) pairs; NULL: tile t is row t
  float c;               // |scale| log2(e), not 0
  uint32_t q_flip;       // the sign bits of two query elements where scale < 0
  int rows, heads, G, tile_rows, blocks, window, sinks, splits;
  float* part;  // [columns][splits][D], then [columns][splits][2]: (reference, sum)
};

// a workgroup's place: a tile, a kv head, a block of the tile's columns; all uniform
struct Where {
  int tile, kh, block, first, n, p0;  // rows first .. first + n - 1 at positions p0 ..; n == 0: nothing to do
  long slot;
};
// x, the same in every lane, in a scalar register. The empty statement hides where x comes from: a value known to be
// uniform is left in vector registers where a division made it, and what is computed from it too, up to the buffer
// loads' addresses, each then in a loop over the lanes.
__device__ __forceinline__ int pg_uniform(int x) {
  asm("" : "+v"(x));
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ long pg_uniform(long x) {
  return (long)((uint64_t)(uint32_t)pg_uniform((int)x) | (uint64_t)(uint32_t)pg_uniform((int)(x >> 32)) << 32);
}
__device__ __forceinline__ Where pg_where(const Paged& c, const PagedAttn& a, uint32_t item) {
  Where w;
  const uint32_t th = item / (uint32_t)a.blocks;
  w.block = pg_uniform((int)(item - th * a.blocks));
  w.tile = pg_uniform((int)(th / (uint32_t)c.kv_heads));
  w.kh = pg_uniform((int)(th - (uint32_t)w.tile * c.kv_heads));
  w.first = w.tile;
  w.n = 1;
  if (a.tiles) {
    w.first = pg_uniform(a.tiles[2 * w.tile]);
    w.n = pg_uniform(a.tiles[2 * w.tile + 1]);
  }
  w.slot = -1;
  w.p0 = -1;
  if (w.first < 0 || w.first >= a.rows || w.n <= 0) {
    w.n = 0;
    return w;
  }
  w.n = min(min(w.n, a.tile_rows), a.rows - w.first);
  w.slot = pg_uniform((long)a.slots[w.first]);
  w.p0 = min(pg_uniform(a.pos[w.first]), 1 << 30);  // positions count past it in 32 bits, and the cache ends before
  return w;
}

// a tile's keys in steps of KT positions
template <int KT> struct Keys {
  int last;          // the last key that some row sees; -1: none
  int sink, skip, nt;  // steps 0 .. sink - 1, then from sink + skip on; their number
  int per, active;   // steps a split; splits that have some
  __device__ __forceinline__ Keys(const Paged& c, const PagedAttn& a, const Where& w, int least) {
    const int cap = c.width << c.shift;
    last = w.slot < 0 || w.slot >= c.slots || w.n == 0 || w.p0 < -w.n ? -1 : min(w.p0 + w.n - 1, cap - 1);
    const int lo = a.window ? max(0, w.p0 - a.window + 1) / KT : 0;
    sink = a.window ? min((min(a.sinks, last + 1) + KT - 1) / KT, lo) : 0;
    skip = pg_uniform(lo - sink);  // (opaque: it also serves lanes that branch, and would be made anew there)
    nt = last < 0 ? 0 : sink + max(0, last / KT + 1 - lo);
    per = pg_uniform(max(least, (nt + a.splits - 1) / a.splits));
    active = pg_uniform((nt + per - 1) / per);
  }
  __device__ __forceinline__ int key(int i) const { return (i + (i < sink ? 0 : skip)) * KT; }
};

// a column's row and head, and the keys it sees
struct Col {
  int j, h, p;  // row of the tile, head of the kv head's G, position
  bool live;
  __device__ __forceinline__ Col(const PagedAttn& a, const Where& w, int col) {
    j = (int)((uint32_t)col / (uint32_t)a.G);
    h = col - j * a.G;
    live = j < w.n;
    p = live ? w.p0 + j : -1;
  }
};
// whether keys key .. of a step may be hidden from some row that another row sees, or lie outside
__device__ __forceinline__ bool pg_hidden(int key, int p, int low, int sinks) { return key > p || (key <= low && key >= sinks); }
// the largest position that the window hides from a row at p (-1: none)
__device__ __forceinline__ int pg_low(const PagedAttn& a, int p) { return a.window ? p - a.window : -1; }

template <int DT> __device__ __forceinline__ uint32_t pg_pack(float x, float y) {
  if constexpr (DT == M3X_F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((pg_f2{x, y}), pg_h2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector((pg_f2{x, y}), pg_bf2));
}
// acc + both numbers of w in fp32
template <int DT> __device__ __forceinline__ float pg_add2(uint32_t w, float acc) {
  if constexpr (DT == M3X_F16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(pg_h2, w), __builtin_bit_cast(pg_h2, 0x3C003C00u), acc, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pg_bf2, w), __builtin_bit_cast(pg_bf2, 0x3F803F80u), acc, false);
}
// bits 15 and 31: which of the two numbers of w are infinite or NaN (an exponent of ones carries into the sign's place)
template <int DT> __device__ __forceinline__ uint32_t pg_wild(uint32_t w) {
  constexpr uint32_t ones = DT == M3X_F16 ? 0x7C007C00u : 0x7F807F80u, unit = DT == M3X_F16 ? 0x04000400u : 0x00800080u;
  return ((w & ones) + unit) & 0x80008000u;
}
// w with those numbers 0
template <int DT> __device__ __forceinline__ uint32_t pg_tame(uint32_t w) {
  const uint32_t x = pg_wild<DT>(w);
  return w & ~((x >> 15) * 0xFFFFu);  // 0xFFFF in each half that has its bit
}
// the number of a half of w where it is infinite or NaN, else 0
template <int DT> __device__ __forceinline__ float pg_wild_number(uint16_t x) {
  return pg_wild<DT>(x) & 0x8000u ? E<DT>::to_f(x) : 0.f;
}

// A column's running maximum (raw score) and its reference ref = maximum * c, what weights' exponents are counted from:
// exp2(s c - ref). Any reference serves as long as all of a column's weights and its sum go by the same one, so its
// rounding is no error; kept finite (no row sees a key below -FLT_MAX).
__device__ __forceinline__ float pg_ref(float m, float c) { return fmaxf(m * c, -3.402823466e38f); }

// 4 outputs O / L (zeros for a column that saw nothing)
template <int DT> __device__ __forceinline__ void pg_store4(uint16_t* p, const f32x4_t& O, float L) {
  const float r = L == 0.f ? 0.f : 1.f / L;
  *reinterpret_cast<pg_u2*>(p) = pg_u2{pg_pack<DT>(O[0] * r, O[1] * r), pg_pack<DT>(O[2] * r, O[3] * r)};
}

// zeros for the block's columns
template <int COLS, int D, int NT> __device__ __forceinline__ void pg_zero(const PagedAttn& a, const Where& w, int tid) {
  for (int i = tid; i < COLS * (D / 4); i += NT) {
    const Col col(a, w, w.block * COLS + i / (D / 4));
    if (col.live)
      *reinterpret_cast<pg_u2*>(a.out + (long)(w.first + col.j) * a.so_b + (long)(w.kh * a.G + col.h) * a.so_h +
                                i % (D / 4) * 4) = pg_u2{0, 0};
  }
}

// 4 NI bytes at a lane's offset of a tile at a uniform address; a tile of `bytes` bytes: beyond it, zeros and no access
__device__ __forceinline__ __amdgpu_buffer_rsrc_t pg_ref_of(const uint16_t* base, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(base), 0, bytes, 0x00020000);
}
template <int NI> struct __align__(4 * NI) PgWords { uint32_t w[NI]; };
template <int NI, bool NT> __device__ __forceinline__ PgWords<NI> pg_load(__amdgpu_buffer_rsrc_t ref, uint32_t off) {
  constexpr int AUX = NT ? 2 : 0;
  PgWords<NI> r;
  if constexpr (NI == 4) {
    const pg_u4 x = __builtin_amdgcn_raw_buffer_load_b128(ref, off, 0, AUX);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = x[i];
  } else {
    const pg_u2 x = __builtin_amdgcn_raw_buffer_load_b64(ref, off, 0, AUX);
    r.w[0] = x[0];
    r.w[1] = x[1];
  }
  return r;
}

constexpr int NARROW_NW = 4;
template <int D> struct NarrowLds {
  __align__(16) float o[NARROW_NW][16][D + 4];
  float ref[NARROW_NW][16], l[NARROW_NW][16];
};
}  // namespace

// Tiles of up to 16 QT columns: single tokens, and the few rows of drafted ones. Bound by the keys' bytes. Each of the 4
// waves takes every fourth step of 32 keys, straight from memory to registers: K as the score product's operand, V as
// rows whose numbers byte permutes pair over keys. The waves' results are merged through LDS.
template <int DT, int D, int QT, bool NT>
__global__ __launch_bounds__(256, D == 64 && QT == 1 ? 3 : 2) void paged_narrow_kernel(Paged c, PagedAttn a) {
  constexpr int KT = 32, NW = NARROW_NW, KS = D / 32, NV = D / 32, COLS = 16 * QT;
  // NV: words of V a lane holds of a key (2 NV dims); AHEAD: steps that a wave's loads run ahead (two fill the registers
  // with 16 columns of 128 dims)
  constexpr int AHEAD = D == 128 && QT == 2 ? 1 : 2;
  const int wave = pg_uniform((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const Where w = pg_where(c, a, blockIdx.x);
  if (w.n == 0 || w.block * COLS >= w.n * a.G) return;
  const int split = blockIdx.y;
  const Keys<KT> keys(c, a, w, NW);
  if (keys.active == 0) {
    if (split == 0) pg_zero<COLS, D, 64 * NW>(a, w, threadIdx.x);
    return;
  }
  if (split >= keys.active) return;
  const int i1 = min(keys.nt, (split + 1) * keys.per);
  int i = split * keys.per + wave;

  u16x8 qop[QT][KS];
  int cp[QT];  // the columns' positions
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const Col col(a, w, w.block * COLS + 16 * t + li);
    cp[t] = col.p;
    // a column past the tile's computes with its first query and is dropped
    const uint16_t* qp = a.q + (long)(w.first + (col.live ? col.j : 0)) * a.sq_b +
                         (long)(w.kh * a.G + (col.live ? col.h : 0)) * a.sq_h;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qop[t][s] = __builtin_bit_cast(u16x8, __builtin_bit_cast(pg_u4, ld16(qp + 32 * s + 8 * lg)) ^ a.q_flip);
  }

  // The pages of the wave's next 32 steps, two 16-key groups each, in its lanes
  const int32_t* row = c.table + w.slot * c.width;
  int ids = -1, left = 0;  // steps whose pages are still ahead in `ids`
  auto fetch_ids = [&](int from) {
    const int at = from + NW * (lane >> 1);
    const int key = keys.key(at) + 16 * (lane & 1);
    ids = -1;
    if (at < i1 && key <= keys.last) ids = row[key >> c.shift];
    if ((unsigned)ids >= (unsigned)c.pages) ids = -1;
    left = 32;
  };
  const int inside = (1 << c.shift) - 1;
  const uint32_t k_at = li * (2 * D) + lg * 16, v_at = lg * (8 * D) + li * (D / 8);
  // AHEAD steps' numbers in turn: a step's keys are loaded behind the score products of the keys that they replace, its
  // values behind the output products. Loads are never conditional (one whose registers are merged behind a
  // branch is waited for there): past the wave's last step they are of no bytes.
  struct Buf {
    PgWords<4> kw[2][KS];
    PgWords<NV> vw[8];
    long off[2];   // where the two groups lie in the pools
    int bytes[2];  // what is there of them
    bool holes;    // one lies in no page
  };
  auto load_k = [&](Buf& b, int at) {
    if (left == 0) fetch_ids(at);
    const int key = at < i1 ? keys.key(at) : 0;
    b.holes = false;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int id = __builtin_amdgcn_readlane(ids, 2 * (32 - left) + g), k0 = key + 16 * g;
      b.bytes[g] = pg_uniform(id < 0 ? 0 : min(16, max(0, keys.last + 1 - k0)) * (2 * D));
      b.holes |= id < 0 && k0 <= keys.last;
      b.off[g] = pg_uniform(max(id, 0) * c.page_stride + (((long)w.kh << c.shift) + (k0 & inside)) * D);
      const auto ref = pg_ref_of(c.k + b.off[g], b.bytes[g]);
#pragma unroll
      for (int s = 0; s < KS; ++s) b.kw[g][s] = pg_load<4, NT>(ref, k_at + 64 * s);
    }
    --left;
  };
  auto load_v = [&](Buf& b) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const auto ref = pg_ref_of(c.v + b.off[g], b.bytes[g]);
#pragma unroll
      for (int e = 0; e < 4; ++e) b.vw[4 * g + e] = pg_load<NV, NT>(ref, v_at + 2 * D * e);
    }
  };

  float m[QT], l[QT];
  f32x4_t acc[QT][2 * NV];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    m[t] = -3.402823466e38f;
    l[t] = 0.f;
#pragma unroll
    for (int T = 0; T < 2 * NV; ++T) acc[t][T] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // keys up to `all` are seen by every row unless the window hides them; those up to `none` may be hidden by it
  const int all = min(w.p0, keys.last), none = a.window ? w.p0 + w.n - 1 - a.window : -1;
  auto step = [&](Buf& b, int i) {
    const int key = keys.key(i);
    const bool edge = key + KT - 1 > all || (key <= none && key + KT > a.sinks) || b.holes;
    uint32_t gone = 0;  // groups in no page
    if (b.holes) gone = (b.bytes[0] == 0 ? 1u : 0u) | (b.bytes[1] == 0 ? 2u : 0u);
    float s[QT][8];
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        f32x4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KS; ++k) x = mfma16x16x32<DT>(__builtin_bit_cast(u16x8, b.kw[g][k]), qop[t][k], x);
#pragma unroll
        for (int r = 0; r < 4; ++r) s[t][4 * g + r] = x[r];
      }
    __builtin_amdgcn_sched_barrier(0);
    const long off[2] = {b.off[0], b.off[1]};
    load_k(b, i + AHEAD * NW);
    __builtin_amdgcn_sched_barrier(0);
    if (edge) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const int p = min(cp[t], keys.last), low = pg_low(a, cp[t]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int k = key + 16 * (e >> 2) + 4 * lg + (e & 3);
          if (pg_hidden(k, p, low, a.sinks) || (gone >> (e >> 2) & 1u)) s[t][e] = -INFINITY;
        }
      }
    }
    pg_u4 pop[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float mx = s[t][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[t][e]);
      mx = fmaxf(m[t], xor32_max(xor16_max(mx)));
      if (__ballot(mx > m[t])) {
        const float f = __builtin_amdgcn_exp2f(pg_ref(m[t], a.c) - pg_ref(mx, a.c));
        l[t] *= f;
#pragma unroll
        for (int T = 0; T < 2 * NV; ++T) acc[t][T] *= f;
        m[t] = mx;
      }
      const float sub = pg_up<DT> - pg_ref(m[t], a.c);
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint32_t x = pg_pack<DT>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e], a.c, sub)),
                                       __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e + 1], a.c, sub)));
        pop[t][e / 2] = x;
        l[t] = pg_add2<DT>(x, l[t]);
      }
    }
    // 0 * V is 0 only for finite V: where some row does not see a key, infinite and NaN numbers of the step stand apart,
    // 0 in the product and added below to the columns that see them (p V of a weight p > 0 is V for these V)
    bool wild = false;
    if (edge) {
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int x = 0; x < NV; ++x) any |= pg_wild<DT>(b.vw[e].w[x]);
      wild = __ballot(any != 0) != 0;
      if (wild) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int x = 0; x < NV; ++x) b.vw[e].w[x] = pg_tame<DT>(b.vw[e].w[x]);
      }
    }
#pragma unroll
    for (int x = 0; x < NV; ++x) {
      pg_u4 lo, hi;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo[e] = __builtin_amdgcn_perm(b.vw[2 * e + 1].w[x], b.vw[2 * e].w[x], 0x05040100u);
        hi[e] = __builtin_amdgcn_perm(b.vw[2 * e + 1].w[x], b.vw[2 * e].w[x], 0x07060302u);
      }
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        acc[t][2 * x] = mfma16x16x32<DT>(__builtin_bit_cast(u16x8, lo), __builtin_bit_cast(u16x8, pop[t]), acc[t][2 * x]);
        acc[t][2 * x + 1] =
            mfma16x16x32<DT>(__builtin_bit_cast(u16x8, hi), __builtin_bit_cast(u16x8, pop[t]), acc[t][2 * x + 1]);
      }
    }
    if (wild) {
      for (int k = 0; k < KT; ++k) {
        if (key + k > keys.last || (gone >> (k >> 4) & 1u)) continue;
        const uint16_t* vp = c.v + (k < 16 ? off[0] : off[1]) + (k & 15) * D;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          uint32_t x[NV];
          if constexpr (NV == 4) *reinterpret_cast<pg_u4*>(x) = *reinterpret_cast<const pg_u4*>(vp + 2 * NV * (4 * lg + r));
          else *reinterpret_cast<pg_u2*>(x) = *reinterpret_cast<const pg_u2*>(vp + 2 * NV * (4 * lg + r));
#pragma unroll
          for (int t = 0; t < QT; ++t)
            if (!pg_hidden(key + k, min(cp[t], keys.last), pg_low(a, cp[t]), a.sinks)) {
#pragma unroll
              for (int T = 0; T < 2 * NV; ++T) acc[t][T][r] += pg_wild_number<DT>((uint16_t)(x[T / 2] >> (16 * (T & 1))));
            }
        }
      }
      __builtin_amdgcn_s_waitcnt(0x0F70);
    }
    __builtin_amdgcn_sched_barrier(0);
    load_v(b);
    __builtin_amdgcn_sched_barrier(0);
  };
  Buf b0, b1;
  load_k(b0, i);
  __builtin_amdgcn_sched_barrier(0);
  load_v(b0);
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (AHEAD == 2) {
    load_k(b1, i + NW);
    __builtin_amdgcn_sched_barrier(0);
    load_v(b1);
    __builtin_amdgcn_sched_barrier(0);
    for (; i + NW < i1; i += 2 * NW) {
      step(b0, i);
      step(b1, i + NW);
    }
    if (i < i1) step(b0, i);
  } else {
    for (; i < i1; i += NW) step(b0, i);
  }

  // merge the waves, 16 columns at a time: lane (column, lg) holds dims 2 NV (4 lg + r) + T
  __shared__ NarrowLds<D> lds;
  const long ncols = (long)gridDim.x * COLS;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    if (t) __syncthreads();
    const float sum = xor32_sum(xor16_sum(l[t]));
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int T = 0; T < 2 * NV; T += 4)
        *reinterpret_cast<f32x4_t*>(&lds.o[wave][li][2 * NV * (4 * lg + r) + T]) =
            f32x4_t{acc[t][T][r], acc[t][T + 1][r], acc[t][T + 2][r], acc[t][T + 3][r]};
    if (lg == 0) {
      lds.ref[wave][li] = pg_ref(m[t], a.c);
      lds.l[wave][li] = sum;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * (D / 4); x += 64 * NW) {
      const int col = x / (D / 4), d = x % (D / 4) * 4;
      const Col cc(a, w, w.block * COLS + 16 * t + col);
      if (!cc.live) continue;
      float M = lds.ref[0][col];
#pragma unroll
      for (int y = 1; y < NW; ++y) M = fmaxf(M, lds.ref[y][col]);
      float L = 0.f;
      f32x4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int y = 0; y < NW; ++y) {
        const float f = __builtin_amdgcn_exp2f(lds.ref[y][col] - M);
        L += lds.l[y][col] * f;
        O += *reinterpret_cast<const f32x4_t*>(&lds.o[y][col][d]) * f;
      }
      if (keys.active == 1) {
        pg_store4<DT>(a.out + (long)(w.first + cc.j) * a.so_b + (long)(w.kh * a.G + cc.h) * a.so_h + d, O, L);
      } else {
        const long at = ((long)blockIdx.x * COLS + 16 * t + col) * a.splits + split;
        *reinterpret_cast<f32x4_t*>(a.part + at * D + d) = O;
        if (d == 0) *reinterpret_cast<float2*>(a.part + ncols * a.splits * D + at * 2) = make_float2(M, L);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------
// Tiles of up to 128 columns and more: prompts. Bound by the matrix and vector units: each of the 4 waves owns 32 columns
// and passes over all keys of the split; steps of 64 keys come to LDS (two in turn) and every
// wave reads them from there, K's 16-byte chunks and V transposed by the LDS's own 16-bit transposing reads.
// Rows in LDS are permuted by 16-byte chunks so that neither read meets a bank twice.
namespace {
constexpr int WIDE_KT = 64;
// chunk x of a row lies at chunk x ^ wide_kx (wide_vx) of its row in LDS
template <int D> __device__ __forceinline__ int wide_kx(int key) { return D == 128 ? key & 15 : (key >> 1) & 7; }
template <int D> __device__ __forceinline__ int wide_vx(int key) { return D == 128 ? 2 * (key & 7) : 2 * ((key >> 1) & 3); }

typedef short pg_s4 __attribute__((ext_vector_type(4)));
}  // namespace

template <int DT, int D>
__global__ __launch_bounds__(256, 2) void paged_wide_kernel(Paged c, PagedAttn a) {
  constexpr int KT = WIDE_KT, KS = D / 32, ND = D / 16, COLS = 128, CH = D / 8, RPI = 64 / CH;  // RPI: rows a wave's load
  constexpr int RB = 2 * D, VB = KT * RB, STAGE = 2 * VB;  // bytes of a row, of a step's K, of a stage (K, then V)
  __shared__ __align__(16) uint8_t lds[2 * STAGE];
  const int wave = pg_uniform((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const Where w = pg_where(c, a, blockIdx.x);
  if (w.n == 0 || w.block * COLS >= w.n * a.G) return;
  const int split = blockIdx.y;
  const Keys<KT> keys(c, a, w, 1);
  if (keys.active == 0) {
    if (split == 0) pg_zero<COLS, D, 256>(a, w, threadIdx.x);
    return;
  }
  if (split >= keys.active) return;
  const int i0 = split * keys.per, i1 = min(keys.nt, i0 + keys.per);

  // the wave's columns
  const int c0 = w.block * COLS + 32 * wave;
  u16x8 qop[2][KS];
  int cp[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const Col col(a, w, c0 + 16 * t + li);
    cp[t] = col.p;
    const uint16_t* qp = a.q + (long)(w.first + (col.live ? col.j : 0)) * a.sq_b +
                         (long)(w.kh * a.G + (col.live ? col.h : 0)) * a.sq_h;
#pragma unroll
    for (int s = 0; s < KS; ++s)
      qop[t][s] = __builtin_bit_cast(u16x8, __builtin_bit_cast(pg_u4, ld16(qp + 32 * s + 8 * lg)) ^ a.q_flip);
  }
  // the wave's rows: the first's position (keys up to it every row sees, unless the window hides them), the last's
  const int jl = w.n - 1, ja = min((int)((uint32_t)c0 / (uint32_t)a.G), jl), jb = min((int)((uint32_t)(c0 + 31) / (uint32_t)a.G), jl);
  const bool some = c0 < w.n * a.G;
  const int pa = w.p0 + ja, pb = some ? w.p0 + jb : -1;
  const int none = a.window ? pb - a.window : -1, low = a.window ? pa - a.window : -1;

  // Lane x: the page of step base + x's group `wave` of 16 keys (-1: none), and which of its four groups lie in no page
  const int32_t* row = c.table + w.slot * c.width;
  const int inside = (1 << c.shift) - 1;
  int ids = -1, gaps = 0, base = 0;
  auto fetch_ids = [&](int from) {
    base = from;
    ids = -1;
    gaps = 0;
    const int at = from + lane;
    if (at < i1) {
      const int key = keys.key(at);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int k = key + 16 * g;
        const bool in = k <= keys.last;
        const int id = in ? row[k >> c.shift] : -1;
        if ((unsigned)id >= (unsigned)c.pages) gaps |= in ? 1 << g : 0;
        else if (g == wave) ids = id;
      }
    }
  };
  // a step's K and V: the wave brings 16 keys of each (one page), RPI a load; then to LDS. A chunk's place is its number
  // XOR a number of its row, so the places of a lane's other rows, key quarters and dims are its first place XOR constants
  // (made anew where they are used: kept, they would not fit the registers), and the other stage's XOR the stage's size.
  const int r0 = lane / CH, ch = lane % CH, rv = 4 * lg + (li >> 2);
  const uint32_t g_at = r0 * RB + ch * 16;
  uint32_t put_k = (16 * wave + r0) * RB + (ch ^ wide_kx<D>(r0)) * 16;
  uint32_t put_v = VB + (16 * wave + r0) * RB + (ch ^ wide_vx<D>(r0)) * 16;
  uint32_t get_k = li * RB + (lg ^ wide_kx<D>(li)) * 16;
  // the lane group's four keys, 16 dims: lane x brings dims 4 (x % 4) .. of key x / 4, and takes dim x of the four
  uint32_t get_v = VB + rv * RB + (((li >> 1) & 1) ^ wide_vx<D>(rv)) * 16 + (li & 1) * 8;
  PgWords<4> kb[16 / RPI], vb[16 / RPI];
  auto bring = [&](int i) {
    if (i - base == 64) fetch_ids(i);
    const int k0 = keys.key(i) + 16 * wave, x = (i - base) & 63;
    const int id = __builtin_amdgcn_readlane(ids, x);
    const uint32_t g = (uint32_t)__builtin_amdgcn_readlane(gaps, x);
    const int bytes = pg_uniform(id < 0 ? 0 : min(16, max(0, keys.last + 1 - k0)) * (2 * D));
    const long off = pg_uniform(max(id, 0) * c.page_stride + (((long)w.kh << c.shift) + (k0 & inside)) * D);
    const auto kr = pg_ref_of(c.k + off, bytes), vr = pg_ref_of(c.v + off, bytes);
#pragma unroll
    for (int x = 0; x < 16 / RPI; ++x) kb[x] = pg_load<4, false>(kr, g_at + x * RPI * RB);
#pragma unroll
    for (int x = 0; x < 16 / RPI; ++x) vb[x] = pg_load<4, false>(vr, g_at + x * RPI * RB);
    return g;
  };
  auto store = [&]() {
#pragma unroll
    for (int x = 0; x < 16 / RPI; ++x) {
      *reinterpret_cast<PgWords<4>*>(lds + (put_k ^ (64 * x)) + x * RPI * RB) = kb[x];
      *reinterpret_cast<PgWords<4>*>(lds + (put_v ^ (D == 128 ? 128 * (x & 1) : 0)) + x * RPI * RB) = vb[x];
    }
    put_k ^= STAGE;
    put_v ^= STAGE;
  };

  float m[2], l[2];
  f32x4_t acc[2][ND];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    m[t] = -3.402823466e38f;
    l[t] = 0.f;
#pragma unroll
    for (int T = 0; T < ND; ++T) acc[t][T] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  fetch_ids(i0);
  uint32_t next = bring(i0);
  store();
  __syncthreads();
  for (int i = i0; i < i1; ++i) {
    asm("" : "+v"(put_k), "+v"(put_v), "+v"(get_k), "+v"(get_v));
    const uint32_t gone = next;
    next = bring(i + 1);
    const int key = keys.key(i);
    // nothing for a wave whose rows end before the step, or from all of which the window hides it
    if (!(key > pb || (key + KT - 1 <= low && key >= a.sinks))) {
    const bool edge = key + KT - 1 > min(pa, keys.last) || (key <= none && key + KT > a.sinks) || gone;

    // operands are read a group ahead of the products that take them, held in place by the scheduling barriers
    float s[2][16];
    u16x8 kop[2][KS];
    auto read_k = [&](int g) {
#pragma unroll
      for (int k = 0; k < KS; ++k)
        kop[g & 1][k] = ld16(reinterpret_cast<const uint16_t*>(lds + (get_k ^ (64 * k)) + 16 * g * RB));
    };
    read_k(0);
#pragma unroll
    for (int g = 0; g < KT / 16; ++g) {
      if (g + 1 < KT / 16) read_k(g + 1);
      __builtin_amdgcn_sched_barrier(0);
      f32x4_t x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int t = 0; t < 2; ++t) x[t] = mfma16x16x32<DT>(kop[g & 1][k], qop[t][k], x[t]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[t][4 * g + r] = x[t][r];
    }
    // V's operands, 64 keys of 16 dims
    pg_u2 vop[2][4];
    auto read_v = [&](int T) {
#pragma unroll
      for (int h = 0; h < 4; ++h)
        vop[T & 1][h] = __builtin_bit_cast(
            pg_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                       (__attribute__((address_space(3))) pg_s4*)(lds + (get_v ^ (32 * T)) + 16 * h * RB)));
    };
    read_v(0);
    __builtin_amdgcn_sched_barrier(0);
    if (edge) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int p = min(cp[t], keys.last), lw = pg_low(a, cp[t]);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int k = key + 16 * (e >> 2) + 4 * lg + (e & 3);
          if (pg_hidden(k, p, lw, a.sinks) || (gone >> (e >> 2) & 1u)) s[t][e] = -INFINITY;
        }
      }
    }
    pg_u4 pop[2][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      float mx = s[t][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[t][e]);
      mx = fmaxf(m[t], xor32_max(xor16_max(mx)));
      if (__ballot(mx > m[t])) {
        const float f = __builtin_amdgcn_exp2f(pg_ref(m[t], a.c) - pg_ref(mx, a.c));
        l[t] *= f;
#pragma unroll
        for (int T = 0; T < ND; ++T) acc[t][T] *= f;
        m[t] = mx;
      }
      const float sub = pg_up<DT> - pg_ref(m[t], a.c);
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        const uint32_t x = pg_pack<DT>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e], a.c, sub)),
                                       __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e + 1], a.c, sub)));
        pop[t][e / 8][e % 8 / 2] = x;
        l[t] = pg_add2<DT>(x, l[t]);
      }
    }
    // as in the narrow kernel: infinite and NaN values stand apart where some row does not see their key
    bool wild = false;
    if (edge) {
      uint32_t any = 0;
#pragma unroll
      for (int x = 0; x < KT * D / 512; ++x) {
        const pg_u4 v = *reinterpret_cast<const pg_u4*>(lds + (get_v & STAGE) + VB + (x * 64 + lane) * 16);
        any |= pg_wild<DT>(v[0]) | pg_wild<DT>(v[1]) | pg_wild<DT>(v[2]) | pg_wild<DT>(v[3]);
      }
      wild = __ballot(any != 0) != 0;
    }
    auto products = [&](auto tame) {
#pragma unroll
      for (int T = 0; T < ND; ++T) {
        if (T + 1 < ND) read_v(T + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) {
          const pg_u2 x = vop[T & 1][2 * u], y = vop[T & 1][2 * u + 1];
          const pg_u4 v = tame ? pg_u4{pg_tame<DT>(x[0]), pg_tame<DT>(x[1]), pg_tame<DT>(y[0]), pg_tame<DT>(y[1])}
                               : pg_u4{x[0], x[1], y[0], y[1]};
#pragma unroll
          for (int t = 0; t < 2; ++t)
            acc[t][T] = mfma16x16x32<DT>(__builtin_bit_cast(u16x8, v), __builtin_bit_cast(u16x8, pop[t][u]), acc[t][T]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (!wild) {
      products(std::false_type{});
    } else {
      products(std::true_type{});
      for (int k = 0; k < KT; ++k) {
        if (key + k > keys.last || (gone >> (k >> 4) & 1u)) continue;
#pragma unroll
        for (int T = 0; T < ND; ++T) {
          const uint16_t* vp = reinterpret_cast<const uint16_t*>(
              lds + (get_v & STAGE) + VB + k * RB + ((2 * T + (lg >> 1)) ^ wide_vx<D>(k & 15)) * 16 + (lg & 1) * 8);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float x = pg_wild_number<DT>(vp[r]);
#pragma unroll
            for (int t = 0; t < 2; ++t)
              if (!pg_hidden(key + k, min(cp[t], keys.last), pg_low(a, cp[t]), a.sinks)) acc[t][T][r] += x;
          }
        }
      }
    }
    }
    store();
    get_k ^= STAGE;
    get_v ^= STAGE;
    __syncthreads();
  }

  // lane (column, lg) holds dims 16 T + 4 lg + r
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const float L = xor32_sum(xor16_sum(l[t]));
    const int col = c0 + 16 * t + li;
    const Col cc(a, w, col);
    if (!cc.live) continue;
    if (keys.active == 1) {
      uint16_t* op = a.out + (long)(w.first + cc.j) * a.so_b + (long)(w.kh * a.G + cc.h) * a.so_h + 4 * lg;
#pragma unroll
      for (int T = 0; T < ND; ++T) pg_store4<DT>(op + 16 * T, acc[t][T], L);
    } else {
      const long ncols = (long)gridDim.x * COLS, at = ((long)blockIdx.x * COLS + 32 * wave + 16 * t + li) * a.splits + split;
#pragma unroll
      for (int T = 0; T < ND; ++T) *reinterpret_cast<f32x4_t*>(a.part + at * D + 16 * T + 4 * lg) = acc[t][T];
      if (lg == 0) *reinterpret_cast<float2*>(a.part + ncols * a.splits * D + at * 2) = make_float2(pg_ref(m[t], a.c), L);
    }
  }
}

// Joins the splits: D / 4 threads a column, in the splits' order
template <int DT, int D, int KT, int LEAST>
__global__ __launch_bounds__(256) void paged_join_kernel(Paged c, PagedAttn a, int cols) {
  constexpr int TD = D / 4, CB = 256 / TD;
  const uint32_t per = cols / CB, item = blockIdx.x / per;
  const Where w = pg_where(c, a, item);
  if (w.n == 0) return;
  const Keys<KT> keys(c, a, w, LEAST);
  if (keys.active <= 1) return;  // written by the attention itself
  const int col = (blockIdx.x - item * per) * CB + threadIdx.x / TD, d = threadIdx.x % TD * 4;
  const Col cc(a, w, w.block * cols + col);
  if (!cc.live) return;
  const long ncols = (long)(gridDim.x / per) * cols, at = ((long)item * cols + col) * a.splits;
  const float* po = a.part + at * D + d;
  const float* ml = a.part + ncols * a.splits * D + at * 2;
  float M = -INFINITY, L = 0.f;
  f32x4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < keys.active; ++s) {
    const float2 x = *reinterpret_cast<const float2*>(ml + 2 * s);
    const f32x4_t o = *reinterpret_cast<const f32x4_t*>(po + (long)s * D);
    const float mx = fmaxf(M, x.x), f0 = __builtin_amdgcn_exp2f(M - mx), f1 = __builtin_amdgcn_exp2f(x.x - mx);
    L = L * f0 + x.y * f1;
    O = O * f0 + o * f1;
    M = mx;
  }
  pg_store4<DT>(a.out + (long)(w.first + cc.j) * a.so_b + (long)(w.kh * a.G + cc.h) * a.so_h + d, O, L);
}

// ---------------------------------------------------------------------------------------------------------
namespace {
template <int DT, int D> void paged_launch(const Paged& c, const PagedAttn& a, int items, int cols, bool single, hipStream_t st) {
  const dim3 grid(items, a.splits);
  if (cols == 128) hipLaunchKernelGGL((paged_wide_kernel<DT, D>), grid, dim3(256), 0, st, c, a);
  else if (cols == 32) hipLaunchKernelGGL((paged_narrow_kernel<DT, D, 2, false>), grid, dim3(256), 0, st, c, a);
  else if (single) hipLaunchKernelGGL((paged_narrow_kernel<DT, D, 1, true>), grid, dim3(256), 0, st, c, a);
  else hipLaunchKernelGGL((paged_narrow_kernel<DT, D, 1, false>), grid, dim3(256), 0, st, c, a);
  if (a.splits == 1) return;
  const dim3 jg(items * (cols / (1024 / D)));
  if (cols == 128) hipLaunchKernelGGL((paged_join_kernel<DT, D, WIDE_KT, 1>), jg, dim3(256), 0, st, c, a, cols);
  else hipLaunchKernelGGL((paged_join_kernel<DT, D, 32, NARROW_NW>), jg, dim3(256), 0, st, c, a, cols);
}
// workgroups a split: tiles x kv heads x blocks of the columns; 0: out of range
long paged_items(long tiles, int kv_heads, int heads, int tile_rows, int cols) {
  if (tiles < 0 || kv_heads <= 0 || heads <= 0 || tile_rows <= 0 || heads % kv_heads) return 0;
  if (cols != 16 && cols != 32 && cols != 128) return 0;
  const long per_tile = kv_heads * (((long)tile_rows * (heads / kv_heads) + cols - 1) / cols);
  return tiles * per_tile < 1L << 24 ? tiles * per_tile : 0;
}
}  // namespace

M3X_API size_t m3x_paged_attn_workspace(int tiles, int kv_heads, int heads, int tile_rows, int cols, int head_dim, int splits) {
  if (splits <= 1 || head_dim <= 0) return 0;
  return (size_t)paged_items(tiles, kv_heads, heads, tile_rows, cols) * cols * splits * (head_dim + 2) * sizeof(float);
}

M3X_API int m3x_paged_attn(const M3xPagedKv* cache, const void* q, long sq_b, long sq_h, void* out, long so_b, long so_h,
                           const int64_t* slots, const int32_t* pos, const int32_t* tiles, int ntiles, int tile_rows,
                           int cols, float scale, int rows, int heads, int window, int sinks, int splits, void* workspace,
                           size_t ws_bytes, void* stream) {
  Paged c;
  if (const int st = paged_take(cache, c)) return st;
  if (rows < 0 || ntiles < 0 || heads <= 0 || window < 0 || sinks < 0 || heads > 65535) return M3X_EINVAL;
  if (heads % c.kv_heads) return M3X_EUNSUPPORTED;
  if (!(fabsf(scale) <= 0x1p126f)) return M3X_EINVAL;  // its factor would not be finite; NaN
  if (splits < 1 || splits > 256) return M3X_EINVAL;
  if (rows == 0 || ntiles == 0) return M3X_OK;
  if (!q || !out || !slots || !pos) return M3X_ENULL;
  if (((sq_b | sq_h | so_b | so_h) & 7) || !m3x_aligned16(q) || !m3x_aligned16(out) || ((uintptr_t)tiles & 3u)) return M3X_EINVAL;
  if (!tiles && (ntiles > rows || tile_rows != 1)) return M3X_EINVAL;
  const long items = paged_items(ntiles, c.kv_heads, heads, tile_rows, cols);
  if (items == 0) return M3X_EINVAL;
  if (splits > 1) {
    if (!workspace) return M3X_ENULL;
    if (ws_bytes < m3x_paged_attn_workspace(ntiles, c.kv_heads, heads, tile_rows, cols, cache->head_dim, splits))
      return M3X_EWORKSPACE;
    if (!m3x_aligned16(workspace)) return M3X_EINVAL;
  }
  // The factor of the scores' exponents, never 0 (0 * -inf of a hidden key). fp32's smallest normal number stands for all
  // below it: scores up to 2^100 weigh alike under either.
  const float factor = std::max(fabsf(scale) * 1.44269504088896341f, 0x1p-126f);
  const int G = heads / c.kv_heads;
  const PagedAttn a = {(const uint16_t*)q, sq_b, sq_h, (uint16_t*)out, so_b, so_h, slots, pos, tiles, factor,
                       scale < 0.f ? 0x80008000u : 0u, rows, heads, G, tile_rows, (tile_rows * G + cols - 1) / cols,
                       std::min(window, 1 << 30), std::min(sinks, 1 << 30), splits, (float*)workspace};
  hipStream_t st = (hipStream_t)stream;
  const bool single = tile_rows == 1;
  const int D = cache->head_dim;
  if (cache->dtype == M3X_BF16 && D == 128) paged_launch<M3X_BF16, 128>(c, a, (int)items, cols, single, st);
  else if (cache->dtype == M3X_BF16) paged_launch<M3X_BF16, 64>(c, a, (int)items, cols, single, st);
  else if (D == 128) paged_launch<M3X_F16, 128>(c, a, (int)items, cols, single, st);
  else paged_launch<M3X_F16, 64>(c, a, (int)items, cols, single, st);
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}
