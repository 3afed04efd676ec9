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
// and divided evenly among the splits. The splits' partial results are joined in the splits' order: few columns' by the
// split that is done last, prompts' by a second launch.
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
  uint32_t over_G;  // ceil(2^32 / G): x / G = x * over_G >> 32 for x, G < 2^16 (0 for G = 1)
  float* part;   // [columns][splits][D], then [columns][splits][2]: (maximum, sum)
  int* arrived;  // narrow: a counter for each (tile, kv head, block), 0 between calls
};

// a workgroup's place: a tile, a kv head, a block of the tile's columns; all uniform
struct Where {
  int tile, kh, block, first, n, p0;  // rows first .. first + n - 1 at positions p0 ..; n == 0: nothing to do
  int splits;  // that may share the tile's keys
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
// x: kv head + kv_heads * block, y: tile (z: split)
__device__ __forceinline__ Where pg_where(const Paged& c, const PagedAttn& a, int x, int tile) {
  Where w;
  w.tile = tile;
  w.block = 0;
  w.kh = x;
  if (a.blocks > 1) {
    w.block = pg_uniform(x / c.kv_heads);
    w.kh = x - w.block * c.kv_heads;
  }
  w.first = tile;
  w.n = 1;
  w.splits = a.splits;
  if (a.tiles) {
    w.first = pg_uniform(a.tiles[2 * tile]);
    const int rows = pg_uniform(a.tiles[2 * tile + 1]);
    w.n = rows < 0 ? 0 : rows & 0xFFFF;
    if (rows >> 16) w.splits = min(w.splits, rows >> 16);
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
__device__ __forceinline__ int pg_row(const PagedAttn& a, int col) {
  return a.over_G ? (int)__umulhi((uint32_t)col, a.over_G) : col;
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
    per = nt;
    active = nt > 0;
    if (a.splits > 1) {
      per = pg_uniform(max(least, (nt + w.splits - 1) / w.splits));
      active = pg_uniform((nt + per - 1) / per);
    }
  }
  __device__ __forceinline__ int key(int i) const { return (i + (i < sink ? 0 : skip)) * KT; }
};

// a column's row and head, and the keys it sees
struct Col {
  int j, h, p;  // row of the tile, head of the kv head's G, position
  bool live;
  __device__ __forceinline__ Col(const PagedAttn& a, const Where& w, int col) {
    j = pg_row(a, col);
    h = col - j * a.G;
    live = j < w.n;
    p = live ? w.p0 + j : -1;
  }
};
// whether a row at p does not see a key; low: pg_low
__device__ __forceinline__ bool pg_hidden(int key, int p, int low, int sinks) { return key > p || (key <= low && key >= sinks); }
// the largest position that the window hides from a row at p (-1: none)
__device__ __forceinline__ int pg_low(const PagedAttn& a, int p) { return a.window ? p - a.window : -1; }

// Scores s[e] of the keys from + 8 (e / 4) * STEP / 8 + e % 4 that a row at p does not see become -inf: later ones, and where
// the window cuts (uniform) those up to `low` behind the sinks. holes: bits of 16-key groups in no page.
template <int N, int STEP, typename T>
__device__ __forceinline__ void pg_mask(T& s, int from, int p, int low, int sinks, bool cuts, uint32_t holes) {
  const int late = p - from;
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (STEP * (e >> 2) + (e & 3) > late) s[e] = -INFINITY;
  if (cuts) {
    const int early = low - from, kept = sinks - from;
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (STEP * (e >> 2) + (e & 3) <= early && STEP * (e >> 2) + (e & 3) >= kept) s[e] = -INFINITY;
  }
  if (holes) {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (holes >> (STEP * (e >> 2) >> 4) & 1u) s[e] = -INFINITY;
  }
}

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
// acc, or NaN where one of the two numbers of w is infinite or NaN (0 times it)
template <int DT> __device__ __forceinline__ float pg_probe(uint32_t w, float acc) {
  if constexpr (DT == M3X_F16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(pg_h2, w), __builtin_bit_cast(pg_h2, 0u), acc, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pg_bf2, w), __builtin_bit_cast(pg_bf2, 0u), acc, false);
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

// A weight's exponent is (s - m) c + up, m the column's running maximum: the difference of the raw scores, exact near the
// maximum, is taken first, so that the largest weight is 2^up whatever the scores' size (s c - m c, each rounded, would be
// off by half a unit of m c, which from 2^24 on is more than the weights' whole range). Waves, key groups and splits hand
// their raw maximum on with their sums, which are then joined by the same differences. A column that has seen nothing
// stands at PG_LEAST, below every score.
constexpr float PG_LEAST = -3.402823466e38f;

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

// Device-scope accesses (SC1), coherent across the XCDs' L2s: partial results that another workgroup of the launch joins.
// A store has arrived where every such load finds it once the storing wave's vmcnt is 0.
constexpr int PG_SC1 = 16;
constexpr int PG_SPAN = 0x7f000000;  // bytes that a place's partial results stay below
__device__ __forceinline__ __amdgpu_buffer_rsrc_t pg_span(float* p) {
  return __builtin_amdgcn_make_buffer_rsrc(p, 0, PG_SPAN, 0x00020000);
}

// dims d .. d + 3 of a column's output from its splits' partial results, in their order; AUX: how they are read. The
// addresses are a place's (uniform, 64-bit) and a column's within it (below PG_SPAN bytes: 128 columns of 256 splits).
template <int DT, int D, int AUX>
__device__ __forceinline__ void pg_join(const PagedAttn& a, const Where& w, const Col& cc, long place, int cols, int col,
                                        long ncols, int active, int d) {
  const auto po = pg_span(a.part + place * cols * a.splits * D);
  const auto ml = pg_span(a.part + ncols * a.splits * D + place * cols * a.splits * 2);
  float M = -INFINITY, L = 0.f;
  f32x4_t O = {0.f, 0.f, 0.f, 0.f};
  // eight splits' loads at a time, of no bytes behind the last
  for (int s0 = 0; s0 < active; s0 += 8) {
    float2 x[8];
    f32x4_t o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = col * a.splits + s0 + e;
      const bool in = s0 + e < active;
      x[e] = __builtin_bit_cast(float2, (pg_u2)__builtin_amdgcn_raw_buffer_load_b64(ml, in ? at * 8 : PG_SPAN, 0, AUX));
      o[e] = __builtin_bit_cast(
          f32x4_t, (pg_u4)__builtin_amdgcn_raw_buffer_load_b128(po, in ? (at * D + d) * 4 : PG_SPAN, 0, AUX));
    }
    float mx = M;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (s0 + e >= active) x[e].x = -INFINITY;
      mx = fmaxf(mx, x[e].x);
    }
    const float f0 = __builtin_amdgcn_exp2f((M - mx) * a.c);
    L *= f0;
    O *= f0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = __builtin_amdgcn_exp2f((x[e].x - mx) * a.c);
      L += x[e].y * f;
      O += o[e] * f;
    }
    M = mx;
  }
  pg_store4<DT>(a.out + (long)(w.first + cc.j) * a.so_b + (long)(w.kh * a.G + cc.h) * a.so_h + d, O, L);
}

constexpr int NARROW_NW = 4;
constexpr int WIDE_LEAST = 2;  // steps a split at least
template <int D, int COLS> struct NarrowLds {
  int order;
  __align__(16) float o[NARROW_NW][COLS][D + 4];
  float m[NARROW_NW][COLS], l[NARROW_NW][COLS];
};
}  // namespace

// Tiles of up to 16 QT columns: single tokens, the few rows of drafted ones, and short prompts cut into such tiles. Bound by
// the keys' bytes. Each of the 4 waves takes every fourth step of 32 keys, straight from memory to registers: K as the score
// product's operand, V as rows whose numbers byte permutes pair over keys. The waves' results are merged through LDS.
// Measured on MI355X (bf16, 16/8 heads of 128, page_size 64, graph-timed): 224 rows of 2048 keys 275 us, 1.87 GB at 6.8
// TB/s; 48 rows of a 1024-key window 37 us, 5.4 TB/s; one row of 2048 keys in 8 splits 7.9 us: launch 2, loads of what the
// next load needs (tile, slot, page, keys) 3, two steps and the merge 1, join 2.
// NT: the keys' loads carry the non-temporal hint, for single rows, whose keys one workgroup reads once (224 rows 276 us
// against 312; 48 rows, whose keys stay in the memory-side cache from call to call, 37 against 35).
template <int DT, int D, int QT, bool NT>
__global__ __launch_bounds__(256, QT > 1 ? 2 : D == 64 ? 4 : 3) void paged_narrow_kernel(Paged c, PagedAttn a) {
  constexpr int KT = 32, NW = NARROW_NW, KS = D / 32, NV = D / 32, COLS = 16 * QT;
  // NV: words of V a lane holds of a key (2 NV dims)
  const int wave = pg_uniform((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const Where w = pg_where(c, a, blockIdx.x, blockIdx.y);
  if (w.n == 0 || w.block * COLS >= w.n * a.G) return;
  const int split = blockIdx.z;
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
  // A step's keys are loaded behind the score products of the keys that they replace, its values behind the output
  // products. Loads are never conditional (one whose registers are merged behind a branch is waited for there): past the
  // wave's last step they are of no bytes. Two steps ahead, in two sets of registers, were no faster over long contexts (224
  // rows of 2048 keys 275 us either way) and slower over short ones, by their fewer waves and longer code: one row 8.6 us
  // against 8.0, 224 rows of 300 keys 47 against 43.6.
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
    m[t] = PG_LEAST;
    l[t] = 0.f;
#pragma unroll
    for (int T = 0; T < 2 * NV; ++T) acc[t][T] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // keys up to `all` are seen by every row unless the window hides them; those up to `none` may be hidden by it
  const int all = min(w.p0, keys.last), none = a.window ? w.p0 + w.n - 1 - a.window : -1;
  auto step = [&](Buf& b, int i) {
    const int key = keys.key(i);
    const bool cuts = key <= none && key + KT > a.sinks;
    const bool edge = key + KT - 1 > all || cuts || b.holes;
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
    load_k(b, i + NW);
    __builtin_amdgcn_sched_barrier(0);
    if (edge) {
#pragma unroll
      for (int t = 0; t < QT; ++t)
        pg_mask<8, 16>(s[t], key + 4 * lg, min(cp[t], keys.last), pg_low(a, cp[t]), a.sinks, cuts, gone);
    }
    pg_u4 pop[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      float mx = s[t][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[t][e]);
      mx = fmaxf(m[t], xor32_max(xor16_max(mx)));
      if (__ballot(mx > m[t])) {
        const float f = __builtin_amdgcn_exp2f((m[t] - mx) * a.c);
        l[t] *= f;
#pragma unroll
        for (int T = 0; T < 2 * NV; ++T) acc[t][T] *= f;
        m[t] = mx;
      }
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint32_t x = pg_pack<DT>(__builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e] - m[t], a.c, pg_up<DT>)),
                                       __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][e + 1] - m[t], a.c, pg_up<DT>)));
        pop[t][e / 2] = x;
        l[t] = pg_add2<DT>(x, l[t]);
      }
    }
    // 0 * V is 0 only for finite V: where some row does not see a key, infinite and NaN numbers of the step stand apart,
    // 0 in the product and added below to the columns that see them (p V of a weight p > 0 is V for these V)
    bool wild = false;
    if (edge) {
      float any = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int x = 0; x < NV; ++x) any = pg_probe<DT>(b.vw[e].w[x], any);
      wild = __ballot(any != any) != 0;
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
  Buf b;
  load_k(b, i);
  __builtin_amdgcn_sched_barrier(0);
  load_v(b);
  __builtin_amdgcn_sched_barrier(0);
  for (; i < i1; i += NW) step(b, i);

  // merge the waves: lane (column, lg) holds dims 2 NV (4 lg + r) + T
  __shared__ NarrowLds<D, COLS> lds;
  const long place = (long)blockIdx.y * gridDim.x + blockIdx.x, ncols = (long)gridDim.y * gridDim.x * COLS;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const float sum = xor32_sum(xor16_sum(l[t]));
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int T = 0; T < 2 * NV; T += 4)
        *reinterpret_cast<f32x4_t*>(&lds.o[wave][16 * t + li][2 * NV * (4 * lg + r) + T]) =
            f32x4_t{acc[t][T][r], acc[t][T + 1][r], acc[t][T + 2][r], acc[t][T + 3][r]};
    if (lg == 0) {
      lds.m[wave][16 * t + li] = m[t];
      lds.l[wave][16 * t + li] = sum;
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int x = threadIdx.x; x < COLS * (D / 4); x += 64 * NW) {
    const int col = x / (D / 4), d = x % (D / 4) * 4;
    const Col cc(a, w, w.block * COLS + col);
    if (!cc.live) continue;
    float M = lds.m[0][col];
#pragma unroll
    for (int y = 1; y < NW; ++y) M = fmaxf(M, lds.m[y][col]);
    float L = 0.f;
    f32x4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int y = 0; y < NW; ++y) {
      const float f = __builtin_amdgcn_exp2f((lds.m[y][col] - M) * a.c);
      L += lds.l[y][col] * f;
      O += *reinterpret_cast<const f32x4_t*>(&lds.o[y][col][d]) * f;
    }
    if (keys.active == 1) {
      pg_store4<DT>(a.out + (long)(w.first + cc.j) * a.so_b + (long)(w.kh * a.G + cc.h) * a.so_h + d, O, L);
    } else {
      const int at = col * a.splits + split;
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(pg_u4, O), pg_span(a.part + place * COLS * a.splits * D),
                                             (at * D + d) * 4, 0, PG_SC1);
      if (d == 0)
        __builtin_amdgcn_raw_buffer_store_b64(
            __builtin_bit_cast(pg_u2, make_float2(M, L)),
            pg_span(a.part + ncols * a.splits * D + place * COLS * a.splits * 2), at * 8, 0, PG_SC1);
    }
  }
  // The split that is done last joins them, in their order whichever it is. Its place's counter is 0 again afterwards.
  if (keys.active == 1) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) lds.order = __hip_atomic_fetch_add(a.arrived + place, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (lds.order != keys.active - 1) return;
  if (threadIdx.x == 0) __hip_atomic_store(a.arrived + place, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (int x = threadIdx.x; x < COLS * (D / 4); x += 64 * NW) {
    const Col cc(a, w, w.block * COLS + x / (D / 4));
    if (cc.live) pg_join<DT, D, PG_SC1>(a, w, cc, place, COLS, x / (D / 4), ncols, keys.active, x % (D / 4) * 4);
  }
}

// ---------------------------------------------------------------------------------------------------------
// Tiles of up to 128 columns and more: prompts. Bound by the matrix and vector units: each of 4 waves owns 32 columns and
// passes over the keys of the split (of its half: where the call has few workgroups, KG = 2 groups of 4 waves share the
// keys) in steps of 32, which come to LDS by loads that need no registers, two steps
// ahead; every wave reads K there in 16-byte chunks and V transposed by the LDS's own 16-bit transposing reads. A row's
// chunks lie in LDS at their number XOR a number of the row, so that neither read meets a bank twice.
// Measured on MI355X (bf16, page_size 64 or 128, graph-timed): 4096 rows onto 12288 keys, 32/8 heads of 128, 895 us, 1075
// TFLOP/s, where an 8192^3 product of the library reaches 1290; the matrix units are busy half of the time, the vector units
// about as long, and the clock is down to 1.9 GHz. 8 x 200 rows onto 300 to 500 keys, 16/8 heads, 21 us: launch 2, tile, slot
// and page numbers 2.5, the first keys and queries 0.6, the first turn 2 to 3 with its code's way into the instruction
// cache, seven more of both key groups 1.3 each, the groups' sums 2.
namespace {
constexpr int WIDE_KT = 32;
// A weight's exponent is counted from a reference m (a raw score) that the scores of a column pass by less than WIDE_SLACK:
// renewing it whenever a maximum grows would mean scaling the outputs in most turns of a wave's 32 columns. Weights stand at
// 2^wide_up of their size, as in the narrow kernel. While m c is up to WIDE_NEAR, exponents are s c + add, one multiply-add,
// add = wide_up - m c rounded to 2^-7 at worst: all of the column's weights are in the same proportion as with m c itself,
// and what it is off by is made good where sums are handed on. A wave that meets a larger score takes the differences
// (s - m) c from then on, in every turn.
constexpr float WIDE_SLACK = 8.f, WIDE_NEAR = 65536.f;
template <int DT> constexpr float wide_up = pg_up<DT> - WIDE_SLACK;

// chunk x of a row lies at chunk x ^ wide_kx (wide_vx) of its row in LDS
template <int D> __device__ __forceinline__ int wide_kx(int key) { return D == 128 ? key & 15 : (key >> 1) & 7; }
template <int D> __device__ __forceinline__ int wide_vx(int key) { return D == 128 ? 4 * (key & 3) : 4 * ((key >> 1) & 1); }

typedef short pg_s4 __attribute__((ext_vector_type(4)));
typedef float pg_f16 __attribute__((ext_vector_type(16)));

// v_mfma_f32_32x32x16: A is 32 x 16, B 16 x 32; lane l holds A[l % 32][8 (l / 32) + e] and B[8 (l / 32) + e][l % 32], e = 0 ..
// 7, and D[8 (r / 4) + 4 (l / 32) + r % 4][l % 32], r = 0 .. 15. It takes the matrix unit 32 clocks and leaves the vector
// unit 24 of them, where two 16 x 16 x 32 leave 16.
template <int DT> __device__ __forceinline__ pg_f16 mfma32x32x16(const u16x8& a, const u16x8& b, pg_f16 c) {
  if constexpr (DT == M3X_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// Lane x's 16 bytes at `off` of a tile of `bytes` bytes at `base` to LDS, `by` + x * 16 bytes behind `to` (all uniform but
// off). The compiler knows neither the load nor what it writes: the caller waits (pg_landed) and then meets the other waves
// before anyone reads. PAUSE: idle slots between what writes the scalar registers and the load that takes them, 4 where a
// vector instruction may have written the tile's, 0 where they stand since the load before (m0 needs one). m0 is free:
// nothing else in the kernels here uses it, and the compiler gives it to no variable.
template <int PAUSE> __device__ __forceinline__ void pg_to_lds(uint64_t base, uint32_t bytes, uint32_t off, uint32_t to, int by) {
  const pg_u4 ref = {(uint32_t)base, (uint32_t)(base >> 32) & 0xFFFFu, bytes, 0x00020000u};
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop %4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(to), "v"(off), "s"(ref),
               "i"(by), "n"(PAUSE)
               : "memory", "scc");
}
// waits until all but the wave's last N loads have arrived
template <int N> __device__ __forceinline__ void pg_landed() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
}  // namespace

template <int DT, int D, int KG>
__global__ __launch_bounds__(256 * KG, 2) void paged_wide_kernel(Paged c, PagedAttn a) {
  constexpr int KT = WIDE_KT, KS = D / 16, ND = D / 32, COLS = 128, CH = D / 8, RPI = 64 / CH;  // RPI: rows a wave's load
  constexpr int RB = 2 * D, SB = KT * RB, LI = 8 / RPI;  // bytes of a row and of a step's K; a wave's loads of them
  // rings of stages, a step's at its number % 4: in turn j K of steps j + 1 .. j + 3 and V of j - 1 .. j + 2 are there or come
  constexpr int NK = 4, NV = 4, RING = 4 * SB;
  constexpr int LDS = (NK + NV + 1) * SB;  // a key group's; the last stage: values without infinite and NaN ones, see below
  __shared__ __align__(16) uint8_t lds[KG * LDS];
  const int group = KG == 1 ? 0 : pg_uniform((int)(threadIdx.x >> 8)), wave = pg_uniform((int)(threadIdx.x >> 6 & 3));
  uint8_t* const lk = lds + group * LDS;
  uint8_t* const lv = lk + NK * SB;
  const int lane = threadIdx.x & 63, li = lane & 31, lh = lane >> 5;
  const Where w = pg_where(c, a, blockIdx.x, blockIdx.y);
  if (w.n == 0 || w.block * COLS >= w.n * a.G) return;
  const int split = blockIdx.z;
  const Keys<KT> keys(c, a, w, WIDE_LEAST);
  if (keys.active == 0) {
    if (split == 0) pg_zero<COLS, D, 256 * KG>(a, w, threadIdx.x);
    return;
  }
  if (split >= keys.active) return;
  // the split's steps, divided among the key groups; n: the most that one has
  const int from = split * keys.per, till = min(keys.nt, from + keys.per);
  const int n = (till - from + KG - 1) / KG, i0 = min(till, from + group * n), i1 = min(till, i0 + n);

  // Lane x, for step base + x's group wave / 2 of 16 keys: where it lies in the pools, the bytes that are there
  const int32_t* row = c.table + w.slot * c.width;
  int off_lo = 0, off_hi = 0, info = 0, base = 0;
  bool holes = false;  // some group lies in no page
  auto fetch = [&](int from) {
    base = from;
    info = 0;
    bool hole = false;
    const int at = from + lane;
    if (at < i1) {
      const int key = keys.key(at);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int k = key + 16 * g;
        if (k > keys.last) continue;
        const int id = row[k >> c.shift];
        if ((unsigned)id >= (unsigned)c.pages) {
          hole = true;
        } else if (g == wave >> 1) {
          const long off = 2 * (id * c.page_stride + (((long)w.kh << c.shift) + (k & ((1 << c.shift) - 1))) * D);
          off_lo = (int)off;
          off_hi = (int)(off >> 32);
          info = min(16, keys.last + 1 - k) * RB;
        }
      }
    }
    holes |= __ballot(hole) != 0;
  };
  // The wave brings 8 rows of a step's K and V. A load writes LDS in the lanes' order: the lanes' addresses do the XOR.
  uint32_t from_k[LI], from_v[LI];
#pragma unroll
  for (int x = 0; x < LI; ++x) {
    const int r = 8 * (wave & 1) + x * RPI + lane / CH;  // of the 16-key group
    from_k[x] = r * RB + ((lane % CH) ^ wide_kx<D>(r)) * 16;
    from_v[x] = r * RB + ((lane % CH) ^ wide_vx<D>(r)) * 16;
  }
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  const uint32_t to = pg_uniform((int)(lds_at + group * LDS + 8 * wave * RB));
  uint64_t v_from = 0;  // V of the step whose K came last
  uint32_t v_bytes = 0;
  auto bring_v = [&](uint32_t stage) __attribute__((always_inline)) {
    pg_to_lds<4>(v_from, v_bytes, from_v[0], to + stage, RING);
    if constexpr (LI == 2) pg_to_lds<0>(v_from, v_bytes, from_v[1], to + stage, RING + RPI * RB);
  };
  auto bring_k = [&](int i, uint32_t stage) __attribute__((always_inline)) {
    const int x = i - base;
    const uint64_t off = (uint32_t)__builtin_amdgcn_readlane(off_lo, x) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane(off_hi, x) << 32;
    v_bytes = (uint32_t)__builtin_amdgcn_readlane(info, x);
    v_from = (uint64_t)c.v + off;
    pg_to_lds<4>((uint64_t)c.k + off, v_bytes, from_k[0], to + stage, 0);
    if constexpr (LI == 2) pg_to_lds<0>((uint64_t)c.k + off, v_bytes, from_k[1], to + stage, RPI * RB);
  };

  // the wave's columns
  const int c0 = w.block * COLS + 32 * wave;
  const Col col(a, w, c0 + li);
  const int cp = col.p;
  const uint16_t* qp = a.q + (long)(w.first + (col.live ? col.j : 0)) * a.sq_b + (long)(w.kh * a.G + (col.live ? col.h : 0)) * a.sq_h;
  u16x8 qop[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s)
    qop[s] = __builtin_bit_cast(u16x8, __builtin_bit_cast(pg_u4, ld16(qp + 16 * s + 8 * lh)) ^ a.q_flip);
  // the wave's rows: the first's position (keys up to it every row sees, unless the window hides them), the last's
  const int jl = w.n - 1, ja = min(pg_row(a, c0), jl), jb = min(pg_row(a, c0 + 31), jl);
  const int pa = min(pg_uniform(w.p0 + ja), keys.last), pb = min(pg_uniform(c0 < w.n * a.G ? w.p0 + jb : -1), keys.last);
  const int none = a.window ? pg_uniform(w.p0 + jb) - a.window : -1;
  // the wave's steps: those up to its last row's key, the sinks' in any case: a window that begins past the table's end lies
  // behind pb, and leaves them alone
  const int steps = pb < 0 ? 0 : max(0, min(i1 - i0, max(pb / KT - keys.skip, keys.sink - 1) - i0 + 1));
  // The turns whose step every row sees whole: from plain on up to edge. Before them the window hides something (or
  // nothing: steps of the sinks).
  const int edge = min(steps, max(0, (pa + 1) / KT - keys.skip - i0));
  int plain = none < 0 ? 0 : none / KT + 1 - keys.skip - i0;

  const uint32_t get_k = li * RB + (lh ^ wide_kx<D>(li)) * 16;
  // Sixteen lanes, four keys, 16 dims: lane x brings dims 4 (x % 4) .. of key x / 4, and takes dim x of the four. The lower
  // 32 lanes take keys 0 .. 3 (and 8 .. 11) of 16, the upper ones 4 .. 7 (and 12 .. 15), as their weights are.
  const int rv = 4 * lh + (lane >> 2 & 3);
  const uint32_t get_v = rv * RB + ((2 * (lane >> 4 & 1) + (lane >> 1 & 1)) ^ wide_vx<D>(rv)) * 16 + (lane & 1) * 8;

  // the column's reference, what is added to a weight's exponent, the score that a higher one renews them for (-inf: the
  // wave takes differences, whose reference is the running maximum), the sum of the weights
  float m = PG_LEAST, add = wide_up<DT> - fmaxf(m * a.c, PG_LEAST), most = m, l = 0.f;
  pg_f16 acc[ND];
#pragma unroll
  for (int T = 0; T < ND; ++T)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[T][e] = 0.f;

  // The wave's work on step j stands in three turns: its scores are made in j - 1's, its weights in its own, its outputs in
  // j + 1's, so that in each turn the matrix unit has one step's keys and another's values to work on while the vector unit
  // makes a third one's weights: all in one block of code, which what is rare only prepares or corrects. A product and
  // half of a pair of weights (two multiply-adds, two exponentials, packing, sum: 32 clocks) are a slot of that block, and the
  // slots stay in order.
  bool wild = false;  // step j - 1 has values that stand apart
  u16x8 kop[KS];
  auto read_k = [&](uint32_t gk) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < KS; ++k) kop[k] = ld16(reinterpret_cast<const uint16_t*>(lk + (gk ^ (32 * k))));
  };
  pg_u2 vop[2 * ND][2];  // of 32 dims, 16 keys
  auto read_v = [&](int n, uint32_t gv) __attribute__((always_inline)) {
#pragma unroll
    for (int q = 0; q < 2; ++q)
      vop[n][q] = __builtin_bit_cast(
          pg_u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) pg_s4*)(
                     lv + (gv ^ (64 * (n / 2))) + (16 * (n % 2) + 8 * q) * RB)));
  };
  auto output = [&](int n, const pg_u4 (&pop)[2]) __attribute__((always_inline)) {
    const pg_u4 v = {vop[n][0][0], vop[n][0][1], vop[n][1][0], vop[n][1][1]};
    acc[n / 2] = mfma32x32x16<DT>(__builtin_bit_cast(u16x8, v), __builtin_bit_cast(u16x8, pop[n % 2]), acc[n / 2]);
  };
  float ex[2];
  auto half_weight = [&](int n, const pg_f16& s, pg_u4 (&pop)[2]) __attribute__((always_inline)) {
    const int e = n / 2;
    if (n % 2 == 0) {
      ex[0] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * e], a.c, add));
      ex[1] = __builtin_fmaf(s[2 * e + 1], a.c, add);
      asm volatile("" : "+v"(ex[0]), "+v"(ex[1]));  // made in this slot, not where it is taken
    } else {
      uint32_t x = pg_pack<DT>(ex[0], __builtin_amdgcn_exp2f(ex[1]));
      l = pg_add2<DT>(x, l);
      asm volatile("" : "+v"(x), "+v"(l));
      pop[e / 4][e % 4] = x;
    }
  };
  // which of the two groups of 16 keys from `key` on lie in no page
  auto gaps = [&](int key) {
    uint32_t r = 0;
    for (int g = 0; g < 2; ++g) {
      const int k = key + 16 * g;
      if (k <= keys.last && (unsigned)pg_uniform(row[k >> c.shift]) >= (unsigned)c.pages) r |= 1u << g;
    }
    return r;
  };
  // Turn j, vn = j % 4 stages; s: the step's scores, next: the next one's; pop: the weights of the one before, made: its
  // own. A wave's last turn, j == steps, sees no key and only makes the outputs of the one before.
  auto turn = [&](int j, uint32_t vn, pg_f16& s, pg_f16& next, const pg_u4 (&pop)[2], pg_u4 (&made)[2]) __attribute__((always_inline)) {
    if (j > steps) return;
    read_k(get_k + ((vn + SB) & (RING - 1)));  // first: what follows covers their way
    __builtin_amdgcn_sched_barrier(0);
    uint32_t vs = (vn - SB) & (RING - 1);  // where the values of the step before lie
    const bool was_wild = wild;
    if (j < plain || j >= edge || holes) {
      const int key = keys.key(i0 + j);
      pg_mask<16, 8>(s, key + 4 * lh, min(cp, j == steps ? -1 : keys.last), pg_low(a, cp), a.sinks,
                     key <= none && key + KT > a.sinks, holes ? gaps(key) : 0u);
      float any = 0.f;
#pragma unroll
      for (int x = 0; x < SB / 1024; ++x) {
        const pg_u4 v = *reinterpret_cast<const pg_u4*>(lv + vn + (x * 64 + lane) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) any = pg_probe<DT>(v[e], any);
      }
      // Infinite and NaN values of a step that not all rows see stand apart: 0 in the product, whose values the wave then
      // takes from the spare stage (every wave that does so in this turn writes the same there), and added below to the
      // columns that see them, as in the narrow kernel.
      if (wild) {
#pragma unroll 1
        for (int x = lane * 16; x < SB; x += 1024) {
          pg_u4 v = *reinterpret_cast<const pg_u4*>(lv + vs + x);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = pg_tame<DT>(v[e]);
          *reinterpret_cast<pg_u4*>(lv + RING + x) = v;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        vs = RING;
      }
      wild = __ballot(any != any) != 0;
      if (wild) plain = max(plain, j + 2);  // the next turn comes here too
    }
    float mx = s[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
    // A reference is renewed once a score passes it by WIDE_SLACK: the column's sum so far goes by the new one, and behind
    // this turn its outputs
    const bool grew = __ballot(mx > most) != 0;
    float f;
    if (grew) {
      const float x = fmaxf(m, xor32_max(mx));
      const bool far = most == -INFINITY;
      const float to = wide_up<DT> - fmaxf(x * a.c, PG_LEAST);
      most = x + WIDE_SLACK * __builtin_amdgcn_rcpf(a.c);
      f = __builtin_amdgcn_exp2f(to - add);
      if (__builtin_expect(__ballot(far || (x > m && !(fabsf(to) <= WIDE_NEAR))) != 0, 0)) {
        f = __builtin_amdgcn_exp2f(far ? (m - x) * a.c : fminf(__builtin_fmaf(-x, a.c, -add) + wide_up<DT>, 1.f));
        add = wide_up<DT>;
        most = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] -= x;
      } else {
        add = to;
      }
      m = x;
      l *= f;
    }
    // one place for the scores behind the branch, or copies of them are made in every turn (8 x 200 rows 21.0 us, 21.6 without)
    asm volatile("" : "+v"(s));
    const uint32_t gv = get_v + vs;
    constexpr int SLOTS = KS + 2 * ND, LEAD = 2;  // LEAD: slots that a value's read is ahead of its product (1: 4 % slower, 4: 1 %)
#pragma unroll
    for (int e = 0; e < 16; ++e) next[e] = 0.f;
#pragma unroll
    for (int n = 0; n < LEAD - KS; ++n) read_v(n, gv);
    // A wave in its products goes before the SIMD's other one, which masks or looks for a maximum: 4096 rows onto 12288 keys 933
    // -> 916 us, 4 x 700 rows onto 3000 165 -> 160. With heads of 64, whose turns are mostly vector work, 5 % less to 8 % more.
    if constexpr (D == 128) __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      if (i + LEAD >= KS && i + LEAD < SLOTS) read_v(i + LEAD - KS, gv);
      if (i < KS) next = mfma32x32x16<DT>(kop[i], qop[i], next);
      else output(i - KS, pop);
#pragma unroll
      for (int h = 0; h < 16 / SLOTS; ++h) half_weight(i * (16 / SLOTS) + h, s, made);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (D == 128) __builtin_amdgcn_s_setprio(0);
    if (was_wild) {
      const int key = keys.key(i0 + j - 1);
      const uint32_t gap = holes ? gaps(key) : 0u;
      for (int k = 0; k < KT; ++k) {
        if (key + k > keys.last || (gap >> (k >> 4) & 1u)) continue;
        if (pg_hidden(key + k, min(cp, keys.last), pg_low(a, cp), a.sinks)) continue;
#pragma unroll
        for (int n = 0; n < 4 * ND; ++n) {
          const pg_u2 x = *reinterpret_cast<const pg_u2*>(lv + ((vn - SB) & (RING - 1)) + k * RB +
                                                          (n ^ wide_vx<D>(k & 15)) * 16 + lh * 8);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[n / 4][4 * (n % 4) + r] += pg_wild_number<DT>((uint16_t)(x[r / 2] >> (16 * (r & 1))));
        }
      }
    }
    if (grew) {
#pragma unroll
      for (int T = 0; T < ND; ++T) acc[T] *= f;
    }
  };

  fetch(i0);
  // the queries came before the pages' numbers: taken here, or the compiler waits for them behind the loads it does not know
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    pg_u4 x = __builtin_bit_cast(pg_u4, qop[k]);
    asm volatile("" : "+v"(x));
    qop[k] = __builtin_bit_cast(u16x8, x);
  }
  bring_k(i0, 0);
  bring_v(0);
  bring_k(i0 + 1, SB);
  bring_v(SB);
  bring_k(i0 + 2, 2 * SB);
  // the first turn's outputs: of weights and values of 0, in the stage that is filled last
  for (int x = (threadIdx.x & 255) * 16; x < SB; x += 4096) *reinterpret_cast<pg_u4*>(lv + 3 * SB + x) = pg_u4{0, 0, 0, 0};
  pg_landed<4 * LI>();
  __syncthreads();
  pg_f16 s0, s1;
  pg_u4 p0[2] = {pg_u4{0, 0, 0, 0}, pg_u4{0, 0, 0, 0}}, p1[2];
  read_k(get_k);
#pragma unroll
  for (int e = 0; e < 16; ++e) s0[e] = 0.f;
#pragma unroll
  for (int k = 0; k < KS; ++k) s0 = mfma32x32x16<DT>(kop[k], qop[k], s0);
  auto round = [&](int j, uint32_t vn, pg_f16& s, pg_f16& next, const pg_u4 (&pop)[2], pg_u4 (&made)[2]) __attribute__((always_inline)) {
    pg_landed<2 * LI>();  // K of step j + 1 and V of step j (behind them: V of j + 1, K of j + 2)
    __syncthreads();      // for everyone; and everyone is done with K of step j and V of j - 2
    bring_v(vn ^ 2 * SB);
    bring_k(i0 + j + 3, (vn + 3 * SB) & (RING - 1));
    turn(j, vn, s, next, pop, made);
  };
  // Two rounds at a time, which hand each other scores and weights. A call of few workgroups is short: its time is the
  // code's first fetch into the instruction cache, so there the round stands once and moves them.
  if constexpr (KG == 1) {
    for (int j = 0, vn = 0; j <= n; j += 2, vn ^= 2 * SB) {
      if (i0 + j + 4 - base >= 64) fetch(i0 + j + 3);
      round(j, vn, s0, s1, p0, p1);
      if (j < n) round(j + 1, vn + SB, s1, s0, p1, p0);
    }
  } else {
    for (int j = 0, vn = 0; j <= n; ++j, vn = (vn + SB) & (RING - 1)) {
      if (i0 + j + 3 - base >= 64) fetch(i0 + j + 3);
      round(j, vn, s0, s1, p0, p1);
      s0 = s1;
      p0[0] = p1[0];
      p0[1] = p1[1];
    }
  }
  pg_landed<0>();

  // by what power of two the sums are to be taken up to stand at 2^wide_up at m (what add's rounding left; a column that saw
  // nothing has sums of 0)
  const float due = most == -INFINITY ? 0.f : __builtin_amdgcn_fmed3f(wide_up<DT> - __builtin_fmaf(m, a.c, add), -1.f, 1.f);
  if constexpr (KG == 1) {  // lane (column, lh) holds dims 8 n + 4 lh + r
    const float L = xor32_sum(l);
    if (!col.live) return;
    if (keys.active == 1) {
      uint16_t* op = a.out + (long)(w.first + col.j) * a.so_b + (long)(w.kh * a.G + col.h) * a.so_h + 4 * lh;
#pragma unroll
      for (int n = 0; n < 4 * ND; ++n) {
        const pg_f16& x = acc[n / 4];
        pg_store4<DT>(op + 8 * n, f32x4_t{x[n % 4 * 4], x[n % 4 * 4 + 1], x[n % 4 * 4 + 2], x[n % 4 * 4 + 3]}, L);
      }
    } else {
      const long place = (long)blockIdx.y * gridDim.x + blockIdx.x, ncols = (long)gridDim.y * gridDim.x * COLS;
      const long at = (place * COLS + 32 * wave + li) * a.splits + split;
      const float g = __builtin_amdgcn_exp2f(due);
#pragma unroll
      for (int n = 0; n < 4 * ND; ++n) {
        const pg_f16& x = acc[n / 4];
        *reinterpret_cast<f32x4_t*>(a.part + at * D + 8 * n + 4 * lh) =
            f32x4_t{x[n % 4 * 4], x[n % 4 * 4 + 1], x[n % 4 * 4 + 2], x[n % 4 * 4 + 3]} * g;
      }
      if (lh == 0) *reinterpret_cast<float2*>(a.part + ncols * a.splits * D + at * 2) = make_float2(m, L * g);
    }
    return;
  }
  // The key groups' sums by way of LDS, and to 16-byte stores of whole rows: few instructions, which matter in a short call,
  // since each is fetched for one use (8 x 200 rows 23.1 us with the groups' sums in registers, 21.0 so; with one group,
  // where the stores above are fewer bytes moved, 3200 rows 28.0 and 28.5). An n's chunks lie at their column XOR a number
  // of n, so that neither side meets a bank twice.
  __syncthreads();
  constexpr int NC = 4 * ND, SW = 16 / NC;
  f32x4_t* const out = reinterpret_cast<f32x4_t*>(lds);
  float4* const ml = reinterpret_cast<float4*>(lds + KG * 4 * NC * 1024);
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const pg_f16& x = acc[n / 4];
    out[((group * 4 + wave) * NC + n) * 64 + (lane ^ SW * n)] = f32x4_t{x[n % 4 * 4], x[n % 4 * 4 + 1], x[n % 4 * 4 + 2], x[n % 4 * 4 + 3]};
  }
  l = xor32_sum(l);
  if (lh == 0) ml[(group * 4 + wave) * 32 + li] = make_float4(m, l, due, 0.f);
  __syncthreads();
#pragma unroll 1
  for (int x = threadIdx.x; x < COLS * NC; x += 256 * KG) {
    const int n = x % NC, y = x / NC, at = ((y / 32) * NC + n) * 64 + (y % 32 ^ SW * n);
    const Col cc(a, w, w.block * COLS + y);
    if (!cc.live) continue;
    const float4 m0 = ml[y], m1 = ml[128 + y];
    const float M = fmaxf(m0.x, m1.x);
    const float f0 = __builtin_amdgcn_exp2f(__builtin_fmaf(m0.x - M, a.c, m0.z));
    const float f1 = __builtin_amdgcn_exp2f(__builtin_fmaf(m1.x - M, a.c, m1.z));
    const f32x4_t o0 = out[at] * f0 + out[at + 4 * NC * 64] * f1, o1 = out[at + 32] * f0 + out[at + 4 * NC * 64 + 32] * f1;
    const float L = m0.y * f0 + m1.y * f1;
    if (keys.active == 1) {
      const float r = L == 0.f ? 0.f : 1.f / L;
      *reinterpret_cast<pg_u4*>(a.out + (long)(w.first + cc.j) * a.so_b + (long)(w.kh * a.G + cc.h) * a.so_h + 8 * n) =
          pg_u4{pg_pack<DT>(o0[0] * r, o0[1] * r), pg_pack<DT>(o0[2] * r, o0[3] * r), pg_pack<DT>(o1[0] * r, o1[1] * r),
                pg_pack<DT>(o1[2] * r, o1[3] * r)};
    } else {
      const long place = (long)blockIdx.y * gridDim.x + blockIdx.x, ncols = (long)gridDim.y * gridDim.x * COLS;
      const long col = (place * COLS + y) * a.splits + split;
      *reinterpret_cast<f32x4_t*>(a.part + col * D + 8 * n) = o0;
      *reinterpret_cast<f32x4_t*>(a.part + col * D + 8 * n + 4) = o1;
      if (n == 0) *reinterpret_cast<float2*>(a.part + ncols * a.splits * D + col * 2) = make_float2(M, L);
    }
  }
}

// Joins the splits: D / 4 threads a column, in the splits' order
template <int DT, int D, int KT, int LEAST>
__global__ __launch_bounds__(256) void paged_join_kernel(Paged c, PagedAttn a, int cols) {
  constexpr int TD = D / 4, CB = 256 / TD;
  const Where w = pg_where(c, a, blockIdx.x, blockIdx.y);
  if (w.n == 0) return;
  const Keys<KT> keys(c, a, w, LEAST);
  if (keys.active <= 1) return;  // written by the attention itself
  const int col = blockIdx.z * CB + threadIdx.x / TD;  // z: which CB of the block's columns
  const Col cc(a, w, w.block * cols + col);
  if (!cc.live) return;
  const long place = (long)blockIdx.y * gridDim.x + blockIdx.x, ncols = (long)gridDim.y * gridDim.x * cols;
  pg_join<DT, D, 0>(a, w, cc, place, cols, col, ncols, keys.active, threadIdx.x % TD * 4);
}

// ---------------------------------------------------------------------------------------------------------
namespace {
template <int DT, int D> void paged_launch(const Paged& c, const PagedAttn& a, int tiles, int cols, bool single, hipStream_t st) {
  const int x = c.kv_heads * a.blocks;
  const dim3 grid(x, tiles, a.splits);
  if (cols == 128) {
    // Up to a workgroup a CU, two groups of waves share its keys (us with two groups, with one: 512 rows onto 16000 keys
    // unsplit 254, 324, 2048 rows onto nothing 45, 50; above, 4 x 700 rows under a window 56, 34, 4096 rows 1030, 917)
    if ((long)x * tiles * a.splits <= 256) hipLaunchKernelGGL((paged_wide_kernel<DT, D, 2>), grid, dim3(512), 0, st, c, a);
    else hipLaunchKernelGGL((paged_wide_kernel<DT, D, 1>), grid, dim3(256), 0, st, c, a);
  } else if (cols == 48) {
    if constexpr (D == 64) hipLaunchKernelGGL((paged_narrow_kernel<DT, D, 3, false>), grid, dim3(256), 0, st, c, a);
  } else if (cols == 32) {
    hipLaunchKernelGGL((paged_narrow_kernel<DT, D, 2, false>), grid, dim3(256), 0, st, c, a);
  } else if (single) {
    hipLaunchKernelGGL((paged_narrow_kernel<DT, D, 1, true>), grid, dim3(256), 0, st, c, a);
  } else {
    hipLaunchKernelGGL((paged_narrow_kernel<DT, D, 1, false>), grid, dim3(256), 0, st, c, a);
  }
  if (a.splits > 1 && cols == 128)
    hipLaunchKernelGGL((paged_join_kernel<DT, D, WIDE_KT, WIDE_LEAST>), dim3(x, tiles, cols / (1024 / D)), dim3(256), 0, st, c,
                       a, cols);
}
// workgroups a split: tiles x kv heads x blocks of the columns; 0: out of range
long paged_items(long tiles, int kv_heads, int heads, int tile_rows, int cols, int head_dim) {
  if (tiles < 0 || tiles > 65535 || kv_heads <= 0 || heads <= 0 || tile_rows <= 0 || heads % kv_heads) return 0;
  if ((long)tile_rows * (heads / kv_heads) >= 65536 - cols) return 0;  // columns are counted in 16 bits
  if (cols != 16 && cols != 32 && cols != 128 && !(cols == 48 && head_dim == 64)) return 0;
  const long per_tile = kv_heads * (((long)tile_rows * (heads / kv_heads) + cols - 1) / cols);
  return tiles * per_tile < 1L << 24 ? tiles * per_tile : 0;
}
}  // namespace

M3X_API size_t m3x_paged_attn_workspace(int tiles, int kv_heads, int heads, int tile_rows, int cols, int head_dim, int splits) {
  if (splits <= 1 || head_dim <= 0) return 0;
  return (size_t)paged_items(tiles, kv_heads, heads, tile_rows, cols, head_dim) * cols * splits * (head_dim + 2) * sizeof(float);
}

M3X_API int m3x_paged_attn(const M3xPagedKv* cache, const void* q, long sq_b, long sq_h, void* out, long so_b, long so_h,
                           const int64_t* slots, const int32_t* pos, const int32_t* tiles, int ntiles, int tile_rows,
                           int cols, float scale, int rows, int heads, int window, int sinks, int splits, void* workspace,
                           size_t ws_bytes, int32_t* arrived, void* stream) {
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
  const long items = paged_items(ntiles, c.kv_heads, heads, tile_rows, cols, cache->head_dim);
  if (items == 0) return M3X_EINVAL;
  if (splits > 1) {
    if (!workspace || (cols != 128 && !arrived)) return M3X_ENULL;
    if (((uintptr_t)arrived & 3u)) return M3X_EINVAL;
    if (ws_bytes < m3x_paged_attn_workspace(ntiles, c.kv_heads, heads, tile_rows, cols, cache->head_dim, splits))
      return M3X_EWORKSPACE;
    if (!m3x_aligned16(workspace)) return M3X_EINVAL;
  }
  // The factor of the scores' exponents, never 0 (0 * -inf of a hidden key). fp32's smallest number stands for all below it:
  // scores up to 2^127 weigh alike under either, within 2^-21.
  const float factor = std::max(fabsf(scale) * 1.44269504088896341f, 0x1p-149f);
  const int G = heads / c.kv_heads;
  const PagedAttn a = {(const uint16_t*)q, sq_b, sq_h, (uint16_t*)out, so_b, so_h, slots, pos, tiles, factor,
                       scale < 0.f ? 0x80008000u : 0u, rows, heads, G, tile_rows, (tile_rows * G + cols - 1) / cols,
                       std::min(window, 1 << 30), std::min(sinks, 1 << 30), splits,
                       G == 1 ? 0u : (uint32_t)(((1ull << 32) + G - 1) / G), (float*)workspace, arrived};
  hipStream_t st = (hipStream_t)stream;
  const bool single = tile_rows == 1;
  const int D = cache->head_dim;
  if (cache->dtype == M3X_BF16 && D == 128) paged_launch<M3X_BF16, 128>(c, a, ntiles, cols, single, st);
  else if (cache->dtype == M3X_BF16) paged_launch<M3X_BF16, 64>(c, a, ntiles, cols, single, st);
  else if (D == 128) paged_launch<M3X_F16, 128>(c, a, ntiles, cols, single, st);
  else paged_launch<M3X_F16, 64>(c, a, ntiles, cols, single, st);
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}
