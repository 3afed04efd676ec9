// The 4-bit KV cache: its writers, its reader and the attention over it (format: m3x_fp4.h).
//
// Layout, D = head_dim, per (slot, kv head), cap positions (a multiple of 32):
//   k   [cap][D / 2]            byte j of a position: dims 2j, 2j + 1. The lane (key, quarter) of the score product's
//                               operand takes D / 8 consecutive bytes: 16 keys are one contiguous load of a wave.
//   ks  [cap][D / 32]           scale bytes of the position's groups
//   v   [cap / 4][16][4][D/32]  four positions together; chunk c holds dims [c D/16, (c + 1) D/16). The lane (chunk,
//                               quarter) of the output product's operand takes four positions of its chunk in one
//                               16-byte load (8 at D = 64), and 16 positions are one contiguous load of a wave, so V
//                               needs no transpose through LDS; a position's write stays whole words.
//   vs  [cap / 4][D / 32][4]    the four positions' bytes of a group are one word
#include <algorithm>
#include <cstring>
#include <type_traits>

#include "m3x_norm.h"
#include "m3x_fp4.h"

// mirror of M3xKv4 (include/m3x.h)
struct M3xKv4 {
  void* k;
  void* ks;
  void* v;
  void* vs;
  int slots, kv_heads, head_dim, cap;
};

namespace {
// Attention's workgroups: 4 waves, 4 on a SIMD (128 registers; no spill, 18 spilled registers cost 30 %). Measured with 4
// waves, 8 and 2, heads 16/8 of 128 (us): 224 rows of 2048 keys 79, 80, 89; of 300 keys 18, 23, 20; 8 x 200 prompt rows over
// 500 keys 21, 26, 25.
constexpr int KV4_NW = 4, KV4_OCC = 4;

struct Kv4 {
  uint8_t* k;
  uint8_t* ks;
  uint8_t* v;
  uint8_t* vs;
  int slots, kv_heads, cap;
};

template <int D> __device__ __forceinline__ long kv4_pos(const Kv4& c, long slot, int kh, int p) {
  return ((slot * c.kv_heads + kh) * c.cap + p);  // position index; * D / 2 (k), * D / 32 (ks, and vs blocks of 4)
}

// store of thread t's 8 elements (dims 8t .. 8t + 7) of one position's key and value
template <int DT, int D>
__device__ __forceinline__ void kv4_store(const Kv4& c, long slot, int kh, int p, int t, const u16x8& kx, const u16x8& vx,
                                          bool active) {
  uint32_t kb, vb;
  const uint32_t kw = fp4_quantise8<DT>(kx, kb);
  const uint32_t vw = fp4_quantise8<DT>(vx, vb);
  if (!active) return;
  const long at = kv4_pos<D>(c, slot, kh, p);
  *reinterpret_cast<uint32_t*>(c.k + at * (D / 2) + 4 * t) = kw;
  const long blk = at >> 2;
  uint8_t* vp = c.v + blk * (2 * D);
  if constexpr (D == 128) {
    *reinterpret_cast<uint32_t*>(vp + 16 * t + 4 * (p & 3)) = vw;
  } else {
    *reinterpret_cast<uint16_t*>(vp + 16 * t + 2 * (p & 3)) = (uint16_t)vw;
    *reinterpret_cast<uint16_t*>(vp + 16 * t + 8 + 2 * (p & 3)) = (uint16_t)(vw >> 16);
  }
  if ((t & 3) == 0) {
    c.ks[at * (D / 32) + (t >> 2)] = (uint8_t)kb;
    c.vs[blk * (D / 8) + (t & ~3) + (p & 3)] = (uint8_t)vb;
  }
}

__device__ __forceinline__ bool kv4_inside(const Kv4& c, long slot, int p) {
  return slot >= 0 && slot < c.slots && p >= 0 && p < c.cap;
}
}  // namespace

// K and V rows into the cache, D / 8 threads per (row, kv head): a thread's eight numbers are one word of codes, four
// threads' a group. Bound by the launch at few rows (1.7 us), by one memory round trip beside the rows' bytes at many: 2048
// rows of 8 heads of 128 (8.4 MB in, 2.2 MB out) 5.4 us.
template <int DT, int D>
__global__ __launch_bounds__(256) void kv4_append_kernel(const uint16_t* __restrict__ k, long sk_r, long sk_h,
                                                         const uint16_t* __restrict__ v, long sv_r, long sv_h, Kv4 c,
                                                         const int64_t* __restrict__ slots,
                                                         const int32_t* __restrict__ pos, int rows) {
  constexpr int TPI = D / 8;
  const int t = threadIdx.x % TPI;
  const long item = (long)blockIdx.x * (256 / TPI) + threadIdx.x / TPI;
  const long row = item / c.kv_heads;
  const int kh = (int)(item % c.kv_heads);
  const long r = row < rows ? row : 0;  // spare threads compute on row 0 and store nothing (quads exchange lanes)
  const u16x8 kx = ld16(k + r * sk_r + kh * sk_h + 8 * t);
  const u16x8 vx = ld16(v + r * sv_r + kh * sv_h + 8 * t);
  const long slot = slots[r];
  const int p = pos[r];
  kv4_store<DT, D>(c, slot, kh, p, t, kx, vx, row < rows && kv4_inside(c, slot, p));
}

// qk_norm_rope_cache_kernel's arithmetic and bits with the keys and values quantised into the 4-bit cache: one pass
// over q|k|v instead of two, and no 16-bit keys in between. Bound as kv4_append_kernel; 16/8 heads of 128: 1 row 2.5 us, 224
// rows 4.2, 2048 rows (27 MB) 10.0, as qk_norm_rope_cache_kernel's 2.6, 4.3 and 9.6.
template <int D>
__global__ __launch_bounds__(256) void qk_norm_rope_kv4_kernel(
    const uint16_t* __restrict__ qkv, long s_qkv, uint16_t* __restrict__ qo, long s_qo_b, long s_qo_h, Kv4 c,
    const int64_t* __restrict__ slots, const int32_t* __restrict__ pos, const uint16_t* __restrict__ cosb,
    const uint16_t* __restrict__ sinb, long s_cos, const uint16_t* __restrict__ wq, const uint16_t* __restrict__ wk,
    float eps, int rows, int H) {
  constexpr int TPI = D / 8;
  const int t = threadIdx.x % TPI;
  const long item = (long)blockIdx.x * (256 / TPI) + threadIdx.x / TPI;
  const int KV = c.kv_heads, NH = H + KV;
  const long row = item / NH;
  const int j = (int)(item % NH);
  const bool active = row < rows;
  const long r = active ? row : 0;
  const int p = pos[r];
  const int ps = min(max(p, 0), c.cap - 1);  // the tables' row, kept inside them
  const long slot = slots[r];
  const int kh = j < H ? 0 : j - H;
  const u16x8 xv = ld16(qkv + r * s_qkv + (long)j * D + 8 * t);
  const u16x8 wv = ld16((j < H ? wq : wk) + 8 * t);
  const u16x8 vv = ld16(qkv + r * s_qkv + (long)(H + KV + kh) * D + 8 * t);
  const u16x8 cv = ld16(cosb + (long)ps * s_cos + 8 * t);
  const u16x8 sv = ld16(sinb + (long)ps * s_cos + 8 * t);
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = bf2f(xv.v[e]);
  const u16x8 ov = qk_norm_rope8<D>(x, wv, cv, sv, eps, t);
  if (active && j < H) st16(qo + row * s_qo_b + (long)j * s_qo_h + 8 * t, ov);
  kv4_store<M3X_BF16, D>(c, slot, kh, p, t, ov, vv, active && j >= H && kv4_inside(c, slot, p));
}

// Positions of the cache as 16-bit rows (zeros for a row outside it). Bound by the rows' bytes: stored with the
// non-temporal hint, passes over 16 x 4095 positions of 8 heads of 64 take 32.2 us (170 MB, 5.3 TB/s; a large copy's
// 5.1), without it 45.6 (each pass then waits for the last one's lines to leave the caches).
__device__ __forceinline__ void st16_nt(uint16_t* p, const u16x8& x) {
  __builtin_nontemporal_store(__builtin_bit_cast(fp4_u4, x), reinterpret_cast<fp4_u4*>(p));
}
template <int DT, int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(Kv4 c, const int64_t* __restrict__ slots,
                                                       const int32_t* __restrict__ pos, uint16_t* __restrict__ k,
                                                       long sk_r, long sk_h, uint16_t* __restrict__ v, long sv_r,
                                                       long sv_h, int rows) {
  constexpr int TPI = D / 8;
  const int t = threadIdx.x % TPI;
  const long item = (long)blockIdx.x * (256 / TPI) + threadIdx.x / TPI;
  const long row = item / c.kv_heads;
  const int kh = (int)(item % c.kv_heads);
  if (row >= rows) return;
  const long slot = slots[row];
  const int p = pos[row];
  u16x8 kx, vx;
  if (kv4_inside(c, slot, p)) {
    const long at = kv4_pos<D>(c, slot, kh, p), blk = at >> 2;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(c.k + at * (D / 2) + 4 * t);
    const uint8_t* vp = c.v + blk * (2 * D);
    uint32_t vw;
    if constexpr (D == 128) {
      vw = *reinterpret_cast<const uint32_t*>(vp + 16 * t + 4 * (p & 3));
    } else {
      vw = *reinterpret_cast<const uint16_t*>(vp + 16 * t + 2 * (p & 3)) |
           (uint32_t)*reinterpret_cast<const uint16_t*>(vp + 16 * t + 8 + 2 * (p & 3)) << 16;
    }
    kx = fp4_eight<DT>(kw, fp4_scale(c.ks[at * (D / 32) + (t >> 2)]));
    vx = fp4_eight<DT>(vw, fp4_scale(c.vs[blk * (D / 8) + (t & ~3) + (p & 3)]));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) kx.v[e] = vx.v[e] = 0;
  }
  st16_nt(k + row * sk_r + kh * sk_h + 8 * t, kx);
  st16_nt(v + row * sv_r + kh * sv_h + 8 * t, vx);
}

// ---------------------------------------------------------------------------------------------------------
// Attention over the cache: out[r, h, :] = softmax(scale q[r, h] . K^T) V over positions 0 .. pos[r] of slot slots[r].
//
// A workgroup takes one (block of rows, kv head, split of the keys). The score product has the keys as its rows and
// 16 columns: the G query heads of up to 16 / G rows that stand next to each other in the call, of one slot at
// consecutive positions (a prompt's), found from slots and pos by the workgroup itself; the block's later rows' own
// workgroups leave at once. A single token is a block of one row. Each of the NW waves takes every NW-th 32-key tile:
//   S^T = K . Q^T   per 16 keys D / 32 MFMA 16x16x32: a lane's words of K become 16-bit operands in registers
//   softmax         running maximum and sum in fp32, exp2; a lane keeps its own column's, its keys' partial sum
//   O^T += V^T . P  D / 16 MFMA per 32 keys: S^T's accumulator is the P operand as it stands, and V's words, which
//                   hold two dims of a key each, are paired over keys by byte permutes
// P is rounded to the 16-bit type (at most half a step, relative 2^-8 bf16 / 2^-11 fp16, per key), and its sum is the
// rounded weights'; everything else between the loads and the output is exact or fp32. A weight's reference is the
// maximum itself: one renewed only when a score passes it by 2^8 saves 3 to 5 % where the arithmetic bounds, but then
// the largest weight is rounded too, and the error against 64 bits rises by a sixth.
//
// Bound, measured on MI355X with 16/8 heads of 128: the cache's bytes where rows fill the GPU (224 rows of 2048 keys
// 77 us, 499 MB at 6.5 TB/s; of 4000 keys 145, 6.7 TB/s; VALU busy 47 %).
// Few rows: the start, the merge and the join beside the bytes (2 rows of 120000 keys, 32/4 heads of 64: 16.3 us of 65 MB
// and 4.0 for the join; one row of 2048 keys 4.5 and 3.4). A prompt over a long context: a tile's own chain of steps, about
// 1 us at two waves a SIMD (512 rows over 4000 keys 34 us); over a short one a block's start and merge (1600 rows over up
// to 500 keys 21 us). Every block of 16 columns converts its keys and values anew.
namespace {
template <int NI> struct Words { uint32_t w[NI]; };
// A tile of the cache at `base`, the same in every lane; where `live` is false its loads give zeros and access nothing:
// the loads ahead past a wave's last tile would read a tile again (what it gave when it came: 1600 single rows of 500 keys
// 181 -> 151 us, 224 of 2048 80.5 -> 77).
typedef __amdgpu_buffer_rsrc_t Kv4Ref;
__device__ __forceinline__ Kv4Ref kv4_ref(const uint8_t* base, bool live, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, live ? bytes : 0, 0x00020000);
}
// 4 NI bytes at a lane's offset; nt: non-temporal
template <int NI, bool NT> __device__ __forceinline__ Words<NI> kv4_load(Kv4Ref ref, uint32_t off) {
  constexpr int AUX = NT ? 2 : 0;
  Words<NI> r;
  if constexpr (NI == 4) {
    const fp4_u4 x = __builtin_amdgcn_raw_buffer_load_b128(ref, off, 0, AUX);
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = x[i];
  } else {
    const fp4_u2 x = __builtin_amdgcn_raw_buffer_load_b64(ref, off, 0, AUX);
    r.w[0] = x[0];
    r.w[1] = x[1];
  }
  return r;
}

struct Kv4Attn {
  const uint16_t* q;
  long sq_b, sq_h;
  uint16_t* out;
  long so_b, so_h;
  const int64_t* slots;
  const int32_t* pos;
  float scale_log2;   // |scale| log2(e), not 0
  uint32_t q_flip;    // the sign bits of two query elements where scale < 0
  int rows, heads, G, hblocks, qb, R, chunk, max_ctx, max_splits;
  uint32_t over_Gc;  // x * over_Gc >> 8 = x / min(G, 16) for x < 16
  float* part;  // [rows * heads][max_splits][D] then [rows * heads][max_splits][2] (largest raw score, sum)
};

// four outputs O / L (one quotient: its rounding and the products' are fp32's)
template <int DT> __device__ __forceinline__ void kv4_store_out(uint16_t* p, const f32x4_t& O, float L) {
  const float r = 1.f / L;
  *reinterpret_cast<uint2*>(p) = make_uint2(E<DT>::from_f(O[0] * r) | (uint32_t)E<DT>::from_f(O[1] * r) << 16,
                                            E<DT>::from_f(O[2] * r) | (uint32_t)E<DT>::from_f(O[3] * r) << 16);
}

// the A operands of dim tiles 2 B and 2 B + 1 over 32 keys (two 16-key groups' words v0, v1 and scale words s0, s1):
// element e is the number of dim 2 B (+ 1) of the lane's chunk at key e
template <int DT, int D, int B>
__device__ __forceinline__ void kv4_vop(const Words<D / 32>& v0, const Words<D / 32>& v1, uint32_t s0, uint32_t s1,
                                        u16x8& lo, u16x8& hi) {
  uint32_t a[8];
#define KV4_PAIR(E, V, S)                                                                              \
  if constexpr (D == 128) a[E] = fp4_pair<DT, B>(V.w[E & 3], fp4_scale_of<E & 3>(S));                 \
  else a[E] = fp4_pair<DT, 2 * (E & 1) + B>(V.w[(E & 3) >> 1], fp4_scale_of<E & 3>(S));
  KV4_PAIR(0, v0, s0) KV4_PAIR(1, v0, s0) KV4_PAIR(2, v0, s0) KV4_PAIR(3, v0, s0)
  KV4_PAIR(4, v1, s1) KV4_PAIR(5, v1, s1) KV4_PAIR(6, v1, s1) KV4_PAIR(7, v1, s1)
#undef KV4_PAIR
  fp4_u4 l, h;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    l[i] = __builtin_amdgcn_perm(a[2 * i + 1], a[2 * i], 0x05040100u);
    h[i] = __builtin_amdgcn_perm(a[2 * i + 1], a[2 * i], 0x07060302u);
  }
  lo = __builtin_bit_cast(u16x8, l);
  hi = __builtin_bit_cast(u16x8, h);
}

template <int DT, int D, int NG, int B = 0>
__device__ __forceinline__ void kv4_pv(const Words<D / 32> (&v)[NG], const uint32_t (&vs)[NG],
                                       const fp4_u4 (&pop)[NG / 2], f32x4_t (&acc)[D / 16]) {
#pragma unroll
  for (int h = 0; h < NG / 2; ++h) {
    u16x8 lo, hi;
    kv4_vop<DT, D, B>(v[2 * h], v[2 * h + 1], vs[2 * h], vs[2 * h + 1], lo, hi);
    const u16x8 p = __builtin_bit_cast(u16x8, pop[h]);
    acc[2 * B] = mfma16x16x32<DT>(lo, p, acc[2 * B]);
    acc[2 * B + 1] = mfma16x16x32<DT>(hi, p, acc[2 * B + 1]);
  }
  if constexpr (B + 1 < D / 32) kv4_pv<DT, D, NG, B + 1>(v, vs, pop, acc);
}

}  // namespace

template <int D, int NW> struct Kv4Lds {
  __align__(16) float o[NW][16][D + 4];
  float m[NW][16], l[NW][16];
  long slot[64];
  int pos[64];
};
// the lane's number, made anew: kept over the loop over the keys it, and what comes from it, would spill
__device__ __forceinline__ int kv4_lane() {
  int x;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
  return x;
}
// a column of a block of n rows, the first at position p0: query head hq of row jq, which sees the keys up to pq
struct Kv4Col {
  int jq, hq, pq;
  bool live;
  __device__ __forceinline__ Kv4Col(const Kv4Attn& a, int li, int n, int Gc, int p0, int plim) {
    jq = li * a.over_Gc >> 8;
    hq = li - jq * min(a.G, 16);
    live = jq < n && hq < Gc;
    pq = live ? min(p0 + jq, plim) : -1;
  }
};
// one block: rows row .. row + n - 1 of slot `slot`, the first at position p0
template <int DT, int D, int NW, bool NT>
__device__ __forceinline__ void kv4_attn_row(const Kv4& c, const Kv4Attn& a, int row, int n, long slot, int p0, int kh,
                                             int h0, int Gc, int split, int wave, Kv4Lds<D, NW>& lds) {
  constexpr int NI = D / 32;   // words a lane holds of 16 keys; score steps
  constexpr int ND = D / 16;   // dim tiles
  constexpr int KT = 32, NG = KT / 16;  // keys of a tile, and its 16-key groups
  const int lane = kv4_lane(), li = lane & 15, lg = lane >> 4;
  const int plim = min(c.cap, a.max_ctx) - 1;  // the caller keeps pos below both; accesses stay inside whatever pos holds
  if (slot < 0 || slot >= c.slots || p0 < 0) {  // no key: zeros
    if (split == 0)
      for (int j = 0; j < n; ++j)
        for (int i = 64 * wave + kv4_lane(); i < Gc * D; i += 64 * NW)
          a.out[(long)(row + j) * a.so_b + (long)(kh * a.G + h0 + i / D) * a.so_h + i % D] = 0;
    return;
  }
  const int plast = min(p0 + n - 1, plim);
  const int kstart = split * a.chunk;
  if (kstart > plast) return;
  const int kend = min(kstart + a.chunk, plast + 1);

  const long base = (slot * c.kv_heads + kh) * (long)c.cap;
  // scale bytes come as whole words (a byte's widening would be waited for where it is loaded): the key's four at
  // D = 128, two keys' two each at D = 64; ks_rot brings the lane's byte to the exponent's place
  const uint32_t k_at = li * (D / 2) + lg * (D / 8), ks_at = (li * NI) & ~3;
  const int ks_rot = (23 - 8 * (D == 128 ? lg : 2 * (li & 1) + (lg >> 1))) & 31;
  const uint32_t v_at = lg * (2 * D) + li * (D / 8), vs_at = lg * (4 * NI) + (D == 128 ? li >> 2 : li >> 3) * 4;
  // a column past the block's rows computes with the first row's queries and is dropped
  u16x8 qop[NI];
  const Kv4Col col(a, li, n, Gc, p0, plim);
  const uint16_t* qp =
      a.q + (long)(row + (col.live ? col.jq : 0)) * a.sq_b + (long)(kh * a.G + h0 + (col.live ? col.hq : 0)) * a.sq_h;
#pragma unroll
  for (int i = 0; i < NI; ++i) qop[i] = ld16(qp + (D / 4) * lg + 8 * i);
  // Two tiles' words in turn: a tile's keys are loaded two tiles ahead, behind the products of the keys they replace, its
  // values likewise. The pointers stand at the tile to be loaded next and are the same in every lane: a load takes them
  // as its scalar address, beside the lane's 32-bit offset. Loads are never conditional (one whose registers are merged
  // behind a branch is waited for there): past the wave's last tile they are of no bytes. cap % 32 == 0: a tile that begins
  // inside the slot ends inside it.
  struct Buf {
    Words<NI> kw[NG], vw[NG];
    uint32_t ks[NG], vs[NG];
  };
  int k0 = kstart + KT * wave;
  const long tile0 = base + k0;
  const uint8_t* kp = c.k + tile0 * (D / 2);
  const uint8_t* ksp = c.ks + tile0 * NI;
  const uint8_t* vp = c.v + tile0 * (D / 2);
  const uint8_t* vsp = c.vs + tile0 * NI;
  int kn = k0, vn = k0;
  auto load_k = [&](Buf& t) {
    const Kv4Ref kr = kv4_ref(kp, kn < kend, KT * D / 2), sr = kv4_ref(ksp, kn < kend, KT * NI);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      t.kw[g] = kv4_load<NI, NT>(kr, k_at + g * (8 * D));
      t.ks[g] = __builtin_amdgcn_raw_buffer_load_b32(sr, ks_at + g * (16 * NI), 0, 0);
    }
    kn += KT * NW;
    kp += KT * NW * (D / 2);
    ksp += KT * NW * NI;
  };
  auto load_v = [&](Buf& t) {
    const Kv4Ref vr = kv4_ref(vp, vn < kend, KT * D / 2), sr = kv4_ref(vsp, vn < kend, KT * NI);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      t.vw[g] = kv4_load<NI, NT>(vr, v_at + g * (8 * D));
      t.vs[g] = __builtin_amdgcn_raw_buffer_load_b32(sr, vs_at + g * (16 * NI), 0, 0);
    }
    vn += KT * NW;
    vp += KT * NW * (D / 2);
    vsp += KT * NW * NI;
  };
  Buf b0, b1;
  __builtin_amdgcn_sched_barrier(0);  // the queries' loads stay first: the loop waits for them with the first keys
  load_k(b0);
  __builtin_amdgcn_sched_barrier(0);
  load_v(b0);
  __builtin_amdgcn_sched_barrier(0);
  load_k(b1);
  __builtin_amdgcn_sched_barrier(0);
  load_v(b1);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < NI; ++i) qop[i] = __builtin_bit_cast(u16x8, __builtin_bit_cast(fp4_u4, qop[i]) ^ a.q_flip);

  float m_run = -INFINITY, l_run = 0.f;
  f32x4_t acc[ND];
#pragma unroll
  for (int T = 0; T < ND; ++T) acc[T] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  const int full = min(min(p0, plim) + 1, kend);  // keys below it are seen by every row of the block
  auto tile = [&](Buf& t, int k0) {
    const bool edge = k0 + KT > full;  // the tile is masked by column
    float sv[4 * NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      f32x4_t s = {0.f, 0.f, 0.f, 0.f};
      const float sc = __uint_as_float(__builtin_rotateleft32(t.ks[g], ks_rot));
#pragma unroll
      for (int i = 0; i < NI; ++i) s = mfma16x16x32<DT>(fp4_eight<DT>(t.kw[g].w[i], sc), qop[i], s);
#pragma unroll
      for (int r = 0; r < 4; ++r) sv[4 * g + r] = s[r];
    }
    __builtin_amdgcn_sched_barrier(0);
    load_k(t);
    __builtin_amdgcn_sched_barrier(0);
    if (edge) {
      const int lane = kv4_lane(), lg = lane >> 4;
      const int klim = min(kend - 1, Kv4Col(a, lane & 15, n, Gc, p0, plim).pq);
#pragma unroll
      for (int e = 0; e < 4 * NG; ++e)
        if (k0 + 16 * (e >> 2) + 4 * lg + (e & 3) > klim) sv[e] = -INFINITY;
    }
    float mx = sv[0];
#pragma unroll
    for (int e = 1; e < 4 * NG; ++e) mx = fmaxf(mx, sv[e]);
    mx = fmaxf(m_run, xor32_max(xor16_max(mx)));
    const float mu = mx == -INFINITY ? 0.f : mx;  // no key seen yet: every weight is exp2(-inf) = 0
    if (__ballot(mx > m_run)) {  // a column's maximum grew
      asm volatile("");  // keeps the products behind the branch
      const float alpha = __builtin_amdgcn_exp2f((m_run - mu) * a.scale_log2);
      l_run *= alpha;
#pragma unroll
      for (int T = 0; T < ND; ++T) acc[T] *= alpha;
    }
    m_run = mx;
    // A weight's exponent is the difference of the raw scores, which is exact near the maximum, times the factor: the
    // largest weight is one power of two whatever the scores' size. fp16 weights stand 2^15 higher (up to 32768), as do
    // their sums: below 2^-14 fp16 loses relative precision, and many keys of small weight would lose their part. bf16
    // weights stand 2^24 lower: the sum over 2^24 keys of the format's largest values, 6 x 2^125, is then finite, as their
    // mean is. It costs weights below 2^-102, which become 0, and values below it some of their digits.
    constexpr float up = DT == M3X_F16 ? 15.f : -24.f;
    fp4_u4 pop[NG / 2];
#pragma unroll
    for (int e = 0; e < 4 * NG; e += 2) {
      const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[e] - mu, a.scale_log2, up));
      const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[e + 1] - mu, a.scale_log2, up));
      pop[e / 8][e % 8 / 2] = fp4_pack<DT>(x, y);
      l_run = fp4_add2<DT>(pop[e / 8][e % 8 / 2], l_run);
    }
    // 0 * V is 0 only for finite V. Keys of an edge tile whose scale is past every written number's (stale bytes, or a
    // NaN that a later row of the block may see) stand apart: cleared here, added below to the columns that see them.
    uint32_t odd = 0;  // bit e: the lane's key e, in any of its groups
    if (edge) {
#pragma unroll
      for (int e = 0; e < 4 * NG; ++e) odd |= (t.vs[e / 4] >> (8 * (e & 3)) & 255u) > fp4_top_of<DT>() ? 1u << e : 0u;
      if (__ballot(odd != 0)) {
        odd |= __builtin_amdgcn_mov_dpp(odd, 0x128, 0xF, 0xF, false);  // row_ror 8, 4, 2, 1: over the lane's row of 16
        odd |= __builtin_amdgcn_mov_dpp(odd, 0x124, 0xF, 0xF, false);
        odd |= __builtin_amdgcn_mov_dpp(odd, 0x122, 0xF, 0xF, false);
        odd |= __builtin_amdgcn_mov_dpp(odd, 0x121, 0xF, 0xF, false);
#pragma unroll
        for (int e = 0; e < 4 * NG; ++e)
          if (odd >> e & 1u) {
            t.vs[e / 4] &= ~(255u << (8 * (e & 3)));  // the smallest scale, of zeros
            if constexpr (D == 128) t.vw[e / 4].w[e & 3] = 0;
            else t.vw[e / 4].w[(e & 3) >> 1] &= (e & 1) ? 0x0000FFFFu : 0xFFFF0000u;
          }
      }
    }
    kv4_pv<DT, D, NG>(t.vw, t.vs, pop, acc);
    if (edge) {
      if (__ballot(odd != 0)) {
        const int lane = kv4_lane(), li = lane & 15, lg = lane >> 4;
        const int klim = min(kend - 1, Kv4Col(a, li, n, Gc, p0, plim).pq);
        for (int q = 0; q < 4; ++q)
          for (uint32_t left = __builtin_amdgcn_readlane(odd, 16 * q); left; left &= left - 1) {
            const int at = __builtin_ctz(left), key = k0 + 16 * (at >> 2) + 4 * q + (at & 3);
            uint32_t mine = 0;
#pragma unroll
            for (int e = 0; e < 4 * NG; e += 2)
              if (e == (at & ~1)) mine = pop[e / 8][e % 8 / 2];
            const int pair = __builtin_amdgcn_ds_bpermute(4 * (16 * q + li), (int)mine);
            const float p = E<DT>::to_f((uint16_t)(pair >> (16 * (at & 1))));
            if (key > klim) continue;
            const uint8_t* wp = c.v + ((base + key) >> 2) * (2 * D) + (key & 3) * NI;
            const uint8_t* sp = c.vs + ((base + key) >> 2) * (4 * NI) + (key & 3);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int ch = 4 * lg + r;
              const float s1 = fp4_scale(sp[4 * (ch * ND >> 5)]);
              uint32_t w;
              if constexpr (D == 128) w = *reinterpret_cast<const uint32_t*>(wp + ch * (4 * NI));
              else w = *reinterpret_cast<const uint16_t*>(wp + ch * (4 * NI));
              const u16x8 x = fp4_eight<DT>(w, s1);
#pragma unroll
              for (int T = 0; T < ND; ++T) acc[T][r] += p * E<DT>::to_f(x.v[T]);
            }
          }
        // all loads of this path have arrived (vmcnt 0), so that behind it the tiles' own are counted as on the other
        __builtin_amdgcn_s_waitcnt(0x0F70);
      }
    }
    load_v(t);
    __builtin_amdgcn_sched_barrier(0);
  };
  for (; k0 + KT * NW < kend; k0 += 2 * KT * NW) {
    tile(b0, k0);
    tile(b1, k0 + KT * NW);
  }
  if (k0 < kend) tile(b0, k0);
  l_run = xor32_sum(xor16_sum(l_run));

  // merge the waves: lane (column, lg) holds dims ND (4 lg + r) + T
  const int tid = 64 * wave + kv4_lane();
  {
    const int li = tid & 15, lg = tid >> 4 & 3;
    if (Kv4Col(a, li, n, Gc, p0, plim).live) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int T = 0; T < ND; T += 4) {
          const f32x4_t x = {acc[T][r], acc[T + 1][r], acc[T + 2][r], acc[T + 3][r]};
          *reinterpret_cast<f32x4_t*>(&lds.o[wave][li][ND * (4 * lg + r) + T]) = x;
        }
    }
    if (lg == 0) {
      lds.m[wave][li] = m_run;
      lds.l[wave][li] = l_run;
    }
  }
  __syncthreads();
  for (int i = tid; i < n * Gc * (D / 4); i += 64 * NW) {
    const int col = i / (D / 4), d = (i % (D / 4)) * 4;
    const int j = col * a.over_Gc >> 8, h = col - j * min(a.G, 16);
    const int pj = min(p0 + j, plim);
    if (kstart > pj) continue;  // the row has no keys in this split
    float M = lds.m[0][col];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = fmaxf(M, lds.m[w][col]);
    const float mu = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    f32x4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f((lds.m[w][col] - mu) * a.scale_log2);
      L += lds.l[w][col] * f;
      O += *reinterpret_cast<const f32x4_t*>(&lds.o[w][col][d]) * f;
    }
    const long rh = (long)(row + j) * a.heads + kh * a.G + h0 + h;
    if (pj < a.chunk) {
      kv4_store_out<DT>(a.out + (long)(row + j) * a.so_b + (long)(kh * a.G + h0 + h) * a.so_h + d, O, L);
    } else {
      const long at = rh * a.max_splits + split;
      *reinterpret_cast<f32x4_t*>(a.part + at * D + d) = O;
      if (d == 0) {
        float* ml = a.part + (long)a.rows * a.heads * a.max_splits * D + at * 2;
        ml[0] = M;
        ml[1] = L;
      }
    }
  }
  __syncthreads();  // the next block's sums take the same place
}

template <int DT, int D, int NW>
__global__ __launch_bounds__(64 * NW, KV4_OCC) void kv4_attn_kernel(Kv4 c, Kv4Attn a) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  int kh = blockIdx.y, h0 = 0;  // h0: first query head of the block within the kv head's G
  if (a.hblocks > 1) {
    kh = blockIdx.y / a.hblocks;
    h0 = (blockIdx.y - kh * a.hblocks) * 16;
  }
  const int Gc = min(a.G - h0, 16);
  __shared__ Kv4Lds<D, NW> lds;

  // The workgroup's candidates: R rows of an aligned group of qb. All first parts of groups, over the heads and the
  // splits, come before all second ones in launch order: a prompt's live workgroups, which its groups' first parts are,
  // spread over the XCDs and do not stand behind those that leave at once (heads 16/8 of 128, against a group's parts next
  // to each other: 512 rows of a prompt over 4000 keys 39 us, 111; 64 rows over 500 6.7, 9.3).
  int part = 0, split = blockIdx.z;
  for (; split >= a.max_splits; split -= a.max_splits) ++part;
  const int first = blockIdx.x * a.qb;
  const int ri = first - 1 + lane;
  const int rc = min(max(ri, 0), a.rows - 1);
  const long slot_i = a.slots[rc];
  const int pos_i = a.pos[rc];
  // the exchanges stand before the conditions: a lane that a condition leaves out gives its neighbour no value
  const long slot_b = __shfl_up(slot_i, 1, 64);
  const int pos_b = __shfl_up(pos_i, 1, 64);
  const bool follows = lane > 1 && lane <= a.qb && ri < a.rows && slot_b == slot_i && pos_i > 0 && pos_b == pos_i - 1;
  const uint64_t chain = __ballot(follows);  // bit i: row first - 1 + i continues the row before it
  lds.slot[lane] = slot_i;  // every wave writes the same, and reads behind its own writes
  lds.pos[lane] = pos_i;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const int last = min(min((part + 1) * a.R, a.qb), a.rows - first);
  for (int cand = part * a.R; cand < last; ++cand) {
    if (chain >> (cand + 1) & 1u) continue;  // in the block of a row before it
    const long slot = lds.slot[cand + 1];
    const int n = 1 + __builtin_ctzll(~(chain >> (cand + 2)));
    const long slot_u = (long)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)slot) |
                               (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(slot >> 32)) << 32);
    const int p0 = __builtin_amdgcn_readfirstlane(lds.pos[cand + 1]);
    // A single row's keys are a stream of their own (non-temporal loads: 224 rows of 2048 keys 80 us, 92 without); a
    // prompt's are read by its next blocks as well (16 x 512 rows over 512 keys: 68 us, 78 with).
    if (n > 1) kv4_attn_row<DT, D, NW, false>(c, a, first + cand, n, slot_u, p0, kh, h0, Gc, split, wave, lds);
    else kv4_attn_row<DT, D, NW, true>(c, a, first + cand, 1, slot_u, p0, kh, h0, Gc, split, wave, lds);
  }
}

// Joins the splits of a row's keys: NG groups of D / 4 threads a (row, head), each every NG-th split in order, then the
// groups in order (the same order whatever the launch). Bound by the launch and two memory round trips; the first
// splits are loaded beside the row's position, before it is known which of them there are. One row's 16 splits: 3.4 us.
template <int DT, int D, int NG>
__global__ __launch_bounds__(256) void kv4_combine_kernel(Kv4 c, Kv4Attn a) {
  constexpr int TD = D / 4, HB = 256 / (TD * NG), U = 4;
  const int row = blockIdx.x;
  const int g = threadIdx.x / TD % NG, d = (threadIdx.x % TD) * 4, hb = threadIdx.x / (TD * NG);
  const int head = min((int)(blockIdx.y * HB + hb), a.heads - 1);  // a group past the last head repeats it
  const long slot = a.slots[row];
  const int pos = a.pos[row];
  const long at = ((long)row * a.heads + head) * a.max_splits;
  const float* ml = a.part + (long)a.rows * a.heads * a.max_splits * D + at * 2;
  const float* po = a.part + at * D;
  float2 x[U];
  f32x4_t o[U];
  auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int s = min(s0 + i * NG, a.max_splits - 1);
      x[i] = *reinterpret_cast<const float2*>(ml + 2 * s);
      o[i] = *reinterpret_cast<const f32x4_t*>(po + (long)s * D + d);
    }
  };
  load(g);
  const int p = min(pos, min(c.cap, a.max_ctx) - 1);
  if (slot < 0 || slot >= c.slots || p < a.chunk) return;  // no key, or one split: the attention wrote the row
  const int ns = p / a.chunk + 1;
  float M = -INFINITY, L = 0.f;
  f32x4_t O = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = g; s0 < ns; s0 += U * NG) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (s0 + i * NG < ns) {
        const float mx = fmaxf(M, x[i].x), mu = mx == -INFINITY ? 0.f : mx;
        const float f0 = __builtin_amdgcn_exp2f((M - mu) * a.scale_log2);
        const float f1 = __builtin_amdgcn_exp2f((x[i].x - mu) * a.scale_log2);
        L = L * f0 + x[i].y * f1;
        O = O * f0 + o[i] * f1;
        M = mx;
      }
    }
    if (s0 + U * NG < ns) load(s0 + U * NG);
  }
  __shared__ __align__(16) float so[HB][NG][D];
  __shared__ float sm[HB][NG], sl[HB][NG];
  *reinterpret_cast<f32x4_t*>(&so[hb][g][d]) = O;
  if (d == 0) {
    sm[hb][g] = M;
    sl[hb][g] = L;
  }
  __syncthreads();
  if (g || blockIdx.y * HB + hb >= a.heads) return;
  M = sm[hb][0];
#pragma unroll
  for (int i = 1; i < NG; ++i) M = fmaxf(M, sm[hb][i]);
  const float mu = M == -INFINITY ? 0.f : M;
  L = 0.f;
  O = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const float f = __builtin_amdgcn_exp2f((sm[hb][i] - mu) * a.scale_log2);
    L += sl[hb][i] * f;
    O += *reinterpret_cast<const f32x4_t*>(&so[hb][i][d]) * f;
  }
  kv4_store_out<DT>(a.out + (long)row * a.so_b + (long)head * a.so_h + d, O, L);
}

// ---------------------------------------------------------------------------------------------------------
namespace {
// the kernels' view of a caller's cache, or a status
int kv4_take(const M3xKv4* p, Kv4& c) {
  if (!p) return M3X_ENULL;
  if (p->slots <= 0 || p->kv_heads <= 0 || p->cap <= 0) return M3X_EINVAL;
  if (p->cap > 1 << 30) return M3X_EINVAL;  // attention counts past the last key in 32 bits
  if (!p->k || !p->ks || !p->v || !p->vs) return M3X_ENULL;
  if (p->head_dim != 64 && p->head_dim != 128) return M3X_EUNSUPPORTED;
  if (p->cap % 32 || !m3x_aligned16(p->k) || !m3x_aligned16(p->v) || !m3x_aligned16(p->ks) || !m3x_aligned16(p->vs))
    return M3X_EINVAL;
  c = Kv4{(uint8_t*)p->k, (uint8_t*)p->ks, (uint8_t*)p->v, (uint8_t*)p->vs, p->slots, p->kv_heads, p->cap};
  return M3X_OK;
}
// whether D / 8 threads for each of `items` fit a launch (fewer than 2^32 threads)
bool kv4_fits(long items, int head_dim) { return items * (head_dim / 8) < (1L << 32) - 256; }
}  // namespace

#define KV4_DISPATCH(KERNEL, GRID, ...)                                                                          \
  do {                                                                                                           \
    if (dtype == M3X_BF16 && head_dim == 128)                                                                    \
      hipLaunchKernelGGL((KERNEL<M3X_BF16, 128>), GRID, dim3(256), 0, (hipStream_t)stream, __VA_ARGS__);         \
    else if (dtype == M3X_BF16)                                                                                  \
      hipLaunchKernelGGL((KERNEL<M3X_BF16, 64>), GRID, dim3(256), 0, (hipStream_t)stream, __VA_ARGS__);          \
    else if (head_dim == 128)                                                                                    \
      hipLaunchKernelGGL((KERNEL<M3X_F16, 128>), GRID, dim3(256), 0, (hipStream_t)stream, __VA_ARGS__);          \
    else                                                                                                         \
      hipLaunchKernelGGL((KERNEL<M3X_F16, 64>), GRID, dim3(256), 0, (hipStream_t)stream, __VA_ARGS__);           \
  } while (0)

M3X_API int m3x_kv4_append(const M3xKv4* cache, const void* k, long sk_r, long sk_h, const void* v, long sv_r, long sv_h,
                           const int64_t* slots, const int32_t* pos, int rows, int dtype, void* stream) {
  Kv4 c;
  if (const int st = kv4_take(cache, c)) return st;
  if (rows < 0) return M3X_EINVAL;
  if (dtype != M3X_BF16 && dtype != M3X_F16) return M3X_EUNSUPPORTED;
  if (rows == 0) return M3X_OK;
  if (!k || !v || !slots || !pos) return M3X_ENULL;
  if (((sk_r | sk_h | sv_r | sv_h) & 7) || !m3x_aligned16(k) || !m3x_aligned16(v)) return M3X_EINVAL;
  const int head_dim = cache->head_dim;
  const long items = (long)rows * c.kv_heads;
  if (!kv4_fits(items, head_dim)) return M3X_EINVAL;
  KV4_DISPATCH(kv4_append_kernel, dim3(m3x_ceil_div(items, 2048 / head_dim)), (const uint16_t*)k, sk_r, sk_h,
               (const uint16_t*)v, sv_r, sv_h, c, slots, pos, rows);
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}

M3X_API int m3x_qk_norm_rope_kv4(const M3xKv4* cache, const void* qkv, long s_qkv, void* q_out, long s_qo_b, long s_qo_h,
                                 const int64_t* slots, const int32_t* pos, const void* cos, const void* sin, long s_cos,
                                 const void* wq, const void* wk, float eps, int rows, int heads, void* stream) {
  Kv4 c;
  if (const int st = kv4_take(cache, c)) return st;
  if (rows < 0 || heads <= 0) return M3X_EINVAL;
  if (rows == 0) return M3X_OK;
  if (!qkv || !q_out || !slots || !pos || !cos || !sin || !wq || !wk) return M3X_ENULL;
  if ((s_qkv | s_qo_b | s_qo_h | s_cos) & 7) return M3X_EINVAL;
  if (!m3x_aligned16(qkv) || !m3x_aligned16(q_out) || !m3x_aligned16(cos) || !m3x_aligned16(sin) ||
      !m3x_aligned16(wq) || !m3x_aligned16(wk))
    return M3X_EINVAL;
  const int head_dim = cache->head_dim;
  const long items = (long)rows * ((long)heads + c.kv_heads);
  if (!kv4_fits(items, head_dim)) return M3X_EINVAL;
  const dim3 grid(m3x_ceil_div(items, 2048 / head_dim));
#define KV4_QKN(DD)                                                                                               \
  hipLaunchKernelGGL((qk_norm_rope_kv4_kernel<DD>), grid, dim3(256), 0, (hipStream_t)stream, (const uint16_t*)qkv, \
                     s_qkv, (uint16_t*)q_out, s_qo_b, s_qo_h, c, slots, pos, (const uint16_t*)cos,                 \
                     (const uint16_t*)sin, s_cos, (const uint16_t*)wq, (const uint16_t*)wk, eps, rows, heads)
  if (head_dim == 128) KV4_QKN(128);
  else KV4_QKN(64);
#undef KV4_QKN
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}

M3X_API int m3x_kv4_read(const M3xKv4* cache, const int64_t* slots, const int32_t* pos, void* k, long sk_r, long sk_h,
                         void* v, long sv_r, long sv_h, int rows, int dtype, void* stream) {
  Kv4 c;
  if (const int st = kv4_take(cache, c)) return st;
  if (rows < 0) return M3X_EINVAL;
  if (dtype != M3X_BF16 && dtype != M3X_F16) return M3X_EUNSUPPORTED;
  if (rows == 0) return M3X_OK;
  if (!k || !v || !slots || !pos) return M3X_ENULL;
  if (((sk_r | sk_h | sv_r | sv_h) & 7) || !m3x_aligned16(k) || !m3x_aligned16(v)) return M3X_EINVAL;
  const int head_dim = cache->head_dim;
  const long items = (long)rows * c.kv_heads;
  if (!kv4_fits(items, head_dim)) return M3X_EINVAL;
  KV4_DISPATCH(kv4_read_kernel, dim3(m3x_ceil_div(items, 2048 / head_dim)), c, slots, pos, (uint16_t*)k, sk_r, sk_h,
               (uint16_t*)v, sv_r, sv_h, rows);
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}

M3X_API size_t m3x_kv4_attn_workspace(int rows, int heads, int head_dim, int max_ctx, int chunk) {
  if (rows <= 0 || heads <= 0 || head_dim <= 0 || max_ctx <= 0 || chunk <= 0) return 0;
  const size_t splits = ((size_t)max_ctx + chunk - 1) / chunk;
  return splits > 1 ? (size_t)rows * heads * splits * (head_dim + 2) * sizeof(float) : 0;
}

namespace {
template <int DT, int D> void kv4_launch(const Kv4& c, const Kv4Attn& a, hipStream_t st) {
  const int parts = m3x_ceil_div(std::min(a.qb, a.rows), a.R);
  const dim3 grid(m3x_ceil_div(a.rows, a.qb), c.kv_heads * a.hblocks, a.max_splits * parts);
  hipLaunchKernelGGL((kv4_attn_kernel<DT, D, KV4_NW>), grid, dim3(64 * KV4_NW), 0, st, c, a);
  if (a.max_splits > 4)
    hipLaunchKernelGGL((kv4_combine_kernel<DT, D, 8>), dim3(a.rows, m3x_ceil_div(a.heads, 128 / D)), dim3(256), 0, st, c, a);
  else if (a.max_splits > 1)
    hipLaunchKernelGGL((kv4_combine_kernel<DT, D, 1>), dim3(a.rows, m3x_ceil_div(a.heads, 1024 / D)), dim3(256), 0, st, c, a);
}
}  // namespace

M3X_API int m3x_kv4_attn(const M3xKv4* cache, const void* q, long sq_b, long sq_h, void* out, long so_b, long so_h,
                         const int64_t* slots, const int32_t* pos, float scale, int rows, int heads, int max_ctx,
                         int chunk, void* workspace, size_t ws_bytes, int dtype, void* stream) {
  Kv4 c;
  if (const int st = kv4_take(cache, c)) return st;
  if (rows < 0 || heads <= 0 || max_ctx <= 0) return M3X_EINVAL;
  if (dtype != M3X_BF16 && dtype != M3X_F16) return M3X_EUNSUPPORTED;
  if (heads % c.kv_heads) return M3X_EUNSUPPORTED;
  if (chunk <= 0 || chunk % 128 || max_ctx > c.cap) return M3X_EINVAL;
  if (!(fabsf(scale) <= 0x1p127f)) return M3X_EINVAL;  // its factor would not be finite; NaN
  if (rows == 0) return M3X_OK;
  if (!q || !out || !slots || !pos) return M3X_ENULL;
  if (((sq_b | sq_h | so_b | so_h) & 7) || !m3x_aligned16(q) || !m3x_aligned16(out)) return M3X_EINVAL;
  const int splits = m3x_ceil_div(max_ctx, chunk);
  const int G = heads / c.kv_heads, hb = m3x_ceil_div(G, 16);
  if (rows > (1 << 20) || (long)c.kv_heads * hb > 65535 || heads > 65535 || splits > 4095) return M3X_EINVAL;
  const int head_dim = cache->head_dim;
  if (splits > 1) {
    if (!workspace) return M3X_ENULL;
    if (ws_bytes < m3x_kv4_attn_workspace(rows, heads, head_dim, max_ctx, chunk)) return M3X_EWORKSPACE;
    if (!m3x_aligned16(workspace)) return M3X_EINVAL;
  }
  const int Gc = std::min(G, 16), qb = hb > 1 ? 1 : 16 / G;
  // R candidate rows a workgroup: fewer workgroups that leave at once, as long as 4096 are left for rows that are no
  // prompt's and differ in length. Measured (us; 4096, 12288, R = 1): prompts of 64 rows x 64 seqs, 8/8 heads 15, 18, 38;
  // 8 x 200 rows over 500 keys, 16/8 heads 21, 21, 25; 512 single rows over up to 1000 keys 58, 54, 55 (2048: 63); 400 over
  // up to 2000 77, 76, 76 (2048: 81, 1024: 96).
  int R = 1;
  while (R < qb && (long)rows * c.kv_heads * hb * splits >= 4096L * R) R *= 2;
  R = R < qb ? R : qb;
  // The raw scores' differences are multiplied by |scale| log2(e): not by a negative factor (the running maximum is the raw
  // scores') and not by 0 (0 * -inf of a masked key). fp32's smallest number stands for 0: no difference of finite scores
  // makes more than 2^-20 of it. A factor below the normal numbers is made from its bits, whether or not the caller's thread
  // flushes them to 0; what its few bits round away is no more than that either.
  const double factor = fabs((double)scale) * 1.44269504088896341;
  float weight = (float)factor;
  if (factor < 0x1p-126) {
    const uint32_t bits = std::max(1u, (uint32_t)(factor * 0x1p149));
    memcpy(&weight, &bits, sizeof weight);
  }
  const Kv4Attn a = {(const uint16_t*)q, sq_b, sq_h, (uint16_t*)out, so_b, so_h, slots, pos,
                     weight, scale < 0.f ? 0x80008000u : 0u, rows, heads, G, hb, qb, R, chunk, max_ctx, splits,
                     (uint32_t)((256 + Gc - 1) / Gc), (float*)workspace};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == M3X_BF16 && head_dim == 128) kv4_launch<M3X_BF16, 128>(c, a, st);
  else if (dtype == M3X_BF16) kv4_launch<M3X_BF16, 64>(c, a, st);
  else if (head_dim == 128) kv4_launch<M3X_F16, 128>(c, a, st);
  else kv4_launch<M3X_F16, 64>(c, a, st);
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}
