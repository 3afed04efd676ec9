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
#include "m3x_norm.h"
#include "m3x_fp4.h"

namespace {
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

// K and V rows into the cache, D / 8 threads per (row, kv head). Bound: the rows' 16-bit bytes at large counts, the
// launch at few.
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

// qk_norm_rope_cache_kernel's arithmetic and bits with the keys and values quantised into the 4-bit cache
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

// positions of the cache as 16-bit rows (zeros for a row outside it)
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
  st16(k + row * sk_r + kh * sk_h + 8 * t, kx);
  st16(v + row * sv_r + kh * sv_h + 8 * t, vx);
}

// ---------------------------------------------------------------------------------------------------------
// Attention over the cache: out[r, h, :] = softmax(scale q[r, h] . K^T) V over positions 0 .. pos[r] of slot slots[r].
//
// A workgroup takes one (block of rows, kv head, split of the keys). The score product has the keys as its rows and
// 16 columns: the G query heads of up to 16 / G rows that stand next to each other in the call, of one slot at
// consecutive positions (a prompt's), found from slots and pos by the workgroup itself; the block's later rows' own
// workgroups leave at once. A single token is a block of one row. Each of the 4 waves takes every 4th 32-key tile:
//   S^T = K . Q^T   per 16 keys D / 32 MFMA 16x16x32: a lane's words of K become 16-bit operands in registers
//   softmax         running maximum and sum in fp32, exp2; a lane keeps its own column's, its keys' partial sum
//   O^T += V^T . P  D / 16 MFMA per 32 keys: S^T's accumulator is the P operand as it stands, and V's words, which
//                   hold two dims of a key each, are paired over keys by byte permutes
// P is rounded to the 16-bit type (at most half a step, relative 2^-8 bf16 / 2^-11 fp16, per key); everything else
// between the loads and the output is exact or fp32.
namespace {
template <int NI> struct Words { uint32_t w[NI]; };
template <int NI> __device__ __forceinline__ Words<NI> kv4_load(const uint8_t* p) {
  Words<NI> r;
  if constexpr (NI == 4) {
    const fp4_u4 x = __builtin_nontemporal_load(reinterpret_cast<const fp4_u4*>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = x[i];
  } else {
    const fp4_u2 x = __builtin_nontemporal_load(reinterpret_cast<const fp4_u2*>(p));
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
  float scale_log2;
  int rows, heads, G, hblocks, chunk, max_ctx, max_splits;
  float* part;  // [rows * heads][max_splits][D] then [rows * heads][max_splits][2] (maximum, sum)
};

// the A operand of dim tile T: element e is the number of dim T of the lane's chunk at key e
template <int DT, int D, int T>
__device__ __forceinline__ void kv4_vop(const Words<D / 32> (&v)[2], const float (&sc)[8], u16x8& lo, u16x8& hi) {
  uint32_t a[8];
#define KV4_PAIR(E)                                                                                             \
  if constexpr (D == 128) a[E] = fp4_pair<DT, T>(v[E / 4].w[E & 3], sc[E]);                                    \
  else a[E] = fp4_pair<DT, 2 * (E & 1) + T>(v[E / 4].w[(E & 3) >> 1], sc[E]);
  KV4_PAIR(0) KV4_PAIR(1) KV4_PAIR(2) KV4_PAIR(3) KV4_PAIR(4) KV4_PAIR(5) KV4_PAIR(6) KV4_PAIR(7)
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

template <int DT, int D, int B = 0>
__device__ __forceinline__ void kv4_pv(const Words<D / 32> (&v)[2], const float (&sc)[8], const u16x8& pop,
                                       f32x4_t (&acc)[D / 16]) {
  u16x8 lo, hi;
  kv4_vop<DT, D, B>(v, sc, lo, hi);
  acc[2 * B] = mfma16x16x32<DT>(lo, pop, acc[2 * B]);
  acc[2 * B + 1] = mfma16x16x32<DT>(hi, pop, acc[2 * B + 1]);
  if constexpr (B + 1 < D / 32) kv4_pv<DT, D, B + 1>(v, sc, pop, acc);
}

// the same where a key that a row of the block does not see may be no number: for each row in turn the keys past its
// limit (lim0 + j, at most lim; key0 = the lane's first key) are cleared, and its columns take the result
template <int DT, int D, int B = 0>
__device__ __forceinline__ void kv4_pv_rows(const Words<D / 32> (&v)[2], const float (&sc)[8], const u16x8& pop,
                                            f32x4_t (&acc)[D / 16], int n, int jq, int key0, int lim0, int lim) {
  u16x8 lo, hi;
  kv4_vop<DT, D, B>(v, sc, lo, hi);
  for (int j = 0; j < n; ++j) {
    const int klim = min(lim, lim0 + j);
    u16x8 l, h;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const bool off = key0 + 16 * (e >> 2) + (e & 3) > klim;
      l.v[e] = off ? 0 : lo.v[e];
      h.v[e] = off ? 0 : hi.v[e];
    }
    const f32x4_t x = mfma16x16x32<DT>(l, pop, acc[2 * B]), y = mfma16x16x32<DT>(h, pop, acc[2 * B + 1]);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      acc[2 * B][r] = jq == j ? x[r] : acc[2 * B][r];
      acc[2 * B + 1][r] = jq == j ? y[r] : acc[2 * B + 1][r];
    }
  }
  if constexpr (B + 1 < D / 32) kv4_pv_rows<DT, D, B + 1>(v, sc, pop, acc, n, jq, key0, lim0, lim);
}
}  // namespace

template <int DT, int D>
__global__ __launch_bounds__(256, 3) void kv4_attn_kernel(Kv4 c, Kv4Attn a) {
  constexpr int NI = D / 32;   // words a lane holds of 16 keys; score steps
  constexpr int ND = D / 16;   // dim tiles
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int li = lane & 15, lg = lane >> 4;
  const int row = blockIdx.x;
  const int kh = blockIdx.y / a.hblocks;
  const int h0 = (blockIdx.y % a.hblocks) * 16;  // first query head of the block within the kv head's G
  const int Gc = min(a.G - h0, 16);
  const int split = blockIdx.z;

  // the block: rows row .. row + n - 1
  const int qb = a.hblocks > 1 ? 1 : 16 / Gc;
  const int ri = row - 1 + lane;
  const int rc = min(max(ri, 0), a.rows - 1);
  const long slot_i = a.slots[rc];
  const int pos_i = a.pos[rc];
  // the exchanges stand before the conditions: a lane that a condition leaves out gives its neighbour no value
  const long slot_b = __shfl_up(slot_i, 1, 64);
  const int pos_b = __shfl_up(pos_i, 1, 64);
  const bool follows = lane > 0 && lane <= qb && ri < a.rows && ri % qb != 0 && slot_b == slot_i && pos_i > 0 &&
                       pos_b == pos_i - 1;
  const uint64_t chain = __ballot(follows);  // bit i: row - 1 + i continues the row before it
  if (chain & 2u) return;
  const int n = 1 + __builtin_ctzll(~(chain >> 2));
  const long slot = __shfl(slot_i, 1, 64);
  const int p0 = __builtin_amdgcn_readfirstlane(__shfl(pos_i, 1, 64));
  const int plim = min(c.cap, a.max_ctx) - 1;  // the host keeps pos below both; every access stays inside whatever pos holds
  const bool inside = __builtin_amdgcn_readfirstlane(slot >= 0 && slot < c.slots && p0 >= 0);
  if (!inside) {  // no key: zeros
    if (split == 0)
      for (int j = 0; j < n; ++j)
        for (int i = threadIdx.x; i < Gc * D; i += 256)
          a.out[(long)(row + j) * a.so_b + (long)(kh * a.G + h0 + i / D) * a.so_h + i % D] = 0;
    return;
  }
  const int plast = min(p0 + n - 1, plim);
  const int kstart = split * a.chunk;
  if (kstart > plast) return;
  const int kend = min(kstart + a.chunk, plast + 1);

  const int jq = li / Gc;  // the column's row within the block
  const int hq = li - jq * Gc;
  const bool live = jq < n;
  const int pq = live ? min(p0 + jq, plim) : -1;  // the column sees keys <= pq
  u16x8 qop[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    if (live) {
      qop[i] = ld16(a.q + (long)(row + jq) * a.sq_b + (long)(kh * a.G + h0 + hq) * a.sq_h + (D / 4) * lg + 8 * i);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) qop[i].v[e] = 0;
    }
  }

  const long base = (slot * c.kv_heads + kh) * (long)c.cap;
  const uint8_t* kb = c.k + base * (D / 2) + li * (D / 2) + lg * (D / 8);
  const uint8_t* ksb = c.ks + base * NI + li * NI + (D == 128 ? lg : lg >> 1);
  const uint8_t* vb = c.v + base * (D / 2) + lg * (2 * D) + li * (D / 8);
  const uint8_t* vsb = c.vs + base * NI + lg * (4 * NI) + (D == 128 ? li >> 2 : li >> 3) * 4;
  Words<NI> kw[2], vw[2];
  uint32_t ks[2], vs[2];
  auto load_k = [&](int k0) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      kw[g] = kv4_load<NI>(kb + (long)(k0 + 16 * g) * (D / 2));
      ks[g] = ksb[(long)(k0 + 16 * g) * NI];
    }
  };
  auto load_v = [&](int k0) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      vw[g] = kv4_load<NI>(vb + (long)(k0 + 16 * g) * (D / 2));
      vs[g] = *reinterpret_cast<const uint32_t*>(vsb + (long)(k0 + 16 * g) * NI);
    }
  };

  float m_run = -INFINITY, l_run = 0.f;
  f32x4_t acc[ND];
#pragma unroll
  for (int T = 0; T < ND; ++T) acc[T] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  // a tile's keys are loaded while the tile before is weighted, its values while its keys are multiplied
  // (cap % 32 == 0: a tile that begins inside the slot ends inside it)
  int k0 = kstart + 32 * wave;
  if (k0 < kend) {
    load_k(k0);
    load_v(k0);
  }
  for (; k0 < kend; k0 += 128) {
    float sv[8];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      f32x4_t s = {0.f, 0.f, 0.f, 0.f};
      const float sc = fp4_scale(ks[g]);
#pragma unroll
      for (int i = 0; i < NI; ++i) s = mfma16x16x32<DT>(fp4_eight<DT>(kw[g].w[i], sc), qop[i], s);
#pragma unroll
      for (int r = 0; r < 4; ++r) sv[4 * g + r] = s[r] * a.scale_log2;
    }
    const bool more = k0 + 128 < kend;
    if (more) load_k(k0 + 128);
    // the tile reaches past what the block's first row sees: mask by column
    const bool edge = k0 + 31 > min(p0, plim);
    if (edge) {
      const int klim = min(kend - 1, pq);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k0 + 16 * (e >> 2) + 4 * lg + (e & 3) > klim) sv[e] = -INFINITY;
    }
    float mx = sv[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, sv[e]);
    mx = fmaxf(m_run, xor32_max(xor16_max(mx)));
    const float mu = mx == -INFINITY ? 0.f : mx;  // no key seen yet: every weight is exp2(-inf) = 0
    const float alpha = __builtin_amdgcn_exp2f(m_run - mu);
    m_run = mx;
    // fp16 weights stand 2^15 higher (up to 32768), as do their sums: below 2^-14 fp16 loses relative precision, and
    // many keys of small weight would lose their part
    const float mp = mu - (DT == M3X_F16 ? 15.f : 0.f);
    u16x8 pop;
    float ps = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float p = __builtin_amdgcn_exp2f(sv[e] - mp);
      ps += p;
      pop.v[e] = E<DT>::from_f(p);
    }
    l_run = l_run * alpha + ps;
#pragma unroll
    for (int T = 0; T < ND; ++T) acc[T] *= alpha;
    float sc[8];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      sc[4 * g] = fp4_scale_of<0>(vs[g]);
      sc[4 * g + 1] = fp4_scale_of<1>(vs[g]);
      sc[4 * g + 2] = fp4_scale_of<2>(vs[g]);
      sc[4 * g + 3] = fp4_scale_of<3>(vs[g]);
    }
    // 0 * V is 0 only for finite V: where a masked key may hold anything (stale or a later row's NaN), each row of the
    // block takes the product with the keys it does not see cleared
    bool bad = false;
    if (edge) {
      bool b = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) b |= sc[e] > fp4_scale(fp4_top_of<DT>());
      bad = __ballot(b) != 0;
    }
    if (!bad) kv4_pv<DT, D>(vw, sc, pop, acc);
    else kv4_pv_rows<DT, D>(vw, sc, pop, acc, n, jq, k0 + 4 * lg, p0, kend - 1);
    if (more) load_v(k0 + 128);
  }
  l_run = xor32_sum(xor16_sum(l_run));

  // merge the waves: lane (column, lg) holds dims ND (4 lg + r) + T
  __shared__ __align__(16) float lo[4][16][D + 4];
  __shared__ float lm[4][16], ll[4][16];
  if (live) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int T = 0; T < ND; T += 4) {
        const f32x4_t x = {acc[T][r], acc[T + 1][r], acc[T + 2][r], acc[T + 3][r]};
        *reinterpret_cast<f32x4_t*>(&lo[wave][li][ND * (4 * lg + r) + T]) = x;
      }
  }
  if (lg == 0) {
    lm[wave][li] = m_run;
    ll[wave][li] = l_run;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * Gc * (D / 4); i += 256) {
    const int col = i / (D / 4), d = (i % (D / 4)) * 4;
    const int j = col / Gc, h = col - j * Gc;
    const int pj = min(p0 + j, plim);
    if (kstart > pj) continue;  // the row has no keys in this split
    float M = fmaxf(fmaxf(lm[0][col], lm[1][col]), fmaxf(lm[2][col], lm[3][col]));
    const float mu = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    f32x4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(lm[w][col] - mu);
      L += ll[w][col] * f;
      O += *reinterpret_cast<const f32x4_t*>(&lo[w][col][d]) * f;
    }
    const long rh = (long)(row + j) * a.heads + kh * a.G + h0 + h;
    if (pj < a.chunk) {
      uint32_t o[2];
      o[0] = E<DT>::from_f(O[0] / L) | (uint32_t)E<DT>::from_f(O[1] / L) << 16;
      o[1] = E<DT>::from_f(O[2] / L) | (uint32_t)E<DT>::from_f(O[3] / L) << 16;
      *reinterpret_cast<uint2*>(a.out + (long)(row + j) * a.so_b + (long)(kh * a.G + h0 + h) * a.so_h + d) =
          make_uint2(o[0], o[1]);
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
}

// Joins the splits of a row's keys, in order within each of 1024 / D groups of splits, then the groups in order. One
// workgroup per (row, head).
template <int DT, int D>
__global__ __launch_bounds__(256) void kv4_combine_kernel(Kv4 c, Kv4Attn a) {
  constexpr int TD = D / 4, NG = 256 / TD;
  const int row = blockIdx.x, head = blockIdx.y;
  const long slot = a.slots[row];
  const int p = min(a.pos[row], min(c.cap, a.max_ctx) - 1);
  if (slot < 0 || slot >= c.slots || p < a.chunk) return;  // no key, or one split: the attention wrote the row
  const int ns = p / a.chunk + 1;
  const long at = ((long)row * a.heads + head) * a.max_splits;
  const float* ml = a.part + (long)a.rows * a.heads * a.max_splits * D + at * 2;
  const float* po = a.part + at * D;
  const int g = threadIdx.x / TD, d = (threadIdx.x % TD) * 4;
  float M = -INFINITY, L = 0.f;
  f32x4_t O = {0.f, 0.f, 0.f, 0.f};
  for (int s = g; s < ns; s += NG) {
    const float m = ml[2 * s], l = ml[2 * s + 1];
    const f32x4_t o = *reinterpret_cast<const f32x4_t*>(po + (long)s * D + d);
    const float mx = fmaxf(M, m), mu = mx == -INFINITY ? 0.f : mx;
    const float f0 = __builtin_amdgcn_exp2f(M - mu), f1 = __builtin_amdgcn_exp2f(m - mu);
    L = L * f0 + l * f1;
    O = O * f0 + o * f1;
    M = mx;
  }
  __shared__ __align__(16) float so[NG][D];
  __shared__ float sm[NG], sl[NG];
  *reinterpret_cast<f32x4_t*>(&so[g][d]) = O;
  if (d == 0) {
    sm[g] = M;
    sl[g] = L;
  }
  __syncthreads();
  if (threadIdx.x >= TD) return;
  M = sm[0];
#pragma unroll
  for (int i = 1; i < NG; ++i) M = fmaxf(M, sm[i]);
  const float mu = M == -INFINITY ? 0.f : M;
  L = 0.f;
  O = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const float f = __builtin_amdgcn_exp2f(sm[i] - mu);
    L += sl[i] * f;
    O += *reinterpret_cast<const f32x4_t*>(&so[i][d]) * f;
  }
  const uint32_t o0 = E<DT>::from_f(O[0] / L) | (uint32_t)E<DT>::from_f(O[1] / L) << 16;
  const uint32_t o1 = E<DT>::from_f(O[2] / L) | (uint32_t)E<DT>::from_f(O[3] / L) << 16;
  *reinterpret_cast<uint2*>(a.out + (long)row * a.so_b + (long)head * a.so_h + d) = make_uint2(o0, o1);
}

// ---------------------------------------------------------------------------------------------------------
namespace {
int kv4_check(const void* k, const void* ks, const void* v, const void* vs, int slots, int kv_heads, int head_dim,
              int cap) {
  if (slots <= 0 || kv_heads <= 0 || cap <= 0) return M3X_EINVAL;
  if (!k || !ks || !v || !vs) return M3X_ENULL;
  if (head_dim != 64 && head_dim != 128) return M3X_EUNSUPPORTED;
  if (cap % 32 || !m3x_aligned16(k) || !m3x_aligned16(v) || !m3x_aligned16(ks) || !m3x_aligned16(vs)) return M3X_EINVAL;
  return M3X_OK;
}
// items of D / 8 threads that a grid of 256-thread workgroups can hold
bool kv4_fits(long items) { return items <= (1L << 31); }
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

M3X_API int m3x_kv4_append(const void* k, long sk_r, long sk_h, const void* v, long sv_r, long sv_h, void* k4, void* ks4,
                           void* v4, void* vs4, const int64_t* slots, const int32_t* pos, int rows, int nslots,
                           int kv_heads, int head_dim, int cap, int dtype, void* stream) {
  if (rows < 0) return M3X_EINVAL;
  if (const int st = kv4_check(k4, ks4, v4, vs4, nslots, kv_heads, head_dim, cap)) return st;
  if (dtype != M3X_BF16 && dtype != M3X_F16) return M3X_EUNSUPPORTED;
  if (rows == 0) return M3X_OK;
  if (!k || !v || !slots || !pos) return M3X_ENULL;
  if (((sk_r | sk_h | sv_r | sv_h) & 7) || !m3x_aligned16(k) || !m3x_aligned16(v)) return M3X_EINVAL;
  const long items = (long)rows * kv_heads;
  if (!kv4_fits(items)) return M3X_EINVAL;
  const Kv4 c = {(uint8_t*)k4, (uint8_t*)ks4, (uint8_t*)v4, (uint8_t*)vs4, nslots, kv_heads, cap};
  KV4_DISPATCH(kv4_append_kernel, dim3(m3x_ceil_div(items, 2048 / head_dim)), (const uint16_t*)k, sk_r, sk_h,
               (const uint16_t*)v, sv_r, sv_h, c, slots, pos, rows);
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}

M3X_API int m3x_qk_norm_rope_kv4(const void* qkv, long s_qkv, void* q_out, long s_qo_b, long s_qo_h, void* k4, void* ks4,
                                 void* v4, void* vs4, const int64_t* slots, const int32_t* pos, const void* cos,
                                 const void* sin, long s_cos, const void* wq, const void* wk, float eps, int rows,
                                 int heads, int nslots, int kv_heads, int head_dim, int cap, void* stream) {
  if (rows < 0 || heads <= 0) return M3X_EINVAL;
  if (const int st = kv4_check(k4, ks4, v4, vs4, nslots, kv_heads, head_dim, cap)) return st;
  if (rows == 0) return M3X_OK;
  if (!qkv || !q_out || !slots || !pos || !cos || !sin || !wq || !wk) return M3X_ENULL;
  if ((s_qkv | s_qo_b | s_qo_h | s_cos) & 7) return M3X_EINVAL;
  if (!m3x_aligned16(qkv) || !m3x_aligned16(q_out) || !m3x_aligned16(cos) || !m3x_aligned16(sin) ||
      !m3x_aligned16(wq) || !m3x_aligned16(wk))
    return M3X_EINVAL;
  const long items = (long)rows * (heads + kv_heads);
  if (!kv4_fits(items)) return M3X_EINVAL;
  const Kv4 c = {(uint8_t*)k4, (uint8_t*)ks4, (uint8_t*)v4, (uint8_t*)vs4, nslots, kv_heads, cap};
  const dim3 grid(m3x_ceil_div(items, 2048 / head_dim));
#define KV4_QKN(DD)                                                                                                   \
  hipLaunchKernelGGL((qk_norm_rope_kv4_kernel<DD>), grid, dim3(256), 0, (hipStream_t)stream, (const uint16_t*)qkv,     \
                     s_qkv, (uint16_t*)q_out, s_qo_b, s_qo_h, c, slots, pos, (const uint16_t*)cos,                     \
                     (const uint16_t*)sin, s_cos, (const uint16_t*)wq, (const uint16_t*)wk, eps, rows, heads)
  if (head_dim == 128) KV4_QKN(128);
  else KV4_QKN(64);
#undef KV4_QKN
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}

M3X_API int m3x_kv4_read(const void* k4, const void* ks4, const void* v4, const void* vs4, const int64_t* slots,
                         const int32_t* pos, void* k, long sk_r, long sk_h, void* v, long sv_r, long sv_h, int rows,
                         int nslots, int kv_heads, int head_dim, int cap, int dtype, void* stream) {
  if (rows < 0) return M3X_EINVAL;
  if (const int st = kv4_check(k4, ks4, v4, vs4, nslots, kv_heads, head_dim, cap)) return st;
  if (dtype != M3X_BF16 && dtype != M3X_F16) return M3X_EUNSUPPORTED;
  if (rows == 0) return M3X_OK;
  if (!k || !v || !slots || !pos) return M3X_ENULL;
  if (((sk_r | sk_h | sv_r | sv_h) & 7) || !m3x_aligned16(k) || !m3x_aligned16(v)) return M3X_EINVAL;
  const long items = (long)rows * kv_heads;
  if (!kv4_fits(items)) return M3X_EINVAL;
  const Kv4 c = {(uint8_t*)k4, (uint8_t*)ks4, (uint8_t*)v4, (uint8_t*)vs4, nslots, kv_heads, cap};
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

M3X_API int m3x_kv4_attn(const void* q, long sq_b, long sq_h, const void* k4, const void* ks4, const void* v4,
                         const void* vs4, void* out, long so_b, long so_h, const int64_t* slots, const int32_t* pos,
                         float scale, int rows, int heads, int nslots, int kv_heads, int head_dim, int cap, int max_ctx,
                         int chunk, void* workspace, size_t ws_bytes, int dtype, void* stream) {
  if (rows < 0 || heads <= 0 || max_ctx <= 0) return M3X_EINVAL;
  if (const int st = kv4_check(k4, ks4, v4, vs4, nslots, kv_heads, head_dim, cap)) return st;
  if (dtype != M3X_BF16 && dtype != M3X_F16) return M3X_EUNSUPPORTED;
  if (heads % kv_heads) return M3X_EUNSUPPORTED;
  if (chunk <= 0 || chunk % 128 || max_ctx > cap) return M3X_EINVAL;
  if (rows == 0) return M3X_OK;
  if (!q || !out || !slots || !pos) return M3X_ENULL;
  if (((sq_b | sq_h | so_b | so_h) & 7) || !m3x_aligned16(q) || !m3x_aligned16(out)) return M3X_EINVAL;
  const int splits = m3x_ceil_div(max_ctx, chunk);
  const int G = heads / kv_heads, hb = m3x_ceil_div(G, 16);
  if ((long)kv_heads * hb > 65535 || heads > 65535 || splits > 65535) return M3X_EINVAL;
  if (splits > 1) {
    if (!workspace) return M3X_ENULL;
    if (ws_bytes < m3x_kv4_attn_workspace(rows, heads, head_dim, max_ctx, chunk)) return M3X_EWORKSPACE;
    if (!m3x_aligned16(workspace)) return M3X_EINVAL;
  }
  const Kv4 c = {(uint8_t*)k4, (uint8_t*)ks4, (uint8_t*)v4, (uint8_t*)vs4, nslots, kv_heads, cap};
  const Kv4Attn a = {(const uint16_t*)q, sq_b, sq_h, (uint16_t*)out, so_b, so_h, slots, pos,
                     scale * 1.44269504088896341f, rows, heads, G, hb, chunk, max_ctx, splits, (float*)workspace};
  KV4_DISPATCH(kv4_attn_kernel, dim3(rows, kv_heads * hb, splits), c, a);
  if (splits > 1) KV4_DISPATCH(kv4_combine_kernel, dim3(rows, heads), c, a);
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}
