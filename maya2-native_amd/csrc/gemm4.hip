// Products of few rows with 4-bit weights and a scale per 32 inputs (format: m3x_fp4.h): y = act(x . W^T).
//
// Packed weight [N, K]: N in tiles of 16 rows (zero rows behind N), K in steps of 128 (zeros behind K). A step's codes
// are 1 KB: lane l's 16 bytes hold row l % 16, inputs 32 (l / 16) .. + 31, i.e. one group; its scale bytes of four
// consecutive steps are one word, so a wave reads contiguous kilobytes and a lane applies one scale to all it holds.
//   codes  [tiles][steps][64][16]      scales [tiles][ceil(steps / 4)][64][4]
//
// Bound: the weights' bytes, 17 / 32 of a byte each, and below some megabytes the launch and one memory round trip. A
// lane's words become 16-bit MFMA operands in registers (16 conversions a KB) and meet the rows of x, the product's
// columns, as read from memory: per step and 16 rows of x four MFMA 16x16x32, the lane's inputs 8 i .. 8 i + 7 in the
// i-th. The waves of a workgroup share the steps out and their sums meet in LDS, added in wave order (deterministic).
// Products and sums are fp32; the one rounding is the store's. Measured on MI355X: 9 rows through 16384 x 8192 (71.3 MB
// of weights) 15.6 us, 4.6 TB/s; one row through 4096 x 1024 3.1 us; 64 rows through 2816 x 1024 twice, gated, 5.5 us. Past 32
// rows the weights are read once per 32 (gated 64) rows: 64 rows through 16384 x 8192 29 us, 256 rows 113.
#include "m3x_fp4.h"

namespace {
struct Lin4 {
  const uint16_t* x;
  long ldx;
  const uint8_t* w[2];
  const uint8_t* s[2];
  uint16_t* y;
  long ldy;
  int M, N, K, steps, tiles;
};
enum { L4_NONE, L4_SWIGLU, L4_GELU };
}  // namespace

// TW output tiles and 16 MT rows of x per workgroup of NW waves.
//
// A lane's operand of x is 64 bytes of one row. Read as such (TURN false), each lane's 16 bytes are an access of their own
// to the vector L1, which from some rows on costs more than the weights do. With TURN a load takes four rows' 256
// contiguous bytes, and the wave turns them over in 4 KB of LDS of its own (places swapped by the row, so that neither
// side meets in a bank).
template <int DT, int TW, int MT, int NW, int ACT, bool TURN>
__global__ __launch_bounds__(64 * NW) void linear4_kernel(Lin4 a) {
  constexpr int P = ACT == L4_SWIGLU ? 2 : 1;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int li = lane & 15, lg = lane >> 4;
  const int tile0 = blockIdx.x * TW;
  const int m0 = blockIdx.y * (16 * MT);
  const int quads = (a.steps + 3) >> 2;
  const int per = (a.steps + NW - 1) / NW;
  const int s0 = wave * per, s1 = min(s0 + per, a.steps);

  f32x4_t acc[TW * P][MT];
#pragma unroll
  for (int t = 0; t < TW * P; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[t][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  // as many output tiles at a time as 64 KB hold the waves' sums of
  constexpr int RT = NW * P * MT * TW <= 64 ? TW : 64 / (NW * P * MT);
  constexpr int SUMS = NW * RT * P * MT * 64, STAGE = TURN ? NW * MT * 256 : 0;  // 16-byte places
  __shared__ fp4_u4 lds[SUMS > STAGE ? SUMS : STAGE];
  fp4_u4* const stage = lds + wave * (MT * 256);

  struct Step {
    fp4_u4 cw[TW * P];
    uint32_t sw[TW * P];
    fp4_u4 x[MT][4];
  };
  const int xr = TURN ? lane >> 4 : li, xp = TURN ? lane & 15 : 4 * lg;  // what the lane loads: row, 16-byte piece
  auto load = [&](Step& q, int s) {
#pragma unroll
    for (int t = 0; t < TW * P; ++t) {
      const long tile = min(tile0 + t / P, a.tiles - 1);  // a tile past the last repeats it and is not stored
      q.cw[t] = __builtin_nontemporal_load(
          reinterpret_cast<const fp4_u4*>(a.w[t % P] + ((tile * a.steps + s) * 64 + lane) * 16));
      q.sw[t] = *reinterpret_cast<const uint32_t*>(a.s[t % P] + ((tile * quads + (s >> 2)) * 64 + lane) * 4);
    }
    const int k = 128 * s + 8 * xp;
    const fp4_u4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if constexpr (TURN) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = m0 + 16 * m + 4 * i + xr;
          q.x[m][i] = r < a.M && k < a.K ? __builtin_bit_cast(fp4_u4, ld16(a.x + (long)r * a.ldx + k)) : zero;
        }
      } else {
        const int r = m0 + 16 * m + xr;
        if (r < a.M && k < a.K) {
#pragma unroll
          for (int i = 0; i < 4; ++i) q.x[m][i] = __builtin_bit_cast(fp4_u4, ld16(a.x + (long)r * a.ldx + k + 8 * i));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) q.x[m][i] = zero;
        }
      }
    }
  };
  auto multiply = [&](Step& q, int s) {
    if constexpr (TURN) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();  // the step before has been read
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) stage[256 * m + 16 * (4 * i + xr) + (xp ^ (4 * i + xr))] = q.x[m][i];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) q.x[m][i] = stage[256 * m + 16 * li + ((4 * lg + i) ^ li)];
    }
#pragma unroll
    for (int t = 0; t < TW * P; ++t) {
      const float sc = fp4_scale((q.sw[t] >> (8 * (s & 3))) & 255u);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u16x8 wv = fp4_eight<DT>(q.cw[t][i], sc);
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[t][m] = mfma16x16x32<DT>(wv, __builtin_bit_cast(u16x8, q.x[m][i]), acc[t][m]);
      }
    }
  };
  for (int s = s0; s < s1; ++s) {
    Step q;
    load(q, s);
    multiply(q, s);
  }

  typedef f32x4_t Sums[RT * P * MT][64];
  Sums* const red = reinterpret_cast<Sums*>(lds);
#pragma unroll
  for (int t0 = 0; t0 < TW; t0 += RT) {
    if (TURN || t0) __syncthreads();  // the waves' x, or the tiles before, have been read
#pragma unroll
    for (int i = 0; i < RT * P * MT; ++i) red[wave][i][lane] = acc[t0 * P + i / MT][i % MT];
    __syncthreads();
    for (int f = wave; f < RT * MT; f += NW) {
      const int t = f / MT, m = f % MT;
      f32x4_t v[P];
#pragma unroll
      for (int p = 0; p < P; ++p) {
        v[p] = red[0][(t * P + p) * MT + m][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) v[p] += red[w][(t * P + p) * MT + m][lane];
      }
      const int row = m0 + 16 * m + li;
      const int n = 16 * (tile0 + t0 + t) + 4 * lg;
      if (row >= a.M || n >= a.N) continue;
      uint16_t o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float y = v[0][r];
        if constexpr (ACT == L4_SWIGLU) y = silu16(y) * v[P - 1][r];
        if constexpr (ACT == L4_GELU) y = 0.5f * y * (1.f + erff(y * 0.70710678118654752f));
        o[r] = E<DT>::from_f(y);
      }
      uint16_t* yp = a.y + (long)row * a.ldy + n;
      if (n + 4 <= a.N && (((uintptr_t)yp) & 7) == 0) {
        *reinterpret_cast<uint2*>(yp) = make_uint2(o[0] | (uint32_t)o[1] << 16, o[2] | (uint32_t)o[3] << 16);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (n + r < a.N) yp[r] = o[r];
      }
    }
  }
}

// A wave per tile and step: a lane reads its group, finds the scale and stores 16 bytes of codes. Once at load time.
template <int DT>
__global__ __launch_bounds__(64) void pack_weight4_kernel(const Elt<DT>* __restrict__ w, long ldw, int N, int K,
                                                          uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                          int steps) {
  const int lane = threadIdx.x;
  const long tile = blockIdx.x / steps;
  const int s = blockIdx.x - (int)tile * steps;
  const int row = 16 * (int)tile + (lane & 15), k = 128 * s + 32 * (lane >> 4);
  float x[32];
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 32; e += 8) {
    const V8<DT> v = row < N && k < K ? ldv<DT>(w + (long)row * ldw + k + e) : zero_v8<DT>();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[e + i] = E<DT>::to_f(v.v[i]);
      m = max(m, __float_as_uint(x[e + i]) & 0x7FFFFFFFu);
    }
  }
  uint32_t byte = 255;
  fp4_u4 c = {0, 0, 0, 0};
  if (m < 0x7F800000u) {
    byte = fp4_scale_byte(__uint_as_float(m), fp4_top_of<DT>());
    const float sc = fp4_scale(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t r = 0;
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[8 * i], x[8 * i + 1], sc, 0);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[8 * i + 2], x[8 * i + 3], sc, 1);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[8 * i + 4], x[8 * i + 5], sc, 2);
      r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[8 * i + 6], x[8 * i + 7], sc, 3);
      c[i] = r;
    }
  }
  *reinterpret_cast<fp4_u4*>(codes + ((tile * steps + s) * 64 + lane) * 16) = c;
  uint8_t* sp = scales + ((tile * ((steps + 3) >> 2) + (s >> 2)) * 64 + lane) * 4;
  sp[s & 3] = (uint8_t)byte;
  if (s == steps - 1)
    for (int i = (s & 3) + 1; i < 4; ++i) sp[i] = 1;  // steps that are not there
}

M3X_API long m3x_packed_weight4_bytes(int N, int K, int scales) {
  if (N <= 0 || K <= 0 || K % 32) return -1;
  const long tiles = (N + 15L) / 16, steps = (K + 127L) / 128;
  return scales ? tiles * ((steps + 3) / 4) * 256 : tiles * steps * 1024;
}

M3X_API int m3x_pack_weight4(const void* w, long ldw, int N, int K, void* codes, void* scales, int dtype,
                             void* stream) {
  if (N <= 0 || K <= 0 || K % 32 || ldw & 7) return M3X_EINVAL;
  if (!w || !codes || !scales) return M3X_ENULL;
  if (!m3x_aligned16(w) || !m3x_aligned16(codes) || !m3x_aligned16(scales)) return M3X_EINVAL;
  const int steps = m3x_ceil_div(K, 128), tiles = m3x_ceil_div(N, 16);
  hipStream_t st = (hipStream_t)stream;
  if ((long)tiles * steps >= 1L << 26) return M3X_EINVAL;  // a launch of fewer than 2^32 threads
  const dim3 grid(tiles * steps);
  if (dtype == M3X_BF16)
    hipLaunchKernelGGL(pack_weight4_kernel<M3X_BF16>, grid, dim3(64), 0, st, (const uint16_t*)w, ldw, N, K,
                       (uint8_t*)codes, (uint8_t*)scales, steps);
  else if (dtype == M3X_F16)
    hipLaunchKernelGGL(pack_weight4_kernel<M3X_F16>, grid, dim3(64), 0, st, (const uint16_t*)w, ldw, N, K,
                       (uint8_t*)codes, (uint8_t*)scales, steps);
  else if (dtype == M3X_F32)
    hipLaunchKernelGGL(pack_weight4_kernel<M3X_F32>, grid, dim3(64), 0, st, (const float*)w, ldw, N, K,
                       (uint8_t*)codes, (uint8_t*)scales, steps);
  else
    return M3X_EUNSUPPORTED;
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}

namespace {
// x turned over in LDS or not, measured on MI355X (us; not, turned): N 1024, K 8192 (1x1x8) 9 rows 8.1, 9.0, 12 rows 9.0,
// 9.0, 16 rows 10.2, 9.5; N 5000, K 8192 (2x1x8) 5 rows 9.5, 10.5, 8 rows 9.7, 10.6, 12 rows 10.6, 10.9, 16 rows 12.1, 11.2,
// gated 8 rows 12.6, 12.7, 12 rows 14.0, 13.5, 16 rows 15.3, 13.9; N 16384, K 8192 (4x1x16) 9 rows 17.4, 17.8, 16 rows 18.8,
// 17.9; 64 rows (8x2x8) 32.9, 29.1; N 11008, K 4096, 128 rows gated (4x4x4, where it takes 304 of a wave's registers) 48, 58.
template <int DT, int TW, int MT, int NW, int ACT> void launch4(const Lin4& a, hipStream_t st) {
  const dim3 grid(m3x_ceil_div(a.tiles, TW), m3x_ceil_div(a.M, 16 * MT)), block(64 * NW);
  if constexpr (MT == 1) {
    if (a.M > 12) hipLaunchKernelGGL((linear4_kernel<DT, TW, MT, NW, ACT, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((linear4_kernel<DT, TW, MT, NW, ACT, false>), grid, block, 0, st, a);
  } else {
    hipLaunchKernelGGL((linear4_kernel<DT, TW, MT, NW, ACT, MT == 2>), grid, block, 0, st, a);
  }
}
template <int DT, int ACT> void plan4(const Lin4& a, hipStream_t st) {
  // Weight tiles times 16-row blocks are dealt out over 256 CUs: a workgroup takes as many as leave every CU about one, so
  // that x, which every group of tiles reads anew, is read the fewest times. Past 16 a CU, and for few steps of K, where a
  // large group's start and sums weigh more, smaller groups run in several rounds. A gated group of 4x4x4 leaves CUs idle below
  // some 2800 units, which costs more than the smaller groups' rounds up to 25 steps. Measured on MI355X (us; TW x MT x NW,
  // the rule's first):
  //   plain, K 8192  N 16384: 16 rows 4x1x16 17.9, 2x1x8 18.9, 1x1x8 25; 32 rows 4x2x8 21.8, 8x2x8 28, 4x1x16 31; 64 rows
  //                  8x2x8 29.1, 4x2x8 35; 256 rows 8x2x8 113, 4x2x8 125. N 5000: 16 rows 2x1x8 11.2, 1x1x8 13.8
  //   plain, K 4096  N 11008: 16 rows 4x1x16 9.4, 2x1x8 11.2; 32 rows 4x2x8 12.8, 4x1x16 16; 256 rows 4x2x8 49, 8x2x8 56
  //   plain, K 1024  N 4096: 16 rows 1x1x8 3.4, 2x1x8 3.8; 64 rows 2x1x8 4.5, 4x1x16 4.8; 128 rows 2x1x8 5.5, 4x2x8 5.4, 8x2x8
  //                  7.7; 256 rows 4x2x8 7.1, 8x2x8 8.0
  //   GELU           N 4096, K 1024: 16 rows 1x1x8 3.9, 2x1x8 4.3; 64 rows 2x1x8 5.0, 4x1x16 5.4; 256 rows 4x2x8 8.1, 8x2x8 8.9;
  //                  N 16384, K 8192: 16 rows 4x1x16 19.5, 2x1x8 20.2; 64 rows 8x2x8 30.7, 4x2x8 37
  //   gated, K 8192  N 16384: 16 rows 2x1x8 30.6, 4x1x8 29.4; 32 rows 4x2x8 34.3, 2x2x8 37.4; 64 rows 4x4x4 46, 4x2x8 65.
  //                  N 11008: 64 rows (2752 units) 4x4x4 44, 2x2x8 50
  //   gated, K 1024  N 4096: 64 rows 2x2x8 5.7, 4x2x8 7.4; 128 rows 2x2x8 7.6, 4x2x8 7.6; 256 rows 2x2x8 11.1, 4x4x4 12.0
  //   gated, 9 to 32 steps (2x2x8, 4x4x4): 2560 units K 1152 11.6, 13.2, K 2048 15.2, 18.3, K 3200 22.4, 25.0, K 4096 27.6, 27.0;
  //                  2752 units K 1536 13.8, 15.8, K 3200 23.1, 25.4; 3072 units K 1152 14.6, 13.0, K 2048 19.5, 18.8; 4096
  //                  units K 1152 14.5, 13.5, K 2048 20.5, 20.4, K 2304 22.3, 20.2
  const int blocks = m3x_ceil_div(a.M, 16);
  const long units = (long)a.tiles * blocks;
  if (units <= 256) return launch4<DT, 1, 1, 8, ACT>(a, st);
  if constexpr (ACT == L4_SWIGLU) {
    if (units <= 512 || blocks == 1) launch4<DT, 2, 1, 8, ACT>(a, st);
    else if (units <= (a.steps <= 8 ? 4096 : 1024) || (units > 2048 && units <= 2816 && a.steps <= 25))
      launch4<DT, 2, 2, 8, ACT>(a, st);
    else if (units <= 2048) launch4<DT, 4, 2, 8, ACT>(a, st);
    else launch4<DT, 4, 4, 4, ACT>(a, st);
  } else {
    if (units <= (a.steps <= 8 ? 2048 : 512)) launch4<DT, 2, 1, 8, ACT>(a, st);
    else if (blocks == 1 || (units <= 1024 && a.steps > 8)) launch4<DT, 4, 1, 16, ACT>(a, st);
    else if (units <= 2048 || a.steps <= 8 || (units > 4096 && a.steps < 64)) launch4<DT, 4, 2, 8, ACT>(a, st);
    else launch4<DT, 8, 2, 8, ACT>(a, st);
  }
}
int linear4_any(const void* x, long ldx, const void* wg, const void* sg, const void* wu, const void* su, void* y,
                long ldy, int M, int N, int K, int act, int dtype, void* stream) {
  if (M < 0 || N <= 0 || K <= 0 || K % 32) return M3X_EINVAL;
  if (dtype != M3X_BF16 && dtype != M3X_F16) return M3X_EUNSUPPORTED;
  if (act != L4_NONE && act != L4_SWIGLU && act != L4_GELU) return M3X_EUNSUPPORTED;
  if (M == 0) return M3X_OK;
  if (!x || !wg || !sg || !y || (act == L4_SWIGLU && (!wu || !su))) return M3X_ENULL;
  if ((ldx & 7) || !m3x_aligned16(x) || !m3x_aligned16(wg) || !m3x_aligned16(sg) || ((uintptr_t)y & 1)) return M3X_EINVAL;
  if (act == L4_SWIGLU && (!m3x_aligned16(wu) || !m3x_aligned16(su))) return M3X_EINVAL;
  if (M > 65535 * 16 || N > (1 << 26)) return M3X_EINVAL;  // launches of fewer than 2^32 threads
  const Lin4 a = {(const uint16_t*)x, ldx, {(const uint8_t*)wg, (const uint8_t*)wu},
                  {(const uint8_t*)sg, (const uint8_t*)su}, (uint16_t*)y, ldy, M, N, K, m3x_ceil_div(K, 128),
                  m3x_ceil_div(N, 16)};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == M3X_BF16) {
    if (act == L4_NONE) plan4<M3X_BF16, L4_NONE>(a, st);
    else if (act == L4_SWIGLU) plan4<M3X_BF16, L4_SWIGLU>(a, st);
    else plan4<M3X_BF16, L4_GELU>(a, st);
  } else {
    if (act == L4_NONE) plan4<M3X_F16, L4_NONE>(a, st);
    else if (act == L4_SWIGLU) plan4<M3X_F16, L4_SWIGLU>(a, st);
    else plan4<M3X_F16, L4_GELU>(a, st);
  }
  M3X_CHECK_LAUNCH();
  return M3X_OK;
}
}  // namespace

M3X_API int m3x_linear4(const void* x, long ldx, const void* codes, const void* scales, void* y, long ldy, int M, int N,
                        int K, int dtype, void* stream) {
  return linear4_any(x, ldx, codes, scales, nullptr, nullptr, y, ldy, M, N, K, L4_NONE, dtype, stream);
}

M3X_API int m3x_linear4_act(const void* x, long ldx, const void* g_codes, const void* g_scales, const void* u_codes,
                            const void* u_scales, void* y, long ldy, int M, int I, int K, int kind, int dtype,
                            void* stream) {
  if (kind != 0 && kind != 1) return M3X_EUNSUPPORTED;  // M3X_ACT_SWIGLU, M3X_ACT_GELU
  return linear4_any(x, ldx, g_codes, g_scales, u_codes, u_scales, y, ldy, M, I, K, kind == 0 ? L4_SWIGLU : L4_GELU,
                     dtype, stream);
}
