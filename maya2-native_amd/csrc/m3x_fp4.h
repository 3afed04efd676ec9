// The 4-bit group format of the KV cache (kv4.hip) and of the packed weights (gemm4.hip).
//
// A group of 32 numbers x is 32 E2M1 codes and one scale byte b standing for s = 2^(b - 127):
//   s     the smallest power of two with max|x| <= 7 s, b in [1, top]; top = 252 (fp16 numbers: 140), so that 6 s, the
//         largest value, is finite in the 16-bit type. b = 255 marks a group that held a NaN or an infinity.
//   code  sign (bit 3) and magnitude 0, .5, 1, 1.5, 2, 3, 4, 6 (bits 0..2) of x / s, to nearest, ties to the even code,
//         6 above 5.
// The numbers up to 7 s that a limit of 6 s would push to the next scale lose at most s, which is also the largest
// rounding error below 6 s (half the step from 4 to 6), so |x - value| <= s either way and a group keeps the finer
// grid whenever it can. Quantising is exact arithmetic (a power-of-two scale, one rounding): the same bits from any
// evaluation. gfx950 converts both ways in hardware, two numbers an instruction with the scale applied
// (v_cvt_scalef32_pk_*): a value is a 16-bit number without error, so no product is rounded before it is summed.
// Measured on MI355X: the conversion runs at the full VALU rate (32.5 T lane-operations/s, as v_perm_b32), rounds
// to nearest even and saturates, and a scale of 255 gives NaN (checked for every bf16 and fp16 number).
#pragma once
#include "m3x_common.h"

typedef __bf16 fp4_bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 fp4_h2 __attribute__((ext_vector_type(2)));
typedef uint32_t fp4_u2 __attribute__((ext_vector_type(2)));
typedef uint32_t fp4_u4 __attribute__((ext_vector_type(4)));

template <int DT> __device__ __forceinline__ constexpr uint32_t fp4_top_of() { return DT == M3X_F16 ? 140u : 252u; }

// scale byte of a group whose largest magnitude is `amax` (finite): 1.m x 2^(E - 127) <= 7 x 2^(b - 127) means
// b = E - 2 up to m = 0.75 and E - 1 above; the sum carries into the exponent exactly there
__device__ __forceinline__ uint32_t fp4_scale_byte(float amax, uint32_t top) {
  const int b = (int)((__float_as_uint(amax) + 0x1FFFFFu) >> 23) - 2;
  return (uint32_t)min(max(b, 1), (int)top);
}

// 2^(b - 127) as the conversions take it: the exponent field counts, sign and mantissa do not (checked on MI355X for
// random words), so what stands beside the byte may stay. b = 255 gives NaN.
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }
// the same from byte I of a word
template <int I> __device__ __forceinline__ float fp4_scale_of(uint32_t w) {
  if constexpr (I == 3) return __uint_as_float(w >> 1);
  else return __uint_as_float(w << (23 - 8 * I));
}

// the two numbers of byte SEL of w, packed 16-bit (low code first)
template <int DT, int SEL> __device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float scale) {
  if constexpr (DT == M3X_F16)
    return __builtin_bit_cast(uint32_t, (fp4_h2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, SEL));
  else
    return __builtin_bit_cast(uint32_t, (fp4_bf2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
// a | b << 16 as 16-bit numbers (to nearest even), one instruction
template <int DT> __device__ __forceinline__ uint32_t fp4_pack(float a, float b) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  if constexpr (DT == M3X_F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), fp4_h2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), fp4_bf2));
}
// acc + both 16-bit numbers of w (none negative), in fp32, one instruction. Measured: within 3.4 x 2^-24 of the sum,
// fp16's subnormal numbers kept (262144 random pairs).
template <int DT> __device__ __forceinline__ float fp4_add2(uint32_t w, float acc) {
  if constexpr (DT == M3X_F16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(fp4_h2, w), __builtin_bit_cast(fp4_h2, 0x3C003C00u), acc, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(fp4_bf2, w), __builtin_bit_cast(fp4_bf2, 0x3F803F80u), acc,
                                           false);
}
// the eight numbers of w in order
template <int DT> __device__ __forceinline__ u16x8 fp4_eight(uint32_t w, float scale) {
  const fp4_u4 r = {fp4_pair<DT, 0>(w, scale), fp4_pair<DT, 1>(w, scale), fp4_pair<DT, 2>(w, scale),
                    fp4_pair<DT, 3>(w, scale)};
  return __builtin_bit_cast(u16x8, r);
}

// Eight consecutive numbers of a group that four adjacent lanes of a quad hold (lane % 4 = the eighth's place): their
// codes as one word, and the group's scale byte. Every lane of the quad calls it.
template <int DT> __device__ __forceinline__ uint32_t fp4_quantise8(const u16x8& x, uint32_t& byte) {
  const fp4_u4 w = __builtin_bit_cast(fp4_u4, x);
  uint32_t m = 0;  // magnitudes order as integers, infinities and NaN above every number
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, (uint32_t)x.v[e] & 0x7FFFu);
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, false));  // quad_perm [1,0,3,2]
  m = max(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, false));  // quad_perm [2,3,0,1]
  if (m >= (DT == M3X_F16 ? 0x7C00u : 0x7F80u)) {
    byte = 255;
    return 0;
  }
  byte = fp4_scale_byte(E<DT>::to_f((uint16_t)m), fp4_top_of<DT>());
  const float s = fp4_scale(byte);
  uint32_t r = 0;
  if constexpr (DT == M3X_F16) {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(fp4_h2, (uint32_t)w[0]), s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(fp4_h2, (uint32_t)w[1]), s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(fp4_h2, (uint32_t)w[2]), s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(fp4_h2, (uint32_t)w[3]), s, 3);
  } else {
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(fp4_bf2, (uint32_t)w[0]), s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(fp4_bf2, (uint32_t)w[1]), s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(fp4_bf2, (uint32_t)w[2]), s, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(fp4_bf2, (uint32_t)w[3]), s, 3);
  }
  return r;
}
