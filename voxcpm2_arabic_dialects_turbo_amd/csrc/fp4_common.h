// The 4-bit KV cache (OCP MXFP4) on gfx950: layout, conversions and the MFMA that takes its codes as they are stored.
//
// Every 32 channels of one token and kv head share a power of two, held as a byte b that stands for 2^(b - 127) (e8m0;
// 255: not a number), and a value is one of {0, .5, 1, 1.5, 2, 3, 4, 6} times it with a sign (e2m1, 4 bits; channel 2i
// in the low nibble of byte i). A head's 128 channels are 64 bytes of codes and 4 scales: 68 bytes, 256 in bf16.
//
// A plane (K or V of one layer) is [num_blocks][block_size * HK * 68] bytes. Inside a block the codes
// [block_size][HK][64] come first, then the scales [block_size][HK][4]: both runs are aligned for 16-byte accesses, a
// token's codes are one run of HK * 64 bytes, and a lane's 16 bytes of codes have exactly one scale.
#pragma once

#include "vox_common.h"

namespace vox {

namespace {

namespace fp4 {

constexpr int kD = 128;
constexpr int kHeadCodes = 64;   // bytes of a head's codes
constexpr int kHeadScales = 4;   // bytes of a head's scales
constexpr int kHeadBytes = kHeadCodes + kHeadScales;
// word 3 of a raw buffer descriptor (32-bit data format; byte offsets, range-checked against num_records)
constexpr int kBufferWord3 = 0x00020000;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__host__ __device__ __forceinline__ int64_t block_bytes(int block_size, int hk) {
  return (int64_t)block_size * hk * kHeadBytes;
}

// The float 2^(b - 127) of a scale byte, as the conversion instructions take it: they use its exponent field alone, so
// byte 0 (a zero float) is 2^-127 and byte 255 (infinity) gives NaN for every code.
__device__ __forceinline__ float scale_float(uint32_t b) { return __uint_as_float(b << 23); }

// The scale byte of a group whose largest magnitude has the bf16 bits `amax` (sign cleared): the least power of two that
// leaves the largest value at most 7 times it, so it is off by at most half a step of its binade ([4, 6], where 7 is
// held as 6); at least 2^-126, a normal float, and at most 2^125, whose 6 is the largest that bf16 holds (at 2^126 a 4 is
// 2^128, an infinity); 255 where the group holds an infinity or NaN.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  const int e = (int)(amax >> 7) - 2 + ((amax & 0x7fu) > 0x60u ? 1 : 0);
  return amax >= 0x7f80u ? 255u : (uint32_t)max(1, min(252, e));
}

// 8 bf16 (packed) to 8 codes: round to nearest, ties to the even code, saturating at 6.
__device__ __forceinline__ uint32_t codes8(u32x4 x, float scale) {
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (uint32_t)x[0]), scale, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (uint32_t)x[1]), scale, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (uint32_t)x[2]), scale, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, (uint32_t)x[3]), scale, 3);
  return r;
}

// The largest magnitude of 8 packed bf16, as bits (so that infinity and NaN count as the largest).
__device__ __forceinline__ uint32_t max_bits(u32x4 x) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x2 m = __builtin_bit_cast(u16x2, (uint32_t)(x[0] & 0x7fff7fffu));
#pragma unroll
  for (int i = 1; i < 4; ++i)
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, (uint32_t)(x[i] & 0x7fff7fffu)));
  return max((uint32_t)m[0], (uint32_t)m[1]);
}

// 8 channels of a row by each of four neighbouring lanes, a group together: this lane's codes, the group's scale byte.
__device__ __forceinline__ void quantise8(u32x4 x, uint32_t& codes, uint32_t& b) {
  uint32_t m = max_bits(x);
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));  // quad_perm [1,0,3,2]
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));  // quad_perm [2,3,0,1]
  b = scale_byte(m);
  codes = b == 255u ? 0u : codes8(x, scale_float(b));
}

// 8 codes to 8 bf16 (packed): exact, a 2-bit significand and the scale's exponent, but for those from 2^128 on, which become
// infinities (a 4 at 2^126, a 2 at 2^127).
__device__ __forceinline__ u32x4 values8(uint32_t codes, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
}

// The same under scale byte b, a quarter of it: exact at every byte (2^-130, three steps of bf16's least one, to 1.5 x 2^127), where
// values8 has infinities from 2^128 on. 255 gives NaN.
__device__ __forceinline__ u32x4 quarter_values8(uint32_t codes, uint32_t b) {
  u32x4 v = values8(codes, scale_float(b == 255u ? 255u : 127u));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = __builtin_ldexpf(__uint_as_float(v[i] << 16), (int)b - 129);
    const float hi = __builtin_ldexpf(__uint_as_float(v[i] & 0xffff0000u), (int)b - 129);
    v[i] = __float_as_uint(lo) >> 16 | (__float_as_uint(hi) & 0xffff0000u);
  }
  return v;
}

// Whether one of a head's four scale bytes is 253 or more: its codes may stand for more than bf16 holds.
__device__ __forceinline__ bool past_bf16(uint32_t scales) {
  return (scales & 0xffu) >= 253u || (scales >> 8 & 0xffu) >= 253u || (scales >> 16 & 0xffu) >= 253u || scales >> 24 >= 253u;
}

// The scale byte b of 32 codes as V's conversion to bf16 takes it: 255 too where they stand for more than bf16 holds, from
// 2^128 on (a 4 at 2^126, a 2 at 2^127: planes that others have written, the store's scales end at 2^125). As an infinity such a
// value would be NaN wherever it meets a probability of 0.
__device__ __forceinline__ uint32_t held_scale(uint32_t b, u32x4 codes) {
  uint32_t past = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) past |= (b == 253u ? codes[i] & (codes[i] << 1) : codes[i]) & 0x44444444u;
  return b >= 253u && past != 0 ? 255u : b;
}

// The scores' MFMAs: D(fp32) += A(fp4 codes) B(fp8 e4m3), each 32 contraction elements with a scale byte of their own
// (byte OP of the lane's register).
//   16x16x128: lane l's codes are A[l % 16][32 (l / 16) + [0, 32)], its scale that block's; its B bytes 0-15 are
//   B[16 (l / 16) + [0, 16)][l % 16] and bytes 16-31 B[64 + 16 (l / 16) + [0, 16)][l % 16], its B scale that of rows
//   32 (l / 16) + [0, 32). D as in mfma_16x16x32.
//   32x32x64: A[l % 32][32 (l / 32) + [0, 32)]; B[16 (l / 32) + [0, 16)][l % 32] and B[32 + 16 (l / 32) + [0, 16)]. D as
//   in mfma_32x32x16.
// The products are exact and the sum is held in fp32; with a score's 128 terms it is off by 2^-18 of the score's size in
// the mean (measured over normal q and K), where the bf16 probabilities are off by up to 2^-8.
__device__ __forceinline__ f32x4 mfma_scores16(u32x4 a, uint32_t sa, i32x8 b, uint32_t sb, f32x4 c) {
  const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, b, c, 4, 0, 0, (int)sa, 0, (int)sb);
}
template <int OP>
__device__ __forceinline__ f32x16 mfma_scores32(u32x4 a, uint32_t sa, i32x8 b, uint32_t sb, f32x16 c) {
  const i32x8 av = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, b, c, 4, 0, OP, (int)sa, 0, (int)sb);
}

// A query value in fp8: q = (hi + lo) 2^(e - 127) with hi the nearest e4m3 and lo what it leaves. bf16 has 8 significant
// bits and e4m3 4, so the pair is exact down to 2^-10 of the row's largest magnitude, and below it off by at most
// 2^-18 of that. e is the row's: its largest magnitude becomes a value in [128, 256).
__device__ __forceinline__ uint32_t query_scale_byte(uint32_t amax_bits) {
  return (uint32_t)max(1, (int)(amax_bits >> 7) - 7);
}
// 1 / scale_float(b) for b in [1, 248]
__device__ __forceinline__ float query_inverse(uint32_t b) { return __uint_as_float((254u - b) << 23); }

// The parts of 4 values (packed bf16) as 4 packed bytes each: the high ones straight from bf16 under the scale 2^(e - 127),
// the low ones from what those leave of x inv, inv = 2^(127 - e) (exact: a power of two, and hi is near).
__device__ __forceinline__ void query_parts4(uint32_t a, uint32_t b, float scale, float inv, int& hi, int& lo) {
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  i16x2 h = {0, 0};
  h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(bf16x2, a), scale, false);
  h = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(h, __builtin_bit_cast(bf16x2, b), scale, true);
  hi = __builtin_bit_cast(int, h);
  const auto y0 = __builtin_amdgcn_cvt_pk_f32_fp8(hi, false), y1 = __builtin_amdgcn_cvt_pk_f32_fp8(hi, true);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(fmaf(__uint_as_float(a << 16), inv, -y0[0]),
                                       fmaf(__uint_as_float(a & 0xffff0000u), inv, -y0[1]), 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(fmaf(__uint_as_float(b << 16), inv, -y1[0]),
                                       fmaf(__uint_as_float(b & 0xffff0000u), inv, -y1[1]), lo, true);
}

}  // namespace fp4

}  // namespace

}  // namespace vox
