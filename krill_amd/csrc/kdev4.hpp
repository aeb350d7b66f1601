// The 4-bit storage mode (affine groups of 64): layout of a block's head
// region, the quantizer's scalar steps and the conversion of codes into matrix
// operands.
#pragma once

#include "kdev.hpp"

namespace krill {

// A (layer, block, KV head) region, D = head_dim, G = D / 64:
//   [0, 32 D)              K codes: D/32 pieces of 64 x 16 bytes (below)
//   [32 D, 64 D)           V codes: D/32 pieces of 64 x 16 bytes
//   [64 D, +256 G)         K (scale, bias) fp16 pairs, (t G + g) 4
//   [64 D + 256 G, +256 G) V (scale, bias) fp16 pairs
// Lane l of a wave loads the 16 bytes at 16 l of a piece, so every load of a
// block is one contiguous KB and arrives as a v_mfma_f32_16x16x32_f16 operand
// (row l % 16, contraction slots 8 (l / 16) .. +7):
//  * K: a 32-bit word holds 8 dims of a token.  Lane (n, q) = (l % 16, l / 16)
//    has words (g, h): dims 64 g + 16 q + 8 h .. +7 of token 16 tg + n.  The
//    four words of a piece are (g, h) of two groups (head_dim 64: of two 16-token
//    groups).  Dim e of a word sits in nibble (e >> 1) + 4 (e & 1), so that masks
//    of the low and of the second nibble of both halves, before and after a shift
//    by 8, leave the pairs (0,1), (2,3), (4,5), (6,7).
//  * V: a byte holds dims d (low nibble) and d + 16 of one token, so a token's
//    bytes are its own and tokens are written without read-modify-write.  Lane
//    (n, q) of piece j has 16 tokens of dims 32 j + n and 32 j + 16 + n: tokens
//    32 ks + 16 a + 4 q + x, x < 4, in word 2 ks + a, byte (x >> 1) + 2 (x & 1):
//    masks of every other byte leave the order in which the scores' tiles leave
//    P.
__host__ __device__ constexpr int q4_region_bytes(int D) { return 64 * D + 512 * (D / 64); }
__host__ __device__ constexpr int q4_v_offset(int D) { return 32 * D; }
__host__ __device__ constexpr int q4_km_offset(int D) { return 64 * D; }
__host__ __device__ constexpr int q4_vm_offset(int D) { return 64 * D + 256 * (D / 64); }
// byte of the K word of dims 8 x .. 8 x + 7 of token t
__host__ __device__ constexpr int q4_k_word(int D, int t, int x) {
  const int g = x >> 3, q = (x >> 1) & 3, h = x & 1, n = t & 15, tg = t >> 4;
  const int piece = D == 64 ? tg >> 1 : tg * (D / 128) + (g >> 1);
  const int word = (D == 64 ? (tg & 1) : (g & 1)) * 2 + h;
  return (piece * 64 + q * 16 + n) * 16 + word * 4;
}
__host__ __device__ constexpr int q4_nibble(int e) { return (e >> 1) + 4 * (e & 1); }
// byte, inside a lane's 16 of a V piece, of token t
__host__ __device__ constexpr int q4_v_slot(int t) {
  return ((t >> 5) & 1) * 8 + ((t >> 4) & 1) * 4 + ((t & 3) >> 1) + 2 * (t & 1);
}
// byte of V dims d and d + 16 (d % 32 < 16) of token t; m = 16 (d / 32) + d % 16
__host__ __device__ constexpr int q4_v_byte(int D, int t, int m) {
  return q4_v_offset(D) + (((m >> 4) * 64 + ((t >> 2) & 3) * 16 + (m & 15)) << 4) + q4_v_slot(t);
}

// ---------------------------------------------------------------- quantizer
// Elements are limited to the fp16 range; per group of 64
//   b = f16(min w),  s = f16(max(0, (max w - b) / 15)),
//   c = min(15, rint((w - b) / s)), 0 where s = 0:
// the codes refer to the scale and bias as they are stored, so the stored
// values err by half a step (the bias by its own rounding, 2^-11 of it).  A
// NaN makes its group's scale and bias NaN.
template <int DT>
__device__ __forceinline__ float q4_limit(float x) {
  // (fp16: the infinities; v_med3 would turn a NaN into a number)
  return x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x;
}
// lo / hi: the group's extremes, nan: whether it holds a NaN
__device__ __forceinline__ uint32_t q4_params(float lo, float hi, bool nan, float &s, float &b) {
  const uint16_t bb = f32_to_f16_bits(lo + 0.0f);  // (a minimum of -0 is stored as +0)
  b = f16_bits_to_f32(bb);
  const float d = hi - b;
  const uint16_t sb = f32_to_f16_bits((d > 0.0f ? d : 0.0f) / 15.0f);
  s = f16_bits_to_f32(sb);
  return nan ? 0x7e007e00u : (uint32_t)sb | ((uint32_t)bb << 16);
}
// r = v_rcp_f32(s): the product with r gives the code of the division (to
// within one unit) except near a rounding tie, where the division decides:
// |fl(a r) - a / s| <= 2^-22 |a / s| < 2^-17 for quotients up to 32, and both
// round alike where a r lies more than 2^-16 from the tie.
__device__ __forceinline__ uint32_t q4_code(float w, float s, float b, float r) {
  const float a = w - b;
  float y = a * r;
  if (!(fabsf(y) < 32.0f && fabsf(__builtin_amdgcn_fractf(y) - 0.5f) > 0x1p-16f)) y = a / s;
  y = rintf(y);
  y = y > 0.0f ? y : 0.0f;  // (s = 0: 0/0, inf and NaN)
  y = y < 15.0f ? y : 15.0f;
  return s > 0.0f ? (uint32_t)y : 0u;
}
// Eight elements (words of pairs of DT) of a group that eight lanes share (x, x ^ 1,
// x ^ 2 and the half row's mirror): the group's metadata word and the codes, a byte
// each.  Two forms of the same codes, the first for groups without infinities, NaN
// and numbers past the fp16 range: rint(a / s) is taken from a r + 1.5 2^23, whose
// low bits are the integer, and stands where what it leaves, a - n s, stays below
// half a step by 2^-18 (the product with r is off by less than 2^-18 of a step);
// ties, near ties and s = 0 take q4_code.
__device__ __forceinline__ float q4_min3(float a, float b, float c) {
  float r;
  asm("v_min3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float q4_max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
__device__ __forceinline__ float q4_max3_abs(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
typedef unsigned short ushort2_t __attribute__((ext_vector_type(2)));
template <int DT>
__device__ __forceinline__ uint32_t q4_codes8(const uint32_t (&w4)[4], uint32_t &lo4, uint32_t &hi4) {
  ushort2_t m2 = __builtin_bit_cast(ushort2_t, w4[0] & 0x7fff7fffu);
#pragma unroll
  for (int k = 1; k < 4; ++k) m2 = __builtin_elementwise_max(m2, __builtin_bit_cast(ushort2_t, w4[k] & 0x7fff7fffu));
  const int top = max((int)m2[0], (int)m2[1]);
  float w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = elem_to_f32<DT>((uint16_t)(w4[e >> 1] >> (16 * (e & 1))));
  bool nan = false;
  if (__any(top >= (DT == DT_BF16 ? 0x4780 : 0x7c00))) {  // 65536 in bf16, infinity in fp16
    const int lane = threadIdx.x & 63;
    nan = ((__ballot(top > (DT == DT_BF16 ? 0x7f80 : 0x7c00)) >> (lane & 56)) & 0xffull) != 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = w[e] != w[e] ? 0.0f : q4_limit<DT>(w[e]);  // (the group's codes do not matter then)
  }
  float lo = q4_min3(q4_min3(w[0], w[1], w[2]), w[3], w[4]), hi = q4_max3(q4_max3(w[0], w[1], w[2]), w[3], w[4]);
  lo = q4_min3(q4_min3(lo, w[5], w[6]), w[7], dpp_f32<0xB1>(q4_min3(q4_min3(lo, w[5], w[6]), w[7], w[7])));
  hi = q4_max3(q4_max3(hi, w[5], w[6]), w[7], dpp_f32<0xB1>(q4_max3(q4_max3(hi, w[5], w[6]), w[7], w[7])));
  lo = fminf(lo, dpp_f32<0x4E>(lo));   // quad_perm [2,3,0,1]
  hi = fmaxf(hi, dpp_f32<0x4E>(hi));
  lo = fminf(lo, dpp_f32<0x141>(lo));  // row_half_mirror
  hi = fmaxf(hi, dpp_f32<0x141>(hi));
  float s, b;
  const uint32_t meta = q4_params(lo, hi, nan, s, b);
  const float r = __builtin_amdgcn_rcpf(s);
  constexpr float M = 12582912.0f;
  float t[8], off = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    float d[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const float a = w[e + f] - b;
      t[e + f] = __builtin_fmaf(a, r, M);
      d[f] = __builtin_fmaf(M - t[e + f], s, a);
    }
    off = q4_max3_abs(off, d[0], d[1]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = __builtin_amdgcn_fmed3f(t[e], M, M + 15.0f);
  // (a NaN among the t has one among the d, which v_max3 may pass over: s = 0 is
  // asked for by itself)
  if (__any(!(off < s * (0.5f - 0x1p-18f)) || !(s > 0.0f))) {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = M + (float)q4_code(w[e], s, b, r);
  }
  uint32_t u[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) u[e] = __builtin_bit_cast(uint32_t, t[e]);
  auto four = [&](int e) -> uint32_t {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[e + 3], u[e + 2], 0x0c0c0400u),
                                 __builtin_amdgcn_perm(u[e + 1], u[e], 0x0c0c0400u), 0x05040100u);
  };
  lo4 = four(0);
  hi4 = four(4);
  return meta;
}
// the K word of eight codes
__device__ __forceinline__ uint32_t q4_k_pack(uint32_t lo4, uint32_t hi4) {
  return __builtin_amdgcn_perm(hi4, lo4, 0x05010400u) | (__builtin_amdgcn_perm(hi4, lo4, 0x07030602u) << 4);
}
// The value a code stands for, as the caches are read back: fp16, within its
// range.
__device__ __forceinline__ uint32_t q4_value_bits(uint32_t c, float s, float b) {
  const float x = __builtin_fmaf((float)c, s, b);  // (the product is exact)
  return f32_to_f16_bits(x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x);
}

// One slice of a row of K or V (lane: E = D/64 consecutive dims, fp32) as codes:
// the wave's form.
template <int D, int DT>
__device__ __forceinline__ uint32_t q4_quantize_row(const float (&x)[D / 64], uint32_t (&code)[D / 64]) {
  constexpr int E = D / 64, LPG = 64 / E;
  float w[E], lo = INFINITY, hi = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    nan |= x[e] != x[e];
    w[e] = q4_limit<DT>(x[e]);
    lo = fminf(lo, w[e]);
    hi = fmaxf(hi, w[e]);
  }
  lo = wave_min_range<1, LPG / 2>(lo);
  hi = wave_max_range<1, LPG / 2>(hi);
  const uint64_t in_group = (LPG == 64 ? ~0ull : ((1ull << (LPG & 63)) - 1)) << ((threadIdx.x & 63) / LPG * LPG);
  const bool any = (__ballot(nan) & in_group) != 0;
  float s, b;
  const uint32_t meta = q4_params(lo, hi, any, s, b);
  const float r = __builtin_amdgcn_rcpf(s);
#pragma unroll
  for (int e = 0; e < E; ++e) code[e] = q4_code(w[e], s, b, r);
  return meta;
}

// ----------------------------------------------------------- matrix operands
// Codes become fp16 numbers of their own exponent (a subnormal 2^-24 c would be
// exact as well, but the matrix instructions align their sums to the operands'
// exponent fields: with subnormal operands a sum over 2000 tokens was off by 1e-4
// of the result, so by 2e-7).

// Centred as well, c - 8: sums of codes of one sign outgrow the result they
// leave.  Two instructions a pair, (1024 + c) - 1032 of the low nibbles of a
// word's halves, (1024 + 16 c) / 16 - 72 of the second nibbles.  `magic` is
// q4_magic() in a vector register: v_and_or_b32 takes one scalar operand and no
// literal (with both constants known to the compiler it becomes two
// instructions).
__device__ __forceinline__ uint32_t q4_magic() {
  uint32_t m;
  asm("v_mov_b32 %0, 0x64006400" : "=v"(m));
  return m;
}
__device__ __forceinline__ uint32_t q4_and_or(uint32_t w, uint32_t mask, uint32_t magic) {
  uint32_t r;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(mask), "v"(magic));
  return r;
}
__device__ __forceinline__ uint32_t q4_centred_lo(uint32_t w, uint32_t magic) {
  return h2_as_u32(u32_as_h2(q4_and_or(w, 0x000f000fu, magic)) + half2_t{(_Float16)-1032.0f, (_Float16)-1032.0f});
}
__device__ __forceinline__ uint32_t q4_centred_hi(uint32_t w, uint32_t magic) {
  const half2_t r = half2_t{(_Float16)0.0625f, (_Float16)0.0625f}, m = half2_t{(_Float16)-72.0f, (_Float16)-72.0f};
  return h2_as_u32(__builtin_elementwise_fma(u32_as_h2(q4_and_or(w, 0x00f000f0u, magic)), r, m));
}
// The eight codes of a K word in dim order.
__device__ __forceinline__ half8_t q4_k_operand(uint32_t w, uint32_t magic) {
  const uint32_t u = w >> 8;
  return __builtin_bit_cast(half8_t, uint4{q4_centred_lo(w, magic), q4_centred_hi(w, magic), q4_centred_lo(u, magic),
                                           q4_centred_hi(u, magic)});
}
// The same as they come, 1024 + c in pairs 0 and 2, 1024 + 16 c in pairs 1 and 3.
__device__ __forceinline__ half8_t q4_k_operand_raw(uint32_t w, uint32_t magic) {
  const uint32_t u = w >> 8;
  return __builtin_bit_cast(half8_t, uint4{q4_and_or(w, 0x000f000fu, magic), q4_and_or(w, 0x00f000f0u, magic),
                                           q4_and_or(u, 0x000f000fu, magic), q4_and_or(u, 0x00f000f0u, magic)});
}
// The eight tokens' codes of two V words: low nibbles (tile 2 j), second nibbles
// (tile 2 j + 1).
__device__ __forceinline__ void q4_v_operands(uint32_t w0, uint32_t w1, uint32_t magic, half8_t &lo, half8_t &hi) {
  const uint32_t u0 = w0 >> 8, u1 = w1 >> 8;
  lo = __builtin_bit_cast(half8_t, uint4{q4_centred_lo(w0, magic), q4_centred_lo(u0, magic), q4_centred_lo(w1, magic),
                                         q4_centred_lo(u1, magic)});
  hi = __builtin_bit_cast(half8_t, uint4{q4_centred_hi(w0, magic), q4_centred_hi(u0, magic), q4_centred_hi(w1, magic),
                                         q4_centred_hi(u1, magic)});
}

// Eight centred codes as the values they stand for, s (c - 8) + z rounded to fp16.
__device__ __forceinline__ half8_t q4_scaled(half8_t c, half8_t s, half8_t z) { return __builtin_elementwise_fma(c, s, z); }
__device__ __forceinline__ half8_t q4_join(half2_t a, half2_t b, half2_t c, half2_t d) {
  return __builtin_bit_cast(half8_t, uint4{h2_as_u32(a), h2_as_u32(b), h2_as_u32(c), h2_as_u32(d)});
}

}  // namespace krill
