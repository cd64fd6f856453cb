// kv4_common.h - the layout of a 4-bit K/V pool, as the kernels that write and read it share it.
//
// A pool is [num_blocks][kv_heads] pages of 128 tokens: two units of 64 tokens each, 8704 bytes that lie
// together. Keys and values are e2m1 codes (sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2,
// 3, 4, 6), 32 neighbouring dims of a token share a scale 2^(e - 127), e one byte (255: not a
// number). A unit holds, for its token t = 32 h + 8 g + t8 (t8 = 4 j + r):
//   0    keys' codes    [64 t][64]: byte i has dims 2 i (low half) and 2 i + 1
//   4096 values' codes  [4 q][4 g][16 n][2 h][8 t8]: dims 8 n + 2 q and the next
//   8192 keys' scales   [4 groups][16: 4 g + r][4: 2 h + j]
//   8448 values' scales [4 groups][4 g][2 h][8 t8]
// The order is that of the decode kernels' operands: a lane takes 16 bytes of a token's keys (one
// group), or of its values the dims 8 n .. + 7 (one group's) of 16 tokens.
#pragma once

#include "ck_common.h"

namespace ck {
namespace kv4 {

constexpr int kD = 128;      // head dim
constexpr int kPage = 128;   // tokens per page
constexpr int kUnit = 64;    // tokens per unit
constexpr int kVAt = kUnit * kD / 2;
constexpr int kKsAt = 2 * kVAt;
constexpr int kVsAt = kKsAt + kUnit * 4;
constexpr int kUnitBytes = kVsAt + kUnit * 4;
constexpr int kPageBytes = 2 * kUnitBytes;
static_assert(kUnitBytes == 8704, "68 cache lines");

// Scale bytes that are written: dequantised values (0.5 to 6 times the scale) then are normal
// numbers of fp32 and bf16, and finite.
constexpr int kLowest = 8, kHighest = 252, kBad = 255;

// Two codes (byte B of w) times a scale, of which the conversion takes the exponent field only:
// sign and mantissa may hold anything.
template <int B>
__device__ __forceinline__ uint32_t pair_bf16(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, B));
}
template <int B>
__device__ __forceinline__ uint32_t pair_f16(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, B));
}
// Byte B of four scales, in the exponent field (the other bits hold what was beside it).
template <int B>
__device__ __forceinline__ float scale_of(uint32_t w) {
    if constexpr (B == 3) return __uint_as_float(w >> 1);
    else return __uint_as_float(w << (23 - 8 * B));
}

}  // namespace kv4
}  // namespace ck
