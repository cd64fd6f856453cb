// latent_common.h - what the latent-attention kernels share: the 16-bit element types,
// their matrix products and the sizes of a cache row.
#pragma once

#include "ck_common.h"

namespace ck {
namespace lat {

constexpr int kR = 512;          // latent dims: the values, and the first part of every key
constexpr int kP = 64;           // rotated key dims
constexpr int kRow = kR + kP;    // a cache row
constexpr int kRowBytes = kRow * 2;
constexpr int kPage = 128;       // tokens per page
constexpr int kPageBytes = kPage * kRowBytes;

// CK_DTYPE_BF16 or CK_DTYPE_F16: conversions (round to nearest even) and the products
// D = A B + C of 16-bit operands with fp32 sums, fragments as raw 16 bytes per lane.
template <int DT>
struct Elem;

template <>
struct Elem<CK_DTYPE_BF16> {
    static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_bf16x2(lo, hi); }
    static __device__ __forceinline__ float lo(uint32_t w) { return bf16_lo(w); }
    static __device__ __forceinline__ float hi(uint32_t w) { return bf16_hi(w); }
    static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                       0, 0, 0);
    }
    // Probabilities enter the second product as 2^kBias p: bf16 has fp32's exponents.
    static constexpr float kBias = 0.f;
};

template <>
struct Elem<CK_DTYPE_F16> {
    typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 f16x8;
    static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
        typedef _Float16 f16x2v __attribute__((ext_vector_type(2)));
        const f16x2v v = {(_Float16)lo, (_Float16)hi};
        return __builtin_bit_cast(uint32_t, v);
    }
    static __device__ __forceinline__ float lo(uint32_t w) {
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xFFFFu));
    }
    static __device__ __forceinline__ float hi(uint32_t w) {
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
    }
    static __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                      0, 0);
    }
    // fp16's normal range ends at 2^-14: 2^7 p keeps all bits of p down to 2^-21, and with
    // the running maximum at most 2^8 behind (kSlack) stays at or below 2^15 < 65504.
    static constexpr float kBias = 7.f;
};

// A value that is the same in all lanes, into scalar registers (divisions leave it in vector ones).
__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t scalar(int64_t x) {
    return ((int64_t)scalar((int)(x >> 32)) << 32) | (uint32_t)scalar((int)x);
}

// Sums of x over the lanes up to each, none above `most`.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x, uint32_t most) {
    auto add = [&](uint32_t y) { x = min(x + y, most); };
    add(__builtin_amdgcn_update_dpp(0u, x, 0x111, 0xf, 0xf, false));  // from 1, 2, 4, 8 lanes below in the row
    add(__builtin_amdgcn_update_dpp(0u, x, 0x112, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0u, x, 0x114, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0u, x, 0x118, 0xf, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0u, x, 0x142, 0xa, 0xf, false));  // the row before's last, in rows 1 and 3
    add(__builtin_amdgcn_update_dpp(0u, x, 0x143, 0xc, 0xf, false));  // lane 31's, in the upper half
    return x;
}

// The largest of three; a NaN among them is passed over. One instruction, and the compiler's:
// inside inline assembly it would not keep the distance from the product that made x, y or z.
__device__ __forceinline__ float max3(float x, float y, float z) { return fmaxf(fmaxf(x, y), z); }

// 16 bytes per lane from r at voff + soff to LDS at base + IMM + 16 * lane, as dma16_buf, with
// the place in two scalar instructions: they issue in the shadow of a product, where a vector
// instruction and its trip to the scalar registers would hold the wave up.
template <int IMM>
__device__ __forceinline__ void dma_tile(const ck_rsrc_t &r, int voff, int soff, int base) {
    asm volatile("s_add_i32 m0, %0, %c1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds"
                 :
                 : "s"(base), "i"(IMM), "v"(voff), "s"(r), "s"(soff)
                 : "memory", "m0", "scc");
}

}  // namespace lat
}  // namespace ck
