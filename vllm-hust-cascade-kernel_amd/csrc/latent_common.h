// latent_common.h - what the latent-attention kernels share: the sizes of a cache row and a load to LDS.
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
