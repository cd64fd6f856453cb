// latent_cache.hip - writes tokens into the pages of a latent cache (gfx950).
//
// Per token t with slot s = slots[t] (page s / 128, row s % 128), in fp32, rounded once:
//   c = kv[t, 0:512], r = kv[t, 512:576]
//   cache[s, 0:512]   = c * rsqrt(mean(c^2) + eps) * gamma
//   cache[s, 512:576] = the 32 pairs (a, b) of r as (a cos - b sin, a sin + b cos), cos and
//                       sin of positions[t]; pairs (2i, 2i + 1) or (i, i + 32)
// A token whose slot or position is outside the cache or the table is not written.
//
// Memory-bound: 1152 B in, 256 B of cos and sin, 1152 B out per token. One wave per token:
// lane l holds 8 latent values (one 16-byte load), the sum of squares is a 6-step
// butterfly, and lanes 0-7 also hold 8 rotated dims each. No load depends on another (the
// cos/sin row on positions[t] aside), so a token costs two memory round trips. The index loads are
// wave-uniform.
#include <cmath>

#include "latent_common.h"

namespace ck {
namespace {

using namespace lat;

struct WriteArgs {
    const uint16_t *kv;
    const uint16_t *gamma;
    const float *cos_sin;
    const int64_t *positions;
    const int64_t *slots;
    uint16_t *cache;
    int64_t tokens;
    int64_t kv_stride;  // elements
    int64_t max_pos;
    int64_t num_slots;
    float eps;
};

constexpr int kWavesPerGroup = 4;

template <int DT, bool INTERLEAVED>
__global__ __launch_bounds__(kWavesPerGroup * 64) void latent_cache_write_kernel(WriteArgs a) {
    using E = Elem<DT>;
    const int lane = threadIdx.x & 63;
    const int64_t t = (int64_t)blockIdx.x * kWavesPerGroup + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= a.tokens) return;
    const int64_t slot = a.slots[t], pos = a.positions[t];
    if (slot < 0 || slot >= a.num_slots || pos < 0 || pos >= a.max_pos) return;

    const uint16_t *src = a.kv + t * a.kv_stride;
    const u32x4 cw = *reinterpret_cast<const u32x4 *>(src + 8 * lane);
    const u32x4 gw = *reinterpret_cast<const u32x4 *>(a.gamma + 8 * lane);
    // rotated dims: lane l < 8 holds dims 8l .. 8l + 7, the lanes above repeat them
    const int rl = lane & 7;
    const u32x4 rw = *reinterpret_cast<const u32x4 *>(src + kR + 8 * rl);
    // interleaved: pairs 4 rl .. + 3; halves: pairs 8 (rl & 3) .. + 7
    constexpr int kPairs = INTERLEAVED ? 4 : 8;
    const float *cs = a.cos_sin + pos * kP + kPairs * (INTERLEAVED ? rl : rl & 3);
    f32x4 cv[kPairs / 4], sv[kPairs / 4];
#pragma unroll
    for (int i = 0; i < kPairs / 4; ++i) {
        cv[i] = *reinterpret_cast<const f32x4 *>(cs + 4 * i);
        sv[i] = *reinterpret_cast<const f32x4 *>(cs + kP / 2 + 4 * i);
    }

    float c[8], ss = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c[2 * i] = E::lo(cw[i]);
        c[2 * i + 1] = E::hi(cw[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(c[i], c[i], ss);
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) ss += __shfl_xor(ss, m);
    const float rstd = 1.0f / sqrtf(ss * (1.0f / kR) + a.eps);
    uint16_t *dst = a.cache + slot * kRow;
    u32x4 ow;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        ow[i] = E::pack2(c[2 * i] * rstd * E::lo(gw[i]), c[2 * i + 1] * rstd * E::hi(gw[i]));
    *reinterpret_cast<u32x4 *>(dst + 8 * lane) = ow;

    u32x4 rr;
    if constexpr (INTERLEAVED) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = E::lo(rw[i]), y = E::hi(rw[i]);
            rr[i] = E::pack2(x * cv[0][i] - y * sv[0][i], x * sv[0][i] + y * cv[0][i]);
        }
    } else {
        // dims i and i + 32 are a pair: lanes 0-3 hold the first, 4-7 the second
        const float sign = rl < 4 ? -1.f : 1.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t ow2 = __shfl_xor(rw[i], 4);
            float o[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int e = 2 * i + j;
                const float x = j ? E::hi(rw[i]) : E::lo(rw[i]);
                const float y = j ? E::hi(ow2) : E::lo(ow2);
                o[j] = x * cv[e / 4][e % 4] + sign * (y * sv[e / 4][e % 4]);
            }
            rr[i] = E::pack2(o[0], o[1]);
        }
    }
    if (lane < 8) *reinterpret_cast<u32x4 *>(dst + kR + 8 * lane) = rr;
}

}  // namespace
}  // namespace ck

using namespace ck;

extern "C" int ck_latent_cache_write(const void *kv, int64_t kv_stride, const void *gamma, const float *cos_sin,
                                     int64_t max_pos, const int64_t *positions, const int64_t *slots, void *cache,
                                     int64_t num_blocks, int64_t tokens, int dtype, float eps, int interleaved,
                                     void *stream) {
    if (dtype != CK_DTYPE_BF16 && dtype != CK_DTYPE_F16) return CK_E_UNSUPPORTED;
    if (tokens < 0 || num_blocks < 0 || max_pos < 0 || kv_stride < lat::kRow || kv_stride % 8 != 0)
        return CK_E_INVALID_ARG;
    if (!(eps > 0.f) || !std::isfinite(eps)) return CK_E_INVALID_ARG;
    if (num_blocks > ((int64_t)1 << 40) || max_pos > ((int64_t)1 << 40) || kv_stride > ((int64_t)1 << 28))
        return CK_E_INVALID_ARG;
    const int64_t groups = tokens / kWavesPerGroup + (tokens % kWavesPerGroup != 0);
    if (!grid_fits(groups, kWavesPerGroup * 64)) return CK_E_INVALID_ARG;
    if (tokens == 0 || num_blocks == 0) return CK_OK;
    if (!kv || !gamma || !cos_sin || !positions || !slots || !cache) return CK_E_NULL_PTR;
    if (!aligned_to(kv, 16) || !aligned_to(gamma, 16) || !aligned_to(cos_sin, 16) || !aligned_to(cache, 16) ||
        !aligned_to(positions, 8) || !aligned_to(slots, 8))
        return CK_E_INVALID_ARG;
    WriteArgs a{static_cast<const uint16_t *>(kv), static_cast<const uint16_t *>(gamma), cos_sin, positions, slots,
                static_cast<uint16_t *>(cache), tokens, kv_stride, max_pos, num_blocks * lat::kPage, eps};
    const dim3 grid((unsigned)groups), block(kWavesPerGroup * 64);
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == CK_DTYPE_BF16) {
        if (interleaved) hipLaunchKernelGGL((latent_cache_write_kernel<CK_DTYPE_BF16, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((latent_cache_write_kernel<CK_DTYPE_BF16, false>), grid, block, 0, s, a);
    } else {
        if (interleaved) hipLaunchKernelGGL((latent_cache_write_kernel<CK_DTYPE_F16, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((latent_cache_write_kernel<CK_DTYPE_F16, false>), grid, block, 0, s, a);
    }
    CK_RETURN_LAUNCH();
}
