// kv4_cache.hip - writes tokens into the pages of a 4-bit K/V pool and reads them back (gfx950).
//
// Write, per token, kv head and group of 32 dims (x the 16-bit values):
//   e = exponent of max |x|, one more where its mantissa exceeds 1.75, minus 2 (so that the largest
//       is in (3.5, 7] units of 2^(e - 127)), kept within [8, 252]; 255 if some x is not finite
//   code = x / 2^(e - 127), rounded to the nearest e2m1 value, ties to the even code, at most 6
// Quotients by a power of two are exact, so the codes are the same bits however they are computed. Against
// the plain exponent (largest in [4, 8), cut to 6) normal values lose 19.0 dB instead of 18.8.
//
// Memory-bound: 512 B of 16-bit rows and 136 B of codes and scales a token and head. 16 lanes take a row of 128
// dims, 8 neighbouring ones each: a group's maximum is two exchanges within 4 lanes, and a lane's 8 codes are one word.
// A token's value codes lie in single bytes, 16 apart, so that in the form for few tokens a lane moves bytes;
// in the form for many, 16 lanes take eight tokens, and where these have eight slots in a row (as a prompt's
// have) their bytes lie together and move as words of 4, 8 and 16 bytes.
// Kernels alone: 64 tokens of 8 heads 2.9 us each way (a launch); 8192 tokens of 8 heads (42 MB) 9.6 us written, 9.4
// read; 65536 tokens of 8 heads read (340 MB) 67.8 us, 5.0 TB/s, what a copy reaches (one token at a time: 92).
#include "kv4_common.h"

namespace ck {
namespace {

using namespace kv4;

constexpr int kThreads = 256;
constexpr int kRowsPerBlock = kThreads / 16;  // tokens of one kv head

// Places of a token in its unit: slot s is page s / 128, token s % 128.
struct Place {
    int64_t unit;  // bytes
    int k, v, ks, vs;
};
__device__ __forceinline__ Place place_of(int64_t slot, int head, int64_t kv_heads, int l16) {
    const int t = (int)(slot & (kUnit - 1)), h = t >> 5, g = (t >> 3) & 3, t8 = t & 7;
    Place p;
    p.unit = (((slot >> 7) * kv_heads + head) * 2 + ((slot >> 6) & 1)) * kUnitBytes;
    p.k = t * 64 + l16 * 4;
    p.v = kVAt + g * 256 + l16 * 16 + h * 8 + t8;  // + 1024 q
    p.ks = kKsAt + (l16 >> 2) * 64 + (g * 4 + (t8 & 3)) * 4 + h * 2 + (t8 >> 2);
    p.vs = kVsAt + (l16 >> 2) * 64 + g * 16 + h * 8 + t8;
    return p;
}

struct WriteArgs {
    const uint16_t *k, *v;
    int64_t k_token, k_head, v_token, v_head;  // element strides
    const int64_t *slots;
    uint8_t *cache;
    int64_t tokens, kv_heads, num_slots;
};

// 8 values of a lane -> a word of codes; e: the scale byte of their group (4 lanes).
template <int DT>
__device__ __forceinline__ uint32_t quantise(u32x4 w, int &e) {
    using E = Elem<DT>;
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = E::lo(w[i]);
        x[2 * i + 1] = E::hi(w[i]);
    }
    // magnitudes as integers: infinities and NaN are the largest
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
    most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0xb1, 0xf, 0xf, false));  // lane ^ 1
    most = max(most, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)most, 0x4e, 0xf, 0xf, false));  // lane ^ 2
    e = min(max((int)((most + 0x1fffffu) >> 23) - 2, kLowest), kHighest);
    const float scale = __uint_as_float((uint32_t)e << 23);
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], scale, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], scale, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], scale, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], scale, 3);
    if (most >= 0x7f800000u) {
        e = kBad;
        c = 0;
    }
    return c;
}

// Writes one token's row: kc, vc the lane's codes, ke, ve its group's scales.
__device__ __forceinline__ void put_token(const WriteArgs &a, int64_t slot, int head, int l16, uint32_t kc, uint32_t vc, int ke, int ve) {
    const Place p = place_of(slot, head, a.kv_heads, l16);
    uint8_t *unit = a.cache + p.unit;
    *reinterpret_cast<uint32_t *>(unit + p.k) = kc;
#pragma unroll
    for (int q = 0; q < 4; ++q) unit[p.v + 1024 * q] = (uint8_t)(vc >> (8 * q));
    if ((l16 & 3) == 0) {
        unit[p.ks] = (uint8_t)ke;
        unit[p.vs] = (uint8_t)ve;
    }
}

template <int DT>
__global__ __launch_bounds__(kThreads) void kv4_write_kernel(WriteArgs a) {
    const int l16 = threadIdx.x & 15, head = blockIdx.y;
    const int64_t t = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 4);
    if (t >= a.tokens) return;
    const u32x4 kw = *reinterpret_cast<const u32x4 *>(a.k + t * a.k_token + head * a.k_head + 8 * l16);
    const u32x4 vw = *reinterpret_cast<const u32x4 *>(a.v + t * a.v_token + head * a.v_head + 8 * l16);
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.num_slots) return;  // the same for the 16 lanes of a row
    int ke, ve;
    const uint32_t kc = quantise<DT>(kw, ke), vc = quantise<DT>(vw, ve);
    put_token(a, slot, head, l16, kc, vc, ke, ve);
}

// ---- many tokens: 16 lanes take 8, whose bytes lie together where their slots are eight in a row ---------------
// The eight slots of a group of lanes' tokens, tokens t0 .. + 7 (some may lie outside the call): base is the first
// token's slot if they are neighbours from a multiple of 8 on, all in the call and in the pool; else -1, and
// each lane holds the slot of token t0 + its place in 8.
struct Eight {
    int64_t t0, base, slot;
};
__device__ __forceinline__ Eight eight_slots(const int64_t *slots, int64_t tokens, int64_t num_slots, int64_t group, int l16) {
    Eight e;
    // groups begin where the first token's neighbours do: a prompt's tokens then meet the multiples of 8
    e.t0 = group * 8 - (slots[0] & 7);
    const int64_t t = e.t0 + (l16 & 7);
    e.slot = t >= 0 && t < tokens ? slots[t] : -1;
    const int64_t first = __shfl(e.slot, 0, 8);
    const bool ok = e.slot >= 0 && e.slot < num_slots && e.slot == first + (l16 & 7) && (first & 7) == 0;
    const uint64_t all = __builtin_amdgcn_ballot_w64(ok);
    const int at = threadIdx.x & 48;
    e.base = ((all >> at) & 0xffff) == 0xffff ? first : -1;
    return e;
}
// Byte q of each of four words.
template <int Q>
__device__ __forceinline__ uint32_t bytes_of(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t x = __builtin_amdgcn_perm(b, a, 0x0c0c0400 + 0x0101 * Q), y = __builtin_amdgcn_perm(d, c, 0x0c0c0400 + 0x0101 * Q);
    return x | y << 16;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void kv4_write8_kernel(WriteArgs a) {
    const int l16 = threadIdx.x & 15, head = blockIdx.y;
    const Eight e = eight_slots(a.slots, a.tokens, a.num_slots, (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 4), l16);
    if (e.t0 >= a.tokens) return;
    u32x4 kw[8], vw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t t = min(max(e.t0 + i, (int64_t)0), a.tokens - 1);
        kw[i] = *reinterpret_cast<const u32x4 *>(a.k + t * a.k_token + head * a.k_head + 8 * l16);
        vw[i] = *reinterpret_cast<const u32x4 *>(a.v + t * a.v_token + head * a.v_head + 8 * l16);
    }
    uint32_t kc[8], vc[8];
    int ke[8], ve[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        kc[i] = quantise<DT>(kw[i], ke[i]);
        vc[i] = quantise<DT>(vw[i], ve[i]);
    }
    if (e.base >= 0) {
        const Place p = place_of(e.base, head, a.kv_heads, l16);
        uint8_t *unit = a.cache + p.unit;
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<uint32_t *>(unit + p.k + 64 * i) = kc[i];
        static_for<4>([&](auto q) __attribute__((always_inline)) {
            *reinterpret_cast<uint2 *>(unit + p.v + 1024 * q) =
                make_uint2(bytes_of<q>(vc[0], vc[1], vc[2], vc[3]), bytes_of<q>(vc[4], vc[5], vc[6], vc[7]));
        });
        if ((l16 & 3) == 0) {
#pragma unroll
            for (int r = 0; r < 4; ++r) *reinterpret_cast<uint16_t *>(unit + p.ks + 4 * r) = (uint16_t)(ke[r] | ke[4 + r] << 8);
            *reinterpret_cast<uint2 *>(unit + p.vs) =
                make_uint2(ve[0] | ve[1] << 8 | ve[2] << 16 | ve[3] << 24, ve[4] | ve[5] << 8 | ve[6] << 16 | ve[7] << 24);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t slot = __shfl(e.slot, i, 8);
            if (slot >= 0 && slot < a.num_slots) put_token(a, slot, head, l16, kc[i], vc[i], ke[i], ve[i]);
        }
    }
}

struct ReadArgs {
    const uint8_t *cache;
    const int64_t *slots;
    uint16_t *k, *v;  // [tokens, kv_heads, 128]
    int64_t tokens, kv_heads, num_slots;
};

// A word of codes times their scale, 8 values of 16 bits, rounded once.
template <int DT>
__device__ __forceinline__ u32x4 dequantise(uint32_t w, float scale) {
    if constexpr (DT == CK_DTYPE_BF16) {
        return u32x4{pair_bf16<0>(w, scale), pair_bf16<1>(w, scale), pair_bf16<2>(w, scale), pair_bf16<3>(w, scale)};
    } else {
        const auto x0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
        const auto x1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
        const auto x2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
        const auto x3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
        using E = Elem<DT>;
        return u32x4{E::pack2(x0[0], x0[1]), E::pack2(x1[0], x1[1]), E::pack2(x2[0], x2[1]), E::pack2(x3[0], x3[1])};
    }
}

// Reads one token's row and writes it out.
template <int DT>
__device__ __forceinline__ void get_token(const ReadArgs &a, int64_t t, int64_t slot, int head, int l16) {
    u32x4 kw = {0, 0, 0, 0}, vw = {0, 0, 0, 0};
    if (slot >= 0 && slot < a.num_slots) {
        const Place p = place_of(slot, head, a.kv_heads, l16);
        const uint8_t *unit = a.cache + p.unit;
        const uint32_t kc = *reinterpret_cast<const uint32_t *>(unit + p.k);
        uint32_t vc = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) vc |= (uint32_t)unit[p.v + 1024 * q] << (8 * q);
        kw = dequantise<DT>(kc, scale_of<0>(unit[p.ks]));
        vw = dequantise<DT>(vc, scale_of<0>(unit[p.vs]));
    }
    const int64_t at = (t * a.kv_heads + head) * kD + 8 * l16;
    *reinterpret_cast<u32x4 *>(a.k + at) = kw;
    *reinterpret_cast<u32x4 *>(a.v + at) = vw;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(ReadArgs a) {
    const int64_t t = (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 4);
    if (t < a.tokens) get_token<DT>(a, t, a.slots[t], blockIdx.y, threadIdx.x & 15);
}

template <int DT>
__global__ __launch_bounds__(kThreads) void kv4_read8_kernel(ReadArgs a) {
    const int l16 = threadIdx.x & 15, head = blockIdx.y;
    const Eight e = eight_slots(a.slots, a.tokens, a.num_slots, (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 4), l16);
    if (e.t0 >= a.tokens) return;
    if (e.base >= 0) {
        const Place p = place_of(e.base, head, a.kv_heads, l16);
        const uint8_t *unit = a.cache + p.unit;
        uint32_t kc[8];
        uint2 vq[4];
#pragma unroll
        for (int i = 0; i < 8; ++i) kc[i] = *reinterpret_cast<const uint32_t *>(unit + p.k + 64 * i);
#pragma unroll
        for (int q = 0; q < 4; ++q) vq[q] = *reinterpret_cast<const uint2 *>(unit + p.v + 1024 * q);
        const u32x4 ks = *reinterpret_cast<const u32x4 *>(unit + (p.ks & ~15));  // [r][h][j]
        const uint2 vs = *reinterpret_cast<const uint2 *>(unit + p.vs);
        const int h = (p.ks >> 1) & 1;
        const int64_t at = (e.t0 * a.kv_heads + head) * kD + 8 * l16, step = a.kv_heads * kD;
        static_for<8>([&](auto i) __attribute__((always_inline)) {
            constexpr int I = i, J = I >> 2, R = I & 3;
            const uint32_t k2 = ks[R] >> (16 * h);  // bytes j = 0, 1
            const uint32_t v4 = J ? vs.y : vs.x;
            *reinterpret_cast<u32x4 *>(a.k + at + I * step) = dequantise<DT>(kc[I], scale_of<J>(k2));
            const uint32_t vc = bytes_of<R>(J ? vq[0].y : vq[0].x, J ? vq[1].y : vq[1].x, J ? vq[2].y : vq[2].x, J ? vq[3].y : vq[3].x);
            *reinterpret_cast<u32x4 *>(a.v + at + I * step) = dequantise<DT>(vc, scale_of<R>(v4));
        });
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t t = e.t0 + i, slot = __shfl(e.slot, i, 8);
            if (t >= 0 && t < a.tokens) get_token<DT>(a, t, slot, head, l16);
        }
    }
}

// Rows (tokens times kv heads) from which 16 lanes take eight tokens. us a call, one / eight, of a prompt's slots: 16384 rows
// write 4.2 / 5.0, read 4.4 / 4.7; 32768 6.1 / 6.2, 6.4 / 5.9; 49152 8.4 / 7.5, 8.5 / 7.0; 131072 20.8 / 16.0,
// 17.7 / 14.3; 524288 79 / 69, 96 / 77. Slots in no order, which the host cannot tell from a prompt's, cost eight more, of
// 8 kv heads: 49152 12.7 / 14.4, 10.1 / 10.4; 65536 15.9 / 19.0, 12.9 / 16.1; 131072 30 / 32, 24 / 30; 262144 63 / 65, 46 / 60;
// 524288 154 / 169, 103 / 120. Calls of so many tokens are prompts; a step's tokens, in no order, are fewer.
constexpr int64_t kManyRows = 49152;
constexpr int64_t kMostHeads = 1 << 10, kMostStride = 1 << 28;

// The kernel of a token for 16 lanes, or that of eight.
template <class K, class A>
void launch(K one, K eight, const A &a, hipStream_t s) {
    const bool many = a.tokens * a.kv_heads >= kManyRows;
    // eight: one group more, as they need not begin with the first token
    const int64_t groups = many ? (a.tokens + 6) / 8 + 1 : a.tokens;
    const dim3 grid((unsigned)((groups - 1) / kRowsPerBlock + 1), (unsigned)a.kv_heads);
    hipLaunchKernelGGL(many ? eight : one, grid, dim3(kThreads), 0, s, a);
}

int check_pool(int64_t num_blocks, int64_t kv_heads, int64_t tokens) {
    if (num_blocks < 0 || num_blocks > ((int64_t)1 << 31) || kv_heads < 1 || kv_heads > kMostHeads || tokens < 0)
        return CK_E_INVALID_ARG;
    if (!grid_fits(tokens / kRowsPerBlock + 1, kThreads)) return CK_E_INVALID_ARG;
    return CK_OK;
}

}  // namespace
}  // namespace ck

using namespace ck;

extern "C" int ck_kv4_cache_write(const void *k, int64_t k_token_stride, int64_t k_head_stride, const void *v,
                                  int64_t v_token_stride, int64_t v_head_stride, const int64_t *slots, void *cache,
                                  int64_t num_blocks, int64_t tokens, int64_t kv_heads, int dtype, void *stream) {
    if (dtype != CK_DTYPE_BF16 && dtype != CK_DTYPE_F16) return CK_E_UNSUPPORTED;
    int rc = check_pool(num_blocks, kv_heads, tokens);
    if (rc != CK_OK) return rc;
    for (int64_t s : {k_token_stride, k_head_stride, v_token_stride, v_head_stride})
        if (s < 0 || s % 8 != 0 || s > kMostStride) return CK_E_INVALID_ARG;
    if (tokens == 0 || num_blocks == 0) return CK_OK;
    if (!k || !v || !slots || !cache) return CK_E_NULL_PTR;
    if (!aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(slots, 8) || !aligned_to(cache, 16))
        return CK_E_INVALID_ARG;
    WriteArgs a{static_cast<const uint16_t *>(k), static_cast<const uint16_t *>(v), k_token_stride, k_head_stride,
                v_token_stride, v_head_stride, slots, static_cast<uint8_t *>(cache), tokens, kv_heads,
                num_blocks * kv4::kPage};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == CK_DTYPE_BF16) launch(kv4_write_kernel<CK_DTYPE_BF16>, kv4_write8_kernel<CK_DTYPE_BF16>, a, s);
    else launch(kv4_write_kernel<CK_DTYPE_F16>, kv4_write8_kernel<CK_DTYPE_F16>, a, s);
    CK_RETURN_LAUNCH();
}

extern "C" int ck_kv4_cache_read(const void *cache, const int64_t *slots, int64_t num_blocks, int64_t tokens,
                                 int64_t kv_heads, int dtype, void *k, void *v, void *stream) {
    if (dtype != CK_DTYPE_BF16 && dtype != CK_DTYPE_F16) return CK_E_UNSUPPORTED;
    int rc = check_pool(num_blocks, kv_heads, tokens);
    if (rc != CK_OK) return rc;
    if (tokens == 0) return CK_OK;
    if (!slots || !k || !v || (num_blocks > 0 && !cache)) return CK_E_NULL_PTR;
    if (!aligned_to(k, 16) || !aligned_to(v, 16) || !aligned_to(slots, 8) || !aligned_to(cache, 16))
        return CK_E_INVALID_ARG;
    ReadArgs a{static_cast<const uint8_t *>(cache), slots, static_cast<uint16_t *>(k), static_cast<uint16_t *>(v),
               tokens, kv_heads, num_blocks * kv4::kPage};
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == CK_DTYPE_BF16) launch(kv4_read_kernel<CK_DTYPE_BF16>, kv4_read8_kernel<CK_DTYPE_BF16>, a, s);
    else launch(kv4_read_kernel<CK_DTYPE_F16>, kv4_read8_kernel<CK_DTYPE_F16>, a, s);
    CK_RETURN_LAUNCH();
}
