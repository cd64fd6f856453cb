// latent_prefill.hip - attention in the expanded form for packed prompts (gfx950).
//
// Query i, head h of request b (ql queries, kl keys):
//   s_j = scale (q[0:128] . k[j, h] + q[128:192] . kr[j]),  j < kl, j <= kl - ql + i if causal
//   o = sum_j softmax(s)_j v[j, h],  lse = log sum_j exp(s_j)
// Nothing seen: o = 0, lse = -inf; so are rows behind the last request.
//
// Bound by the matrix cores: 640 flops per (query, key) pair of a head, K and V read once
// per 256 queries. The form is that of the stage-1 kernel with a key of two parts:
// * A wave owns 32 queries of one head and every key they see, 8 waves a workgroup (256
//   queries; 4 and 128 for small calls). Q stays in registers (48), so does O (64).
// * 64-key tiles land in a ring of 3 slots by buffer -> LDS DMA: the head's keys (16 KB), the
//   rotated part all heads share (8 KB) and the values (16 KB), two tiles in flight. The
//   resources end with the request's last key, so nothing past it is read.
// * S^T = K Q^T (24 MFMAs a tile of 32x32x16) puts one query on a lane; P^T is in the operand's
//   place as it leaves; V^T comes through ds_read_b64_tr_b16 (16 MFMAs).
// * A query's reference point of the softmax moves only when a score passes it by 2^kSlack.
// * Row tiles of a request are dealt last first: under a causal mask those are the longest.
//   Tiles of one head run on one XCD, whose L2 then holds that head's K and V.
#include <cmath>

#include "latent_common.h"

namespace ck {
namespace {

using namespace lat;

typedef __attribute__((__vector_size__(2 * sizeof(unsigned)))) unsigned u32x2;

constexpr int kD = 128;            // a head's key part, and its value
constexpr int kQ = kD + kP;        // query row
constexpr int kTok = 64;           // keys per tile
constexpr int kKBytes = kTok * kD * 2;
constexpr int kRBytes = kTok * kP * 2;
constexpr int kStage = 2 * kKBytes + kRBytes;  // keys | rotated | values: 40 KB
constexpr int kSlots = 3;
constexpr int kLds = kSlots * kStage + 256;
constexpr float kSlack = 8.f;

struct PrefillArgs {
    const uint16_t *q;
    const uint16_t *k;
    const uint16_t *kr;
    const uint16_t *v;
    const int64_t *q_lens;
    const int64_t *kv_lens;
    int64_t k_ts, k_hs, kr_ts, v_ts, v_hs;  // element strides
    int64_t tokens;
    int64_t keys;
    int batch;
    int heads;
    int tiles;  // row tiles per head that the grid holds
    int causal;
    float scale_log2;
    uint16_t *out;
    float *lse;
};

// 16-byte chunk c of row r: keys and values (256-byte rows) and the rotated part (128-byte
// rows). Over 16 consecutive rows one chunk lies in 16 distinct bank groups, over 4
// consecutive rows a 64-byte group in 16.
__device__ __forceinline__ int swz(int r) { return ((r & 3) << 2) | ((r >> 2) & 3); }
__device__ __forceinline__ int kv_off(int r, int c) { return r * (kD * 2) + ((c ^ swz(r)) << 4); }
__device__ __forceinline__ int rope_off(int r, int c) { return r * (kP * 2) + ((c ^ ((r >> 1) & 7)) << 4); }

// Sum of x over the threads before this one, and over all (in *total); NW waves.
template <int NW>
__device__ __forceinline__ int64_t block_scan(int64_t x, CK_LDS int64_t *room, int64_t *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t incl = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t up = __shfl_up(incl, o);
        if (lane >= o) incl += up;
    }
    __syncthreads();
    if (lane == 63) room[wave] = incl;
    __syncthreads();
    int64_t before = incl - x, all = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
        if (i < wave) before += room[i];
        all += room[i];
    }
    *total = all;
    return before;
}

template <int DT, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2))) void latent_prefill_kernel(PrefillArgs a) {
    using E = Elem<DT>;
    constexpr int kRows = NW * 32;
    constexpr int kBlk = 16 / NW;   // 1-KB DMAs of the keys (and of the values) per wave and tile
    constexpr int kRBlk = 8 / NW;   // and of the rotated part
    constexpr int kDmas = 2 * kBlk + kRBlk;
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    CK_LDS char *smem = (CK_LDS char *)smem_raw;
    CK_LDS int64_t *room = (CK_LDS int64_t *)(smem + kSlots * kStage);  // [0, 8): scans; [8, 13): the tile

    const int tid = threadIdx.x;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int hh = lane >> 5, n32 = lane & 31;

    const uint32_t w = xcd_remap(blockIdx.x, gridDim.x);
    const int head = w / a.tiles;
    const int64_t tile = w % a.tiles;

    // ---- which request's rows ---------------------------------------------------------------
    // Thread t looks at requests [t per, t per + per); a pseudo request without keys follows
    // the last one and takes the rows left.
    auto len_of = [](const int64_t *lens, int b, int64_t most) {
        const int64_t n = lens[b];
        return n < 0 ? (int64_t)0 : n > most ? most : n;
    };
    const int per = (a.batch + NW * 64 - 1) / (NW * 64);
    const int b_lo = min(tid * per, a.batch), b_hi = min(b_lo + per, a.batch);
    int64_t ql_sum = 0, kl_sum = 0, q_all, k_all, t_all;
    for (int b = b_lo; b < b_hi; ++b) {
        ql_sum += len_of(a.q_lens, b, a.tokens);
        kl_sum += len_of(a.kv_lens, b, a.keys);
    }
    int64_t q_at = block_scan<NW>(ql_sum, room, &q_all), k_at = block_scan<NW>(kl_sum, room, &k_all);
    // rows [min(q_at, tokens), min(q_at + ql, tokens)): what passes the end is cut off
    auto cut = [](int64_t at, int64_t n, int64_t most) { return min(at + n, most) - min(at, most); };
    int64_t mine = 0;
    {
        int64_t at = q_at;
        for (int b = b_lo; b < b_hi; ++b) {
            const int64_t n = len_of(a.q_lens, b, a.tokens);
            mine += (cut(at, n, a.tokens) + kRows - 1) / kRows;
            at += n;
        }
    }
    int64_t t_at = block_scan<NW>(mine, room, &t_all);
    if (tile >= t_all) {
        if (tid == 0) {
            const int64_t from = min(q_all, a.tokens);
            room[8] = from;
            room[9] = a.tokens - from;
            room[10] = 0;
            room[11] = 0;
            room[12] = tile - t_all;
        }
    } else {
        for (int b = b_lo; b < b_hi; ++b) {
            const int64_t n = len_of(a.q_lens, b, a.tokens), m = len_of(a.kv_lens, b, a.keys);
            const int64_t rows = cut(q_at, n, a.tokens), nt = (rows + kRows - 1) / kRows;
            if (tile >= t_at && tile < t_at + nt) {
                room[8] = q_at;
                room[9] = rows;
                room[10] = min(k_at, a.keys);
                room[11] = cut(k_at, m, a.keys);
                room[12] = nt - 1 - (tile - t_at);
            }
            q_at += n;
            k_at += m;
            t_at += nt;
        }
    }
    __syncthreads();
    const int64_t q0 = room[8], k0 = room[10];
    const int ql = __builtin_amdgcn_readfirstlane((int)room[9]), kl = __builtin_amdgcn_readfirstlane((int)room[11]);
    const int row0 = __builtin_amdgcn_readfirstlane((int)room[12]) * kRows;
    if (row0 >= ql) return;  // the same in every thread

    const int wrow0 = row0 + wid * 32;
    const int i_q = wrow0 + n32;
    const bool row_valid = i_q < ql;
    const int64_t qrow = (q0 + i_q) * a.heads + head;
    // keys seen by this lane's query, by the wave's first and last, and by the workgroup's last
    auto seen = [&](int i) { return a.causal ? max(0, min(kl, kl - ql + 1 + i)) : kl; };
    const int limit = row_valid ? seen(i_q) : 0;
    const int w_last = min(wrow0 + 31, ql - 1);
    const int w_most = wrow0 < ql ? seen(w_last) : 0, w_least = seen(wrow0);
    const int most = seen(min(row0 + kRows - 1, ql - 1));
    const int ntiles = (most + kTok - 1) / kTok;

    u32x4 qf[12];
#pragma unroll
    for (int kk = 0; kk < 12; ++kk) {
        qf[kk] = u32x4{0, 0, 0, 0};
        if (row_valid) qf[kk] = *reinterpret_cast<const u32x4 *>(a.q + qrow * kQ + 16 * kk + 8 * hh);
    }

    // ---- DMA ----------------------------------------------------------------------------------
    // 1-KB block j of a wave: 4 rows of keys or values, 8 rows of the rotated part
    uint32_t k_dma[kBlk], v_dma[kBlk], r_dma[kRBlk];
#pragma unroll
    for (int j = 0; j < kBlk; ++j) {
        const int r = (wid * kBlk + j) * 4 + (lane >> 4), c = (lane & 15) ^ swz(r);
        k_dma[j] = (uint32_t)(r * a.k_ts + c * 8) * 2;
        v_dma[j] = (uint32_t)(r * a.v_ts + c * 8) * 2;
    }
#pragma unroll
    for (int j = 0; j < kRBlk; ++j) {
        const int r = (wid * kRBlk + j) * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        r_dma[j] = (uint32_t)(r * a.kr_ts + c * 8) * 2;
    }
    auto issue = [&](int t, int slot) {
        const int64_t at = k0 + (int64_t)t * kTok;
        const int n = min(kTok, kl - t * kTok);  // rows of the request in this tile
        const ck_rsrc_t rk = buf_rsrc(a.k + at * a.k_ts + head * a.k_hs, (uint32_t)((n - 1) * a.k_ts + kD) * 2);
        const ck_rsrc_t rr = buf_rsrc(a.kr + at * a.kr_ts, (uint32_t)((n - 1) * a.kr_ts + kP) * 2);
        const ck_rsrc_t rv = buf_rsrc(a.v + at * a.v_ts + head * a.v_hs, (uint32_t)((n - 1) * a.v_ts + kD) * 2);
        CK_LDS char *dst = smem + slot * kStage;
#pragma unroll
        for (int j = 0; j < kBlk; ++j) {
            dma16_buf(rk, (int)k_dma[j], 0, dst + (wid * kBlk + j) * 1024);
            dma16_buf(rv, (int)v_dma[j], 0, dst + kKBytes + kRBytes + (wid * kBlk + j) * 1024);
        }
#pragma unroll
        for (int j = 0; j < kRBlk; ++j) dma16_buf(rr, (int)r_dma[j], 0, dst + kKBytes + (wid * kRBlk + j) * 1024);
    };

    f32x16 oacc[4];
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[db][i] = 0.f;
    float m_run = -INFINITY, l_part = 0.f;

    const int trG = (lane >> 4) & 3, tr_row = (lane & 15) >> 2, tr_e4 = lane & 3;
    auto vt_off = [&](int s16, int db, int second) {
        const int t1 = 16 * s16 + 4 * (trG >> 1) + tr_row + 8 * second;
        const int d = 32 * db + 16 * (trG & 1) + 4 * tr_e4;
        return kv_off(t1, d >> 3) + (d & 7) * 2;
    };

    wait_vmcnt<0>();
    for (int t = 0; t < kSlots - 1 && t < ntiles; ++t) issue(t, t);
    int slot = 0;
    for (int t = 0; t < ntiles; ++t) {
        if (t + 1 < ntiles) wait_vmcnt<kDmas>();
        else wait_vmcnt<0>();
        const int nv = kl - t * kTok;  // rows of the request from here on
        CK_LDS char *kb = smem + slot * kStage, *rbuf = kb + kKBytes, *vb = rbuf + kRBytes;
        if (nv < kTok) {  // values past the request's end, in this wave's blocks: 0 * V must not be NaN
#pragma unroll
            for (int j = 0; j < kBlk; ++j)
                if ((wid * kBlk + j) * 4 + (lane >> 4) >= nv)
                    *reinterpret_cast<CK_LDS u32x4 *>(vb + (wid * kBlk + j) * 1024 + lane * 16) = u32x4{0, 0, 0, 0};
        }
        __syncthreads();  // tile t is in; every wave is done with tile t - 1, whose slot is next
        if (t + 2 < ntiles) issue(t + 2, slot == 0 ? 2 : slot - 1);
        slot = slot == 2 ? 0 : slot + 1;
        if (t * kTok >= w_most) continue;  // the wave's queries see none of it

        f32x16 sb[2];
        {
            const f32x16 zero16 = {};
            auto kfrag = [&](int f) {
                const int r = 32 * (f & 1) + n32, ks = f >> 1;
                return *reinterpret_cast<const CK_LDS u32x4 *>(ks < 8 ? kb + kv_off(r, 2 * ks + hh)
                                                                      : rbuf + rope_off(r, 2 * (ks - 8) + hh));
            };
            constexpr int kAhead = 4;
            u32x4 kfr[kAhead];
#pragma unroll
            for (int f = 0; f < kAhead; ++f) kfr[f] = kfrag(f);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int f = 0; f < 24; ++f) {
                sb[f & 1] = E::mfma32(kfr[f % kAhead], qf[f >> 1], f < 2 ? zero16 : sb[f & 1]);
                if (f + kAhead < 24) kfr[f % kAhead] = kfrag(f + kAhead);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (t * kTok + kTok > w_least) {
#pragma unroll
            for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int tok = t * kTok + 32 * q2 + (e & 3) + 8 * (e >> 2) + 4 * hh;
                    if (tok >= limit) sb[q2][e] = -INFINITY;
                }
        }
        float smax = -INFINITY;
#pragma unroll
        for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
            for (int e = 0; e < 16; ++e) smax = fmaxf(smax, sb[q2][e]);
        smax = max_xor32(smax) * a.scale_log2;
        const bool moves = smax > m_run + kSlack;
        if (__builtin_amdgcn_ballot_w64(moves)) {
            const float dm = moves ? exp2_fast(m_run - smax) : 1.f;
            if (moves) m_run = smax;
            l_part *= dm;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int e = 0; e < 16; ++e) oacc[db][e] *= dm;
        }
        const float sub = (m_run == -INFINITY ? 0.f : m_run) - E::kBias;
        float ls = 0.f;
        u32x4 pb[4];
#pragma unroll
        for (int q2 = 0; q2 < 2; ++q2) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float pv = exp2_fast(fmaf(sb[q2][e], a.scale_log2, -sub));
                sb[q2][e] = pv;
                ls += pv;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) pb[2 * q2 + (j >> 2)][j & 3] = E::pack2(sb[q2][2 * j], sb[q2][2 * j + 1]);
        }
        l_part += ls;
        // O^T += V^T P^T, V^T fragments read one 16-key group ahead
        {
            uint2 vlo[2][4], vhi[2][4];
#pragma unroll
            for (int db = 0; db < 4; ++db) {
                vlo[0][db] = lds_read_tr16(vb + vt_off(0, db, 0));
                vhi[0][db] = lds_read_tr16(vb + vt_off(0, db, 1));
            }
#pragma unroll
            for (int s16 = 0; s16 < 4; ++s16) {
                if (s16 + 1 < 4) {
#pragma unroll
                    for (int db = 0; db < 4; ++db) {
                        vlo[(s16 + 1) & 1][db] = lds_read_tr16(vb + vt_off(s16 + 1, db, 0));
                        vhi[(s16 + 1) & 1][db] = lds_read_tr16(vb + vt_off(s16 + 1, db, 1));
                    }
                }
#pragma unroll
                for (int db = 0; db < 4; ++db) {
                    const uint2 lo = vlo[s16 & 1][db], hi = vhi[s16 & 1][db];
                    oacc[db] = E::mfma32(u32x4{lo.x, lo.y, hi.x, hi.y}, pb[s16], oacc[db]);
                }
            }
        }
    }

    // ---- normalise, write whole rows through the idle ring ----------------------------------
    const float l_run = l_part + __shfl_xor(l_part, 32);
    __syncthreads();  // every wave is past its last ring read
    if (wrow0 >= ql) return;
    // l is 0 where nothing was seen (or every score was -inf)
    const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
    if (row_valid && hh == 0)
        a.lse[qrow] = l_run == 0.f ? -INFINITY : (m_run - E::kBias + __log2f(l_run)) * kLn2;
    CK_LDS char *slab = smem + wid * (32 * kD * 2);
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
            // dims 32 db + 8 c4 + 4 hh .. + 3
            const u32x2 o = {E::pack2(oacc[db][4 * c4] * inv, oacc[db][4 * c4 + 1] * inv),
                             E::pack2(oacc[db][4 * c4 + 2] * inv, oacc[db][4 * c4 + 3] * inv)};
            *reinterpret_cast<CK_LDS u32x2 *>(slab + n32 * 256 + (((4 * db + c4) ^ (n32 & 15)) << 4) + hh * 8) = o;
        }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int r = 4 * j + (lane >> 4), c = lane & 15;
        const u32x4 o = *reinterpret_cast<const CK_LDS u32x4 *>(slab + r * 256 + ((c ^ (r & 15)) << 4));
        if (wrow0 + r < ql)
            *reinterpret_cast<u32x4 *>(a.out + ((q0 + wrow0 + r) * a.heads + head) * kD + c * 8) = o;
    }
}

template <int DT, int NW>
int launch(PrefillArgs a, hipStream_t s) {
    constexpr int kRows = NW * 32;
    // every request's last tile may be a part, and so may that of the rows behind the last
    const int64_t tiles = a.tokens / kRows + a.batch + 1;
    const int64_t grid = tiles * a.heads;
    if (grid > 0x7FFFFFFF) return CK_E_INVALID_ARG;
    a.tiles = (int)tiles;
    static std::atomic<uint64_t> lds_set{0};
    int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(&latent_prefill_kernel<DT, NW>), kLds, lds_set);
    if (rc != CK_OK) return rc;
    hipLaunchKernelGGL((latent_prefill_kernel<DT, NW>), dim3((unsigned)grid), dim3(NW * 64), kLds, s, a);
    CK_RETURN_LAUNCH();
}

}  // namespace
}  // namespace ck

using namespace ck;

extern "C" int ck_latent_prefill(const void *q, const void *k, int64_t k_token_stride, int64_t k_head_stride,
                                 const void *k_rope, int64_t kr_stride, const void *v, int64_t v_token_stride,
                                 int64_t v_head_stride, const int64_t *q_seqlens, const int64_t *kv_seqlens,
                                 int64_t batch, int64_t num_tokens, int64_t num_keys, int64_t num_heads, int dtype,
                                 float scale, int causal, void *out, float *lse, void *stream) {
    if (dtype != CK_DTYPE_BF16 && dtype != CK_DTYPE_F16) return CK_E_UNSUPPORTED;
    if (batch < 0 || batch > (1 << 16) || num_tokens < 0 || num_keys < 0 || num_heads < 1 || num_heads > (1 << 16) ||
        num_tokens >= (int64_t)1 << 30 || num_keys >= (int64_t)1 << 30)
        return CK_E_INVALID_ARG;
    for (int64_t st : {k_token_stride, k_head_stride, kr_stride, v_token_stride, v_head_stride})
        if (st < 0 || st > (1 << 24) || st % 8 != 0) return CK_E_INVALID_ARG;
    if (!(scale > 0.f) || !std::isfinite(scale)) return CK_E_INVALID_ARG;
    if (num_tokens == 0) return CK_OK;
    if (!q || !out || !lse || (batch > 0 && (!q_seqlens || !kv_seqlens)) || (num_keys > 0 && (!k || !k_rope || !v)))
        return CK_E_NULL_PTR;
    if (!aligned_to(q, 16) || !aligned_to(k, 16) || !aligned_to(k_rope, 16) || !aligned_to(v, 16) ||
        !aligned_to(out, 16) || !aligned_to(lse, 4) || !aligned_to(q_seqlens, 8) || !aligned_to(kv_seqlens, 8))
        return CK_E_INVALID_ARG;
    PrefillArgs a = {};
    a.q = static_cast<const uint16_t *>(q);
    a.k = static_cast<const uint16_t *>(k);
    a.kr = static_cast<const uint16_t *>(k_rope);
    a.v = static_cast<const uint16_t *>(v);
    a.q_lens = q_seqlens;
    a.kv_lens = kv_seqlens;
    a.k_ts = k_token_stride;
    a.k_hs = k_head_stride;
    a.kr_ts = kr_stride;
    a.v_ts = v_token_stride;
    a.v_hs = v_head_stride;
    a.tokens = num_tokens;
    a.keys = num_keys;
    a.batch = (int)batch;
    a.heads = (int)num_heads;
    a.causal = causal != 0;
    a.scale_log2 = scale * kLog2e;
    a.out = static_cast<uint16_t *>(out);
    a.lse = lse;
    hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == CK_DTYPE_BF16) return launch<CK_DTYPE_BF16, 8>(a, s);
    return launch<CK_DTYPE_F16, 8>(a, s);
}
