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
//   queries). Q stays in registers (48), so does O (64).
// * 64-key tiles land in a ring of 3 slots by buffer -> LDS DMA: the head's keys (16 KB), the
//   rotated part all heads share (8 KB) and the values (16 KB), one in flight. The
//   resources end with the request's last key, so nothing past it is read.
// * S^T = K Q^T (24 products of 32x32x16 a tile) puts one query on a lane; P^T is in the operand's
//   place as it leaves; V^T comes through ds_read_b64_tr_b16 (16 products). P of tile t is made in the
//   shadow of tile t + 1's scores, the largest of those in that of tile t's second product. A step
//   of the two waves of a SIMD takes about 4200 cycles, its 80 products 2560.
// * A query's reference point of the softmax moves only when a score passes it by 2^kSlack.
// * Row tiles of a request are dealt last first: under a causal mask those are the longest.
// P is rounded to the 16-bit type before the second product, its sum is not.
// One workgroup walks all keys of its rows: with few queries most CUs have none, and the time is that of
// the walk. Measured, inputs changing from call to call: 6000 tokens x 32 heads, causal, 370 us (1.00
// PFLOP/s; 354 on the same inputs each time), every key seen 654 (1.13 PFLOP/s); 13 ragged prompts of
// about 580 on contexts, 16 heads, 91 us; 147 tokens x 16 heads 11.2 us, most of it the first passage through
// the code; 32 queries behind 8000 keys 136 us, with 8 heads or 32.
#include <cmath>

#include "latent_common.h"

namespace ck {
namespace {

using namespace lat;

typedef __attribute__((__vector_size__(2 * sizeof(unsigned)))) unsigned u32x2;

constexpr int kD = 128;            // a head's key part, and its value
constexpr int kQ = kD + kP;        // query row
constexpr int kTok = 64;           // keys per tile
constexpr int kWaves = 8, kThreads = kWaves * 64;
constexpr int kRows = kWaves * 32;  // queries per workgroup
// A tile in LDS. Keys: pieces of 4 rows (1 KB, one DMA) 1088 bytes apart, chunk c (16 bytes) of
// the piece's row i at c ^ i: the 16 rows that a 16-byte read is served for lie in 16 bank groups, and
// all chunks of a row are two registers and immediates away. Rotated part: pieces of 8 rows 1056
// bytes apart, chunk c at c ^ (i / 2 % 2). Values: pieces of 4 rows, chunk c at c ^ 4 i, for the
// transpose reads, which take 4 rows x 64 bytes.
constexpr int kKPiece = 1024 + 64, kRPiece = 1024 + 32, kVPiece = 1024;
constexpr int kRAt = kTok / 4 * kKPiece;
constexpr int kVAt = kRAt + kTok / 8 * kRPiece;
constexpr int kStage = kVAt + kTok / 4 * kVPiece;  // 41 KB
static_assert(kRAt % 256 == 0 && kVAt % 256 == 0 && kStage % 256 == 0, "addresses are XORed below bit 8");
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

// The 16-bit halves of w that are infinite or NaN, as 0x8000 each: without their sign those are
// the largest, kGap below the sign bit.
template <int DT>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    constexpr uint32_t kGap = DT == CK_DTYPE_BF16 ? 0x00800080u : 0x04000400u;
    return ((w & 0x7fff7fffu) + kGap) & 0x80008000u;
}

template <int DT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void latent_prefill_kernel(PrefillArgs a) {
    using E = Elem<DT>;
    constexpr int kBlk = 16 / kWaves;   // 1-KB DMAs of the keys (and of the values) per wave and tile
    constexpr int kRBlk = 8 / kWaves;   // and of the rotated part
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    CK_LDS char *smem = (CK_LDS char *)smem_raw;
    CK_LDS int *odd = (CK_LDS int *)(smem + kSlots * kStage);

    const int tid = threadIdx.x;
    const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int hh = lane >> 5, n32 = lane & 31;

    // Heads in pairs, a pair's row tiles longest first: an XCD's CUs end together, and its L2 holds
    // two heads' keys and values.
    const uint32_t w = xcd_remap(blockIdx.x, gridDim.x);
    const int pair = scalar((int)(w / (uint32_t)(2 * a.tiles))), in_pair = (int)w - pair * 2 * a.tiles;
    const bool two = 2 * pair + 1 < a.heads;
    const int head = 2 * pair + (two ? in_pair & 1 : 0);
    const uint32_t tile = two ? in_pair >> 1 : in_pair;

    // ---- which request's rows: each wave by itself, 64 requests at a time ---------------------
    // What passes the last token or key is cut off; behind the last request follow rows without keys.
    int64_t q0, k0 = 0;
    int ql, kl = 0, row0;
    {
        const uint32_t tokens = (uint32_t)a.tokens, keys = (uint32_t)a.keys;
        auto len_of = [](const int64_t *lens, int b, uint32_t most) {
            const int64_t n = lens[b];
            return n < 0 ? 0u : n > most ? most : (uint32_t)n;
        };
        uint32_t q_end = 0, k_end = 0, t_end = 0;
        bool found = false;
        for (int b0 = 0; b0 < a.batch && !found; b0 += 64) {
            const int b = b0 + lane;
            uint32_t n = 0, m = 0;
            if (b < a.batch) {
                n = len_of(a.q_lens, b, tokens);
                m = len_of(a.kv_lens, b, keys);
            }
            const uint32_t q_to = min(wave_scan(n, tokens) + q_end, tokens), k_to = min(wave_scan(m, keys) + k_end, keys);
            // where the request begins: where the one before ends
            uint32_t q_at = __builtin_amdgcn_update_dpp(0u, q_to, 0x138, 0xf, 0xf, false);  // the lane below's
            uint32_t k_at = __builtin_amdgcn_update_dpp(0u, k_to, 0x138, 0xf, 0xf, false);
            if (lane == 0) {
                q_at = q_end;
                k_at = k_end;
            }
            const uint32_t nt = (q_to - q_at + kRows - 1) / kRows;
            const uint32_t t_to = wave_scan(nt, ~0u >> 1) + t_end;
            const uint64_t hit = __builtin_amdgcn_ballot_w64(tile < t_to);
            if (hit) {
                const int from = (int)__ffsll((unsigned long long)hit) - 1;
                auto of = [&](uint32_t x) { return (int)__builtin_amdgcn_readlane(x, from); };
                q0 = of(q_at);
                ql = of(q_to - q_at);
                k0 = of(k_at);
                kl = of(k_to - k_at);
                row0 = (of(t_to) - 1 - (int)tile) * kRows;  // the last first: under a causal mask the longest
                found = true;
            }
            q_end = __builtin_amdgcn_readlane(q_to, 63);
            k_end = __builtin_amdgcn_readlane(k_to, 63);
            t_end = __builtin_amdgcn_readlane(t_to, 63);
        }
        if (!found) {
            q0 = q_end;
            ql = (int)(tokens - q_end);
            row0 = (int)(tile - t_end) * kRows;
        }
    }
    if (row0 >= ql) return;  // the same in every thread

    const int wrow0 = row0 + wid * 32;
    const int i_q = wrow0 + n32;
    const bool row_valid = i_q < ql;
    const int64_t qrow = (q0 + min(i_q, ql - 1)) * a.heads + head;
    // keys seen by this lane's query, by the wave's first and last, and by the workgroup's last
    auto seen = [&](int i) { return a.causal ? max(0, min(kl, kl - ql + 1 + i)) : kl; };
    const int limit = row_valid ? seen(i_q) : 0;
    const int w_last = min(wrow0 + 31, ql - 1);
    const int w_most = wrow0 < ql ? seen(w_last) : 0, w_least = seen(wrow0);
    const int most = seen(min(row0 + kRows - 1, ql - 1));
    const int ntiles = (most + kTok - 1) / kTok;

    // ---- DMA ----------------------------------------------------------------------------------
    // The wave's pieces: rows 4 (kBlk wid + j) .. + 3 of keys and values, 8 (kRBlk wid + j) .. + 7 of
    // the rotated part.
    const int p_i = lane >> 4, r_i = lane >> 3;  // the lane's row in a piece
    const uint32_t k_dma = (uint32_t)((wid * kBlk * 4 + p_i) * a.k_ts + ((lane & 15) ^ p_i) * 8) * 2;
    const uint32_t v_dma = (uint32_t)((wid * kBlk * 4 + p_i) * a.v_ts + ((lane & 15) ^ (4 * p_i)) * 8) * 2;
    const uint32_t r_dma = (uint32_t)((wid * kRBlk * 8 + r_i) * a.kr_ts + ((lane & 7) ^ ((r_i >> 1) & 1)) * 8) * 2;
    // The next tile that is moved: where it begins, and the request's rows from there on. Bytes past
    // those are not read; past the last tile nothing comes, but as many DMAs are counted.
    uint64_t k_from = (uint64_t)(uintptr_t)(a.k + k0 * a.k_ts + head * a.k_hs);
    uint64_t r_from = (uint64_t)(uintptr_t)(a.kr + k0 * a.kr_ts);
    uint64_t v_from = (uint64_t)(uintptr_t)(a.v + k0 * a.v_ts + head * a.v_hs);
    const uint32_t k_row = 2 * (uint32_t)a.k_ts, r_row = 2 * (uint32_t)a.kr_ts, v_row = 2 * (uint32_t)a.v_ts;
    int left = kl;
    const int lds0 = scalar((int)(uintptr_t)smem);
    auto issue = [&](int slot) {
        const int more = min(kTok, left) - 1;
        auto from = [&](uint64_t at, uint32_t row, int width) {
            ck_rsrc_t r;
            r[0] = (int)(uint32_t)at;
            r[1] = (int)((uint32_t)(at >> 32) & 0xffffu);
            r[2] = more >= 0 ? (int)(more * row + 2 * width) : 0;
            r[3] = 0x00020000;
            return r;
        };
        const ck_rsrc_t rk = from(k_from, k_row, kD), rr = from(r_from, r_row, kP), rv = from(v_from, v_row, kD);
        const int to = lds0 + slot * kStage;
        static_for<kBlk>([&](auto j) __attribute__((always_inline)) {
            dma_tile<j * kKPiece>(rk, (int)(k_dma + j * 4 * k_row), 0, to + wid * (kBlk * kKPiece));
            dma_tile<kVAt + j * kVPiece>(rv, (int)(v_dma + j * 4 * v_row), 0, to + wid * (kBlk * kVPiece));
        });
        static_for<kRBlk>([&](auto j) __attribute__((always_inline)) {
            dma_tile<kRAt + j * kRPiece>(rr, (int)(r_dma + j * 8 * r_row), 0, to + wid * (kRBlk * kRPiece));
        });
        k_from += (uint64_t)kTok * k_row;
        r_from += (uint64_t)kTok * r_row;
        v_from += (uint64_t)kTok * v_row;
        left -= kTok;
    };
    // What this wave has moved of tile t is in. Where not every query of the workgroup sees all of it,
    // values that 0 * V would turn into NaN become zeros: those past the request's end, and infinite
    // or NaN ones, which set the tile's bit in *odd and reach the queries that see them at the end.
    const int w_first = scalar(seen(row0)), first_odd = w_first / kTok;
    auto look = [&](int t, int slot) {
        if (t * kTok + kTok <= w_first) return;
        int l = tid & 63;
        asm volatile("" : "+v"(l));
        uint32_t bad = 0;
#pragma unroll
        for (int j = 0; j < kBlk; ++j) {
            const int r = (wid * kBlk + j) * 4 + (l >> 4);
            CK_LDS u32x4 *at = reinterpret_cast<CK_LDS u32x4 *>(smem + slot * kStage + kVAt + (wid * kBlk + j) * kVPiece + l * 16);
            u32x4 x = *at;
            if (t * kTok + r >= kl) {
                *at = u32x4{0, 0, 0, 0};
            } else {
                const u32x4 odd_ones = {not_finite<DT>(x[0]), not_finite<DT>(x[1]), not_finite<DT>(x[2]), not_finite<DT>(x[3])};
                const uint32_t any = odd_ones[0] | odd_ones[1] | odd_ones[2] | odd_ones[3];
                if (any != 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] &= ~((odd_ones[i] >> 15) * 0xffffu);
                    *at = x;
                }
                bad |= any;
            }
        }
        if (bad != 0) __hip_atomic_fetch_or(odd, 1 << (t - first_odd), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    };

    f32x16 oacc[4];
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[db][i] = 0.f;
    float m_run = -INFINITY, sub = -E::kBias, l_part = 0.f;
    bool fresh = true;  // O is zero

    // A lane's place in a tile: of keys n32 (+ 32), chunk hh, and their rotated part; of values by
    // transpose reads. (That of the rotated part is found again in every step: with it a register
    // would spill, whose reload waits for the DMAs.)
    auto rope_at = [&]() {
        int l = lane;
        asm volatile("" : "+v"(l));
        return kRAt + ((l >> 3) & 3) * kRPiece + (l & 7) * 128 + ((l >> 5) ^ ((l >> 1) & 1)) * 16;
    };
    const int trG = (lane >> 4) & 3, tr_row = (lane & 15) >> 2, tr_e4 = lane & 3;
    const int key_at = (n32 >> 2) * kKPiece + (n32 & 3) * 256 + ((hh ^ n32) & 3) * 16;
    const int value_at = kVAt + (trG >> 1) * kVPiece + tr_row * 256 + (4 * tr_row + 2 * (trG & 1) + (tr_e4 >> 1)) * 16 + (tr_e4 & 1) * 8;

    u32x4 qf[12];
    // S^T = K Q^T of the tile in `slot`; between(f) is placed after the f-th product.
    auto scores = [&](int slot, f32x16 (&x)[2], auto &&between) __attribute__((always_inline)) {
        const CK_LDS char *tile = smem + slot * kStage;
        const CK_LDS char *k_even = tile + key_at, *k_odd = tile + (key_at ^ 32), *rope = tile + rope_at();
        auto kfrag = [&](int f) {
            const int ks = f >> 1;
            return *reinterpret_cast<const CK_LDS u32x4 *>(
                ks < 8 ? (ks & 1 ? k_odd : k_even) + (ks >> 1) * 64 + (f & 1) * 8 * kKPiece
                       : rope + (ks - 8) * 32 + (f & 1) * 4 * kRPiece);
        };
        constexpr int kAhead = 3, kHeld = kAhead + 1;
        const f32x16 zero16 = {};
        u32x4 kf[kHeld];
#pragma unroll
        for (int f = 0; f < kAhead; ++f) kf[f] = kfrag(f);
        __builtin_amdgcn_sched_barrier(0);
        static_for<24>([&](auto f) __attribute__((always_inline)) {
            x[f & 1] = E::mfma32(kf[f % kHeld], qf[f >> 1], f < 2 ? zero16 : x[f & 1]);
            if (f + kAhead < 24) kf[(f + kAhead) % kHeld] = kfrag(f + kAhead);
            between(f);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    u32x4 pb[4];
    // The lane's 32 probabilities in pairs: begun, and a product later, when the exponentials are
    // there, summed and packed (left for the end, the 32 would need twice the registers).
    float p0, p1;
    auto p_begin = [&](const f32x16 (&x)[2], int pair) __attribute__((always_inline)) {
        const int q2 = pair >> 3, j = pair & 7;
        p0 = exp2_fast(fmaf(x[q2][2 * j], a.scale_log2, -sub));
        p1 = exp2_fast(fmaf(x[q2][2 * j + 1], a.scale_log2, -sub));
    };
    auto p_end = [&](int pair) __attribute__((always_inline)) {
        const int q2 = pair >> 3, j = pair & 7;
        l_part += p0;
        l_part += p1;
        uint32_t both = E::pack2(p0, p1);
        asm volatile("" : "+v"(both));
        pb[2 * q2 + (j >> 2)][j & 3] = both;
    };
    // Values' fragment: keys 16 s .. + 15 of the tile, dims 32 db .. + 31.
    auto vfrag = [&](int slot, int s, int db) __attribute__((always_inline)) {
        const CK_LDS char *at = smem + slot * kStage + (value_at ^ (db * 64)) + s * 4 * kVPiece;
        const uint2 lo = lds_read_tr16(at), hi = lds_read_tr16(at + 2 * kVPiece);
        return u32x4{lo.x, lo.y, hi.x, hi.y};
    };
    // O^T += V^T P^T.
    auto products = [&](int slot, auto &&between) __attribute__((always_inline)) {
        constexpr int kAhead = 3, kHeld = kAhead + 1;
        u32x4 vf[kHeld];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) vf[i] = vfrag(slot, i >> 2, i & 3);
        __builtin_amdgcn_sched_barrier(0);
        static_for<16>([&](auto i) __attribute__((always_inline)) {
            oacc[i & 3] = E::mfma32(vf[i % kHeld], pb[i >> 2], oacc[i & 3]);
            if (i + kAhead < 16) vf[(i + kAhead) % kHeld] = vfrag(slot, (i + kAhead) >> 2, (i + kAhead) & 3);
            between(i);
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    auto nothing = [](auto &&...) {};
    float v = -INFINITY;  // the query's largest score of the lane's keys
    auto largest = [&](const f32x16 (&x)[2]) {
        v = max3(x[0][0], x[0][1], x[0][2]);
#pragma unroll
        for (int e = 3; e < 31; e += 2) v = max3(v, x[e >> 4][e & 15], x[(e + 1) >> 4][(e + 1) & 15]);
        v = max_xor32(fmaxf(v, x[1][15])) * a.scale_log2;
    };
    auto next_slot = [](int slot) { return slot == kSlots - 1 ? 0 : slot + 1; };

    issue(0);
    // Q in pieces of 8 rows x 128 bytes, turned into operands (row n32, chunk 2 kk + hh) through the
    // wave's 4 KB of the slot that is used last: an operand's own place, 64 lanes in 32 rows, costs a
    // cycle a lane, 6100 for a workgroup. A row past the last repeats it: it is not stored.
    if (wrow0 < ql) {
        const uint16_t *q = a.q + (q0 * a.heads + head) * kQ + 8 * (lane & 7);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint16_t *row = q + (int64_t)min(wrow0 + 8 * e + (lane >> 3), ql - 1) * a.heads * kQ;
#pragma unroll
            for (int m = 0; m < 3; ++m) qf[4 * m + e] = *reinterpret_cast<const u32x4 *>(row + 64 * m);
        }
    }
    wait_vmcnt<0>();
    issue(1);
    if (wrow0 < ql) {
        CK_LDS char *at = smem + (kSlots - 1) * kStage + wid * 4096;
        auto piece = [&](int row, int chunk) {
            return reinterpret_cast<CK_LDS u32x4 *>(at + row * 128 + ((chunk ^ (row >> 1)) & 7) * 16);
        };
#pragma unroll
        for (int m = 0; m < 3; ++m) {
#pragma unroll
            for (int e = 0; e < 4; ++e) *piece(8 * e + (lane >> 3), lane & 7) = qf[4 * m + e];
#pragma unroll
            for (int e = 0; e < 4; ++e) qf[4 * m + e] = *piece(n32, 2 * e + hh);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // before tile 2 is moved there
    }
    if (tid == 0) *odd = 0;
    __syncthreads();
    look(0, 0);
    __syncthreads();
    int slot = 0, t = 0;  // tile t's
    // A step: P of tile t (scores x) beside the scores y of tile t + 1, then the products of tile t
    // beside the largest of y: the matrix cores wait for neither.
    auto step = [&](f32x16 (&x)[2], f32x16 (&y)[2]) __attribute__((always_inline)) {
        const int s1 = next_slot(slot), s2 = next_slot(s1);
        wait_vmcnt<0>();
        look(t + 1, s1);
        __syncthreads();  // tile t + 1 is in; every wave is done with tile t - 1, whose slot is next
        issue(s2);
        const int first = t * kTok;
        if (first < w_most) {
            const bool hides = first + kTok > w_least;
            if (hides) {
                int half = hh;  // again: what it gives is not to be held over the steps
                asm volatile("" : "+v"(half));
#pragma unroll
                for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (first + 32 * q2 + (e & 3) + 8 * (e >> 2) + 4 * half >= limit) x[q2][e] = -INFINITY;
                largest(x);
            }
            if (__builtin_amdgcn_ballot_w64(v > m_run + kSlack)) {
                const bool mine = v > m_run + kSlack;
                const float dm = mine ? exp2_fast(m_run - v) : 1.f;
                if (mine) m_run = v;
                l_part *= dm;
                sub = (m_run == -INFINITY ? 0.f : m_run) - E::kBias;
                if (!fresh) {
#pragma unroll
                    for (int db = 0; db < 4; ++db)
#pragma unroll
                        for (int e = 0; e < 16; ++e) oacc[db][e] *= dm;
                }
            }
            fresh = false;
            if (first + kTok < w_most) {
                __builtin_amdgcn_s_setprio(1);
                scores(s1, y, [&](auto f) __attribute__((always_inline)) {
                    if constexpr (f % 3 != 0) {
                        constexpr int pair = f - 1 - f / 3;
                        if constexpr (pair > 0) p_end(pair - 1);
                        p_begin(x, pair);
                    }
                });
                p_end(15);
                __builtin_amdgcn_s_setprio(0);
            } else {
                // unlike the scores above: their exponents are to be made beside the products there, not before
                asm volatile("" : "+v"(x[0]), "+v"(x[1]));
                static_for<16>([&](auto i) __attribute__((always_inline)) {
                    p_begin(x, i);
                    p_end(i);
                });
                asm volatile("" : "=v"(y[0]), "=v"(y[1]));  // not looked at
            }
            products(slot, [&](auto i) __attribute__((always_inline)) {
                if constexpr (i == 0) v = max3(y[0][0], y[0][1], y[0][2]);
                else if constexpr (i < 15) v = max3(v, y[(2 * i + 1) >> 4][(2 * i + 1) & 15], y[(2 * i + 2) >> 4][(2 * i + 2) & 15]);
                else v = max_xor32(fmaxf(v, y[1][15])) * a.scale_log2;
            });
        } else {
            asm volatile("" : "=v"(y[0]), "=v"(y[1]));
        }
        slot = s1;
        ++t;
    };
    f32x16 s[2], y[2];
    asm volatile("" : "=v"(y[0]), "=v"(y[1]));
    if (w_most > 0) {
        scores(0, s, nothing);
        largest(s);
    } else {
        asm volatile("" : "=v"(s[0]), "=v"(s[1]));
    }
    while (true) {
        step(s, y);
        if (t >= ntiles) break;
        step(y, s);
        if (t >= ntiles) break;
    }
    wait_vmcnt<0>();  // the empty moves too

    // ---- normalise, write whole rows through the idle ring ----------------------------------
    const float l_run = l_part + __shfl_xor(l_part, 32);
    __syncthreads();  // every wave is past its last ring read
    if (wrow0 >= ql) return;
    // Infinite and NaN values that were left out, for the queries that see them (whose p is
    // positive): as they are, no finite weight or sum changes what they give.
    const int odd_tiles = scalar(*odd);
    for (int t = first_odd; odd_tiles >> (t - first_odd) != 0 && t * kTok < w_most; ++t) {
        if (!((odd_tiles >> (t - first_odd)) & 1)) continue;
        for (int k = 0; k < kTok; ++k) {
            if (t * kTok + k >= limit) break;
            const uint16_t *row = a.v + (k0 + t * kTok + k) * a.v_ts + head * a.v_hs + 4 * hh;
#pragma unroll
            for (int c = 0; c < 16; ++c) {
                const u32x2 w = *reinterpret_cast<const u32x2 *>(row + 8 * c);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (not_finite<DT>(w[j >> 1]) & (j & 1 ? 0x80000000u : 0x8000u))
                        oacc[c >> 2][4 * (c & 3) + j] += j & 1 ? E::hi(w[j >> 1]) : E::lo(w[j >> 1]);
            }
        }
    }
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

template <int DT>
int launch(PrefillArgs a, hipStream_t s) {
    // every request's last tile may be a part, and so may that of the rows behind the last
    const int64_t tiles = a.tokens / kRows + a.batch + 1;
    const int64_t grid = tiles * a.heads;
    if (!grid_fits(grid, kThreads)) return CK_E_INVALID_ARG;
    a.tiles = (int)tiles;
    static std::atomic<uint64_t> lds_set{0};
    int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(&latent_prefill_kernel<DT>), kLds, lds_set);
    if (rc != CK_OK) return rc;
    hipLaunchKernelGGL((latent_prefill_kernel<DT>), dim3((unsigned)grid), dim3(kThreads), kLds, s, a);
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
    if (!(scale > 0.f) || !std::isfinite(scale * kLog2e)) return CK_E_INVALID_ARG;
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
    if (dtype == CK_DTYPE_BF16) return launch<CK_DTYPE_BF16>(a, s);
    return launch<CK_DTYPE_F16>(a, s);
}
