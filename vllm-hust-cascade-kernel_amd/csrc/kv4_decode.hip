// kv4_decode.hip - decode attention over a paged K/V cache in 4 bits (gfx950), alone or with a prefix that all
// sequences share.
//
// Row (token i, head h) of request b, k_j and v_j the dequantised cache of its kv head:
//   s_j = scale q . k_j, j < len_b - q_len + 1 + i
//   o = sum_j softmax(s)_j v_j,  lse = log sum_j exp(s_j)
// A row that sees no token gets o = 0, lse = -inf.
//
// A token and kv head are 136 bytes and 512 flops a row: up to some 32 rows a kv head memory
// bounds the call. A wave computes alone, for 16 NB rows of a kv head (tokens of a request times query
// heads of the kv head):
// * A unit of 64 tokens (8704 bytes that lie together) is 10 loads of a wave, straight into registers in
//   the operands' order; the next unit's are under way while one is computed.
// * S^T = K Q^T on 16x16x32 products: lane (g, n) holds group g of a token's key, four codes-to-bf16
//   conversions (two values each, the scale in the instruction) make an operand. O^T = V^T P^T: lane (g, n)
//   holds dims 8 n .. + 7 of tokens 8 g .. + 7; two conversions give (token, dim pair) words, two byte
//   permutations turn them to (dim, token pair). P is in its operand's place as it leaves the scores.
// * bf16 holds every dequantised value; P enters as two bf16 terms, within 2^-17 of fp32; an fp16 query as
//   two bf16 terms, which hold all of it.
// * The softmax's reference point m of a row moves only when a score passes it by 2^kSlack (any point gives the
//   same result), so that O is hardly ever rescaled.
// * The units of all requests and kv heads form one list, cut evenly over the waves of a grid that fills the
//   chip once, so ragged lengths balance. An item (request and kv head) inside one share is written as it is;
//   parts of a cut one go to the workspace, and kv4_combine_kernel folds them.
// * Rows past 16 NB are row tiles of their own, given to neighbouring waves, which read the same units.
// * Shared prefix: the batch is one request's rows over the prefix; then the suffixes; one fold for both.
#include <cmath>

#include "kv4_common.h"
#include "kv4_map.h"

namespace ck {
namespace {

using namespace kv4;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kGroups = 512;  // workgroups: two per CU
constexpr int kFoldRows = 4096;  // from which on a row's parts are folded by one group of lanes
constexpr float kSlack = 8.f;
constexpr uint32_t kRsrcFlags = 0x00020000;

struct DecodeArgs {
    const uint16_t *q;  // [batch * q_len, heads, 128]
    const uint8_t *cache;
    const int32_t *bt;
    const int64_t *lens;
    int64_t bt_cols;
    int64_t num_blocks;
    int batch, q_len, heads, kv_heads;
    int group;   // query heads per kv head
    int rows;    // q_len * group: of an item
    int tiles;   // row tiles of an item
    int waves;   // that share the list, per row tile
    int causal;
    int merge;   // every part goes to the workspace
    float scale_log2;
    uint16_t *out;
    float *lse;
    // Parts, not normalised: [slot][tile][8][tile's rows][4 g][4], dims 32 g + 4 j + e
    float *part_o;
    float2 *part_ml;  // [slot][tile][tile's rows]: reference point (log2), sum of p
    int32_t *sums;    // [batch + 1]: units before each request (of one kv head)
};

__device__ __forceinline__ int len_of(const DecodeArgs &a, int b) {
    const int64_t cap = a.bt_cols * kPage;
    int64_t n = a.lens[b];
    if (n > cap) n = cap;
    return n < 0 || a.num_blocks <= 0 ? 0 : (int)n;
}
__device__ __forceinline__ int units_of(int len) { return (len + kUnit - 1) / kUnit; }

// A unit as a wave's lanes hold it: lane (g, n) has group g of keys 8 (n / 4) + n % 4 + {0, 4, 32, 36}
// and their scales, dims 8 n + 2 q, + 1 of values 8 g .. + 7 and 32 + 8 g .. + 7, and these tokens' scales of dim
// group n / 4.
struct Unit {
    u32x4 k[4], v[4], vs;
    uint32_t ks;
};
__device__ __forceinline__ void load_unit(Unit &u, const char *base, int range, int lane) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base), (short)0, range, kRsrcFlags);
    const int n = lane & 15, g = lane >> 4;
    const int k_at = (8 * (n >> 2) + (n & 3)) * 64 + 16 * g, v_at = kVAt + 16 * lane;
#pragma unroll
    for (int t = 0; t < 4; ++t)
        u.k[t] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, k_at + (t >> 1) * 2048 + (t & 1) * 256, 0, 0));
    u.ks = __builtin_amdgcn_raw_buffer_load_b32(r, kKsAt + 4 * lane, 0, 0);
    u.vs = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, kVsAt + (n >> 2) * 64 + 16 * g, 0, 0));
#pragma unroll
    for (int q = 0; q < 4; ++q)
        u.v[q] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, v_at + 1024 * q, 0, 0));
}

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 x, u32x4 y, f32x4 c) { return Elem<CK_DTYPE_BF16>::mfma16(x, y, c); }

// The rows of a wave: row 16 i + n in lanes (g, n).
template <int DT, int NB>
struct Rows {
    static constexpr int kTerms = DT == CK_DTYPE_BF16 ? 1 : 2;
    u32x4 q[NB][kTerms][4];  // dims 32 g + 8 c .. + 7
    f32x4 o[NB][8];          // O^T: dims 32 g + 8 r + block of the row
    float m[NB], l[NB];      // reference point (log2; the same for all g), this lane's share of the sum
};

// Bytes of four scales whose tokens are the first `n` of the four.
__device__ __forceinline__ uint32_t first_bytes(uint32_t w, int n) {
    return n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1);
}

// O^T += V^T P^T over a unit, vs the values' scales; P of row block i as operands hi, lo [i][half].
template <int DT, int NB>
__device__ __forceinline__ void add_values(Rows<DT, NB> &s, const Unit &u, u32x4 vs, const u32x4 (&hi)[NB][2],
                                           const u32x4 (&lo)[NB][2]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float sc[8];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            sc[4 * w] = scale_of<0>(vs[2 * h + w]);
            sc[4 * w + 1] = scale_of<1>(vs[2 * h + w]);
            sc[4 * w + 2] = scale_of<2>(vs[2 * h + w]);
            sc[4 * w + 3] = scale_of<3>(vs[2 * h + w]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            u32x4 even, odd;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const uint32_t c = u.v[q][2 * h + w];
                const uint32_t t0 = pair_bf16<0>(c, sc[4 * w]), t1 = pair_bf16<1>(c, sc[4 * w + 1]);
                const uint32_t t2 = pair_bf16<2>(c, sc[4 * w + 2]), t3 = pair_bf16<3>(c, sc[4 * w + 3]);
                even[2 * w] = __builtin_amdgcn_perm(t1, t0, 0x05040100);
                odd[2 * w] = __builtin_amdgcn_perm(t1, t0, 0x07060302);
                even[2 * w + 1] = __builtin_amdgcn_perm(t3, t2, 0x05040100);
                odd[2 * w + 1] = __builtin_amdgcn_perm(t3, t2, 0x07060302);
            }
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                s.o[i][2 * q] = mfma_bf16(even, hi[i][h], s.o[i][2 * q]);
                s.o[i][2 * q + 1] = mfma_bf16(odd, hi[i][h], s.o[i][2 * q + 1]);
                s.o[i][2 * q] = mfma_bf16(even, lo[i][h], s.o[i][2 * q]);
                s.o[i][2 * q + 1] = mfma_bf16(odd, lo[i][h], s.o[i][2 * q + 1]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// One unit. Where tail: tokens from sees[i] on are hidden from row block i's row, those from `left` on
// (counted from the unit's first) hold anything.
template <int DT, int NB>
__device__ __forceinline__ void compute(Rows<DT, NB> &s, const Unit &u, float scale_log2, int lane, bool tail,
                                        const int (&sees)[NB], int left) {
    const int g = lane >> 4;
    f32x4 sc[NB][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const float ks = t == 0 ? scale_of<0>(u.ks) : t == 1 ? scale_of<1>(u.ks) : t == 2 ? scale_of<2>(u.ks) : scale_of<3>(u.ks);
#pragma unroll
        for (int i = 0; i < NB; ++i) sc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint32_t w = u.k[t][c];
            const u32x4 a = {pair_bf16<0>(w, ks), pair_bf16<1>(w, ks), pair_bf16<2>(w, ks), pair_bf16<3>(w, ks)};
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int x = 0; x < Rows<DT, NB>::kTerms; ++x) sc[i][t] = mfma_bf16(a, s.q[i][x][c], sc[i][t]);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    u32x4 vs = u.vs;
    if (tail) {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int n = sees[i] - 8 * g;  // token of sc[i][t][r]: 32 (t / 2) + 8 g + 4 (t % 2) + r
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (32 * (e >> 3) + (e & 7) >= n) sc[i][e >> 2][e & 3] = -INFINITY;
        }
        // Values that are not numbers would reach rows that do not see them (0 times them is none): their scales
        // become the least one, and rows that do see one get it added. A lane (g, n) has the dims of group g.
        int first_bad = kUnit;
#pragma unroll
        for (int w = 3; w >= 0; --w) {
            const int t0 = 32 * (w >> 1) + 8 * g + 4 * (w & 1);
            vs[w] = first_bytes(vs[w], left - t0);
#pragma unroll
            for (int b = 3; b >= 0; --b) {
                if (((vs[w] >> (8 * b)) & 0xff) != kBad) continue;
                first_bad = t0 + b;
                vs[w] &= ~(0xffu << (8 * b));
            }
        }
        if (__builtin_amdgcn_ballot_w64(first_bad < kUnit)) {
            first_bad = (int)over_groups((float)first_bad, [](float x, float y) { return fminf(x, y); });
            first_bad = __shfl(first_bad, 4 * g);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                if (first_bad >= sees[i]) continue;
#pragma unroll
                for (int k = 0; k < 8; ++k)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s.o[i][k][r] = NAN;
            }
        }
    }
    u32x4 hi[NB][2], lo[NB][2];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        float most = max3(sc[i][0][0], sc[i][0][1], sc[i][0][2]);
#pragma unroll
        for (int e = 3; e < 15; e += 2) most = max3(most, sc[i][e >> 2][e & 3], sc[i][(e + 1) >> 2][(e + 1) & 3]);
        most = fmaxf(most, sc[i][3][3]) * scale_log2;
        if (__builtin_amdgcn_ballot_w64(most > s.m[i] + kSlack)) {
            const float all = over_groups(most, [](float x, float y) { return fmaxf(x, y); });
            const float m = all > s.m[i] + kSlack ? all : s.m[i];
            const float f = m == s.m[i] ? 1.f : exp2_fast(s.m[i] - m);
            s.l[i] *= f;
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r) s.o[i][k][r] *= f;
            s.m[i] = m;
        }
        const float sub = s.m[i] == -INFINITY ? 0.f : s.m[i];
        float p[16], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            p[e] = exp2_fast(fmaf(sc[i][e >> 2][e & 3], scale_log2, -sub));
            sum += p[e];
        }
        s.l[i] += sum;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t h = pack_bf16x2(p[2 * e], p[2 * e + 1]);
            hi[i][e >> 2][e & 3] = h;
            lo[i][e >> 2][e & 3] = pack_bf16x2(p[2 * e] - bf16_lo(h), p[2 * e + 1] - bf16_hi(h));
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    add_values(s, u, vs, hi, lo);
}

template <int DT, int NB>
__global__ __launch_bounds__(kThreads, 2) void kv4_decode_kernel(DecodeArgs a) {
    __shared__ int starts[kThreads], scan[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6);
    constexpr int kRows = 16 * NB;
    constexpr bool kAhead = NB == 1;  // the next item's queries are loaded ahead

    // ---- units before each thread's requests, and in all (of one kv head) --------------------------
    const int per = (a.batch + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += units_of(len_of(a, b));
    const int incl = (int)wave_scan((uint32_t)mine, 0x7fffffffu);
    if (lane == 63) scan[wave] = incl;
    __syncthreads();
    int start = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) start += scan[w];
        total += scan[w];
    }
    total = scalar(total);
    starts[tid] = start;
    if (blockIdx.x == 0) {
        int at = start;
        for (int b = b0; b < b1; ++b) {
            a.sums[b] = at;
            at += units_of(len_of(a, b));
        }
        if (tid == 0) a.sums[a.batch] = total;
    }
    __syncthreads();

    // ---- this wave's share ---------------------------------------------------------------------------
    // One row tile: neighbouring shares on different CUs, so that few units spread over all of
    // them; several: a unit's row tiles side by side.
    const int nw = (int)gridDim.x * kWaves;
    const int id = a.tiles == 1 ? wave * (int)gridDim.x + (int)blockIdx.x : (int)blockIdx.x * kWaves + wave;
    if (id >= a.waves * a.tiles) return;
    const int w = scalar(id / a.tiles), tile = scalar(id - w * a.tiles);
    const Cut cut = list_cut(total * a.kv_heads, a.waves);
    if (w >= cut.chunks) return;
    const int lo = scalar(cut_lo(cut, w)), hi = scalar(cut_lo(cut, w + 1));
    const int tile_rows = min(kRows, a.rows - kRows * tile), slot_rows = min(kRows, a.rows);

    Rows<DT, NB> s;
    u32x4 next_q[NB][4];
    int tok[NB];  // of row block i's row, among the request's
#pragma unroll
    for (int i = 0; i < NB; ++i) tok[i] = (kRows * tile + 16 * i + (lane & 15)) / a.group;

    // The lane again, so that addresses of rows and parts are not held over the units.
    auto lane_again = [&]() {
        int x = lane;
        asm volatile("" : "+v"(x));
        return x;
    };
    auto load_q = [&](int item) {
        const int b = scalar(item / a.kv_heads), h = item - b * a.kv_heads;
        const int x = lane_again(), n16 = x & 15, g4 = x >> 4;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int r = kRows * tile + 16 * i + n16;
            const uint16_t *p = a.q + (((int64_t)b * a.q_len + tok[i]) * a.heads + h * a.group + (r - tok[i] * a.group)) * kD + 32 * g4;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                next_q[i][c] = u32x4{0, 0, 0, 0};
                if (r < a.rows) next_q[i][c] = *reinterpret_cast<const u32x4 *>(p + 8 * c);
            }
        }
    };
    auto open_item = [&](int item) {
        if constexpr (!kAhead) load_q(item);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if constexpr (DT == CK_DTYPE_BF16) {
                    s.q[i][0][c] = next_q[i][c];
                } else {
                    using E = Elem<DT>;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = E::lo(next_q[i][c][e]), y = E::hi(next_q[i][c][e]);
                        const uint32_t top = pack_bf16x2(x, y);
                        s.q[i][0][c][e] = top;
                        s.q[i][Rows<DT, NB>::kTerms - 1][c][e] = pack_bf16x2(x - bf16_lo(top), y - bf16_hi(top));
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) s.o[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
            s.m[i] = -INFINITY;
            s.l[i] = 0.f;
        }
    };
    auto close_item = [&](int item, bool before, bool after) {
        const int b = scalar(item / a.kv_heads), h = item - b * a.kv_heads;
        const int x = lane_again(), n16 = x & 15, g4 = x >> 4;
        const bool whole = !before && !after && !a.merge;
        const int64_t slot = part_slot(before, after, w, a.waves, item) * a.tiles + tile;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int r = kRows * tile + 16 * i + n16;
            const float l = over_groups(s.l[i], [](float x, float y) { return x + y; });
            if (r >= a.rows) continue;
            if (whole) {
                using E = Elem<DT>;
                const int64_t row = ((int64_t)b * a.q_len + tok[i]) * a.heads + h * a.group + (r - tok[i] * a.group);
                const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    u32x4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = E::pack2(s.o[i][2 * e][d] * inv, s.o[i][2 * e + 1][d] * inv);
                    *reinterpret_cast<u32x4 *>(a.out + row * kD + 32 * g4 + 8 * d) = x;
                }
                if (g4 == 0) a.lse[row] = l == 0.f ? -INFINITY : (s.m[i] + __log2f(l)) * kLn2;
            } else {
                const int at = 16 * i + n16;
                float *p = a.part_o + slot * slot_rows * kD;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // dims 32 g + 4 j + e: 8 (j / 2) + block 4 (j % 2) + e
                    const f32x4 x = {s.o[i][4 * (j & 1)][j >> 1], s.o[i][4 * (j & 1) + 1][j >> 1],
                                     s.o[i][4 * (j & 1) + 2][j >> 1], s.o[i][4 * (j & 1) + 3][j >> 1]};
                    *reinterpret_cast<f32x4 *>(p + ((j * slot_rows + at) * 4 + g4) * 4) = x;
                }
                if (g4 == 0) a.part_ml[slot * slot_rows + at] = make_float2(s.m[i], l);
            }
        }
    };

    // ---- the units, 64 described at a time: one a lane ---------------------------------------------------
    int item = -1;
    bool before = false, goes_on = false;  // the open item: begun in an earlier share; its last unit not seen yet
    for (int base = lo; base < hi; base += 64) {
        const int n = min(64, hi - base);
        int d_item = 0, d_first = 0, d_len = 0;
        uint64_t d_at = 0;
        if (lane < n) {
            const int u = base + lane;
            int x = 0;  // the last thread whose requests begin at or before u and that has some
#pragma unroll
            for (int step = kThreads / 2; step > 0; step >>= 1)
                if (starts[x + step] * a.kv_heads <= u) x += step;
            int b = min(x * per, a.batch - 1), at = starts[x] * a.kv_heads;
            int len = len_of(a, b);
            while (b + 1 < a.batch && at + units_of(len) * a.kv_heads <= u) {  // the thread's request that holds u
                at += units_of(len) * a.kv_heads;
                len = len_of(a, ++b);
            }
            const int each = units_of(len), h = (u - at) / each, i = u - at - h * each;
            const int page = a.bt[(int64_t)b * a.bt_cols + (i >> 1)];
            const bool ok = page >= 0 && page < a.num_blocks;
            d_item = b * a.kv_heads + h;
            d_first = i * kUnit;
            d_len = len;
            d_at = (uint64_t)(uintptr_t)a.cache;  // 16-byte aligned: bit 0 marks an invalid page
            d_at += ok ? (((uint64_t)(uint32_t)page * a.kv_heads + h) * 2 + (i & 1)) * kUnitBytes : 1;
        }
        auto unit_at = [&](Unit &u, int j) {
            const uint64_t at = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(d_at >> 32), j) << 32) |
                                (uint32_t)__builtin_amdgcn_readlane((int)d_at, j);
            // a range of nothing reads zeros
            load_unit(u, reinterpret_cast<const char *>((uintptr_t)(at & ~1ull)), at & 1 ? 0 : kUnitBytes, lane);
        };
        Unit next;
        unit_at(next, 0);
        if (const int first = __builtin_amdgcn_readlane(d_item, 0); kAhead && first != item) load_q(first);
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
            const Unit u = next;
            const int it = __builtin_amdgcn_readlane(d_item, j), first = __builtin_amdgcn_readlane(d_first, j);
            const int len = __builtin_amdgcn_readlane(d_len, j);
            if (it != item) {
                if (item >= 0) close_item(item, before, goes_on);
                open_item(it);
                item = it;
                before = first != 0;
            }
            goes_on = first + kUnit < len;
            if (j + 1 < n) {
                unit_at(next, j + 1);
                if (const int then = __builtin_amdgcn_readlane(d_item, j + 1); kAhead && then != it) load_q(then);
            }
            const int left = len - first, first_sees = a.causal ? left - a.q_len + 1 : left;
            int sees[NB];
#pragma unroll
            for (int i = 0; i < NB; ++i) sees[i] = a.causal ? first_sees + tok[i] : left;
            compute<DT, NB>(s, u, a.scale_log2, lane, first_sees < kUnit, sees, left);
        }
    }
    close_item(item, before, goes_on);
}

// ---- the fold of cut items, and of a prefix with its suffixes ---------------------------------------------
struct FoldSide {
    const float *part_o;
    const float2 *part_ml;
    const int32_t *sums;
    int batch, waves, tiles, tile_rows, slot_rows;
};
struct FoldArgs {
    FoldSide own, prefix;
    int q_len, heads, kv_heads, group;
    int64_t rows;  // batch * q_len * heads
    int merge;     // with a prefix, and every part there
    uint16_t *out;
    float *lse;
};

// The parts of a row: `count` of them, from wave c0's on.
struct Parts {
    const float *o;
    const float2 *ml;
    int64_t o_step, ml_step;  // a slot
    int c0, count, waves, item;
    __device__ __forceinline__ int64_t slot(int i) const { return part_slot(i > 0, i + 1 < count, c0 + i, waves, item); }
};
__device__ __forceinline__ Parts parts_of(const FoldSide &f, int kv_heads, int b, int h, int r) {
    Parts p;
    const int before = f.sums[b], each = f.sums[b + 1] - before, total = f.sums[f.batch];
    const int tile = r / f.tile_rows, at = r - tile * f.tile_rows;
    p.item = b * kv_heads + h;
    p.waves = f.waves;
    p.o_step = (int64_t)f.tiles * f.slot_rows * kD;
    p.ml_step = (int64_t)f.tiles * f.slot_rows;
    p.o = f.part_o + ((int64_t)tile * f.slot_rows * kD + at * 16);
    p.ml = f.part_ml + ((int64_t)tile * f.slot_rows + at);
    p.c0 = p.count = 0;
    if (each > 0) {
        const Cut cut = list_cut(total * kv_heads, f.waves);
        const int u = before * kv_heads + h * each;
        p.c0 = cut_chunk(cut, u);
        p.count = cut_chunk(cut, u + each - 1) - p.c0 + 1;
    }
    return p;
}

// 32 lanes hold a row's dims, lane (j, g) dims 32 g + 4 j .. + 3; PG such groups share its parts.
template <int DT, int PG>
__global__ __launch_bounds__(256) void kv4_combine_kernel(FoldArgs a) {
    constexpr int kBlockRows = 8 / PG;
    const int group = threadIdx.x >> 5, lane = threadIdx.x & 31, pg = group % PG, g4 = lane & 3, j = lane >> 2;
    const int64_t row = (int64_t)blockIdx.x * kBlockRows + group / PG;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    bool done = row >= a.rows;  // or written by the wave that had all of it
    if (!done) {
        const int64_t t = row / a.heads;
        const int head = (int)(row - t * a.heads), b = (int)(t / a.q_len), tok = (int)(t - (int64_t)b * a.q_len);
        const int h = head / a.group, hg = head - h * a.group;
        auto fold = [&](const Parts &p, int slot_rows) {
            constexpr int kBatch = 4;
            for (int i0 = pg; i0 < p.count; i0 += kBatch * PG) {
                f32x4 po[kBatch];
                float2 ml[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const int64_t slot = p.slot(min(i0 + i * PG, p.count - 1));
                    ml[i] = p.ml[slot * p.ml_step];
                    po[i] = *reinterpret_cast<const f32x4 *>(p.o + slot * p.o_step + (int64_t)j * slot_rows * 16 + 4 * g4);
                }
                float top = m;
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    if (i0 + i * PG < p.count) top = fmaxf(top, ml[i].x);
                const float old = m == -INFINITY ? 0.f : exp2_fast(m - top);
                l *= old;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] *= old;
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    if (i0 + i * PG >= p.count) continue;
                    const float f = ml[i].x == -INFINITY ? 0.f : exp2_fast(ml[i].x - top);
                    l = fmaf(ml[i].y, f, l);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = fmaf(po[i][e], f, o[e]);
                }
                m = top;
            }
        };
        const Parts own = parts_of(a.own, a.kv_heads, b, h, tok * a.group + hg);
        done = own.count == 1 && !a.merge;
        if (!done) fold(own, a.own.slot_rows);
        if (a.merge) fold(parts_of(a.prefix, a.kv_heads, 0, h, b * a.group + hg), a.prefix.slot_rows);
    }
    if constexpr (PG > 1) {
        __shared__ f32x4 part[PG][32];
        __shared__ float2 part_ml[PG];
        part[pg][lane] = o;
        if (lane == 0) part_ml[pg] = make_float2(m, l);
        __syncthreads();
        if (pg > 0) return;
        float top = m;
#pragma unroll
        for (int i = 1; i < PG; ++i) top = fmaxf(top, part_ml[i].x);
        l = 0.f;
        o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < PG; ++i) {
            const float2 ml = part_ml[i];
            const float f = ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - top);
            l = fmaf(ml.y, f, l);
            const f32x4 x = part[i][lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f, o[e]);
        }
        m = top;
    }
    if (done) return;
    using E = Elem<DT>;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const uint2 x = make_uint2(E::pack2(o[0] * inv, o[1] * inv), E::pack2(o[2] * inv, o[3] * inv));
    *reinterpret_cast<uint2 *>(a.out + row * kD + 32 * g4 + 4 * j) = x;
    if (lane == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

int64_t ceil_div(int64_t x, int64_t y) { return (x + y - 1) / y; }
int64_t pad256(int64_t n) { return (n + 255) & ~(int64_t)255; }

// One list over the waves (a call's requests, or its prefix) and its part of the workspace.
struct Side {
    int64_t rows, blocks, tiles, groups, waves, slot_rows, slots;
    int64_t off_sums, off_ml, off_o, end;
};

int plan_side(int64_t batch, int64_t rows, int64_t kv_heads, int64_t kv_cap, bool merge, int64_t at, Side *p) {
    p->rows = rows;
    p->blocks = rows <= 16 ? 1 : 2;
    p->tiles = ceil_div(rows, 16 * p->blocks);
    p->groups = kGroups;
    if (p->groups * kWaves < p->tiles) p->groups = ceil_div(p->tiles, kWaves);
    if (!grid_fits(p->groups, kThreads)) return CK_E_INVALID_ARG;
    p->waves = p->groups * kWaves / p->tiles;
    // the list's places are 32-bit, and its shares' numbers
    if (batch * kv_heads >= (int64_t)1 << 31 || batch * kv_heads * ceil_div(kv_cap, kUnit) >= (int64_t)1 << 31)
        return CK_E_INVALID_ARG;
    p->slot_rows = rows < 16 * p->blocks ? rows : 16 * p->blocks;
    p->slots = (2 * p->waves + (merge ? batch * kv_heads : 0)) * p->tiles;
    p->off_sums = at;
    p->off_ml = p->off_sums + pad256((batch + 1) * 4);
    p->off_o = p->off_ml + pad256(p->slots * p->slot_rows * 8);
    p->end = p->off_o + p->slots * p->slot_rows * kD * 4;
    return CK_OK;
}

struct Plan {
    Side own, prefix;
    int64_t ws_bytes;
};

int make_plan(int64_t batch, int64_t q_len, int64_t heads, int64_t kv_heads, int64_t kv_cap, bool merge,
              int64_t prefix_cap, Plan *p) {
    if (batch < 0 || q_len < 1 || heads < 1 || kv_heads < 1 || kv_cap < 0 || prefix_cap < 0) return CK_E_INVALID_ARG;
    if (batch > (1 << 24) || q_len > (1 << 24) || heads > (1 << 16) || kv_heads > (1 << 10) || heads % kv_heads != 0 ||
        kv_cap > ((int64_t)1 << 30) || prefix_cap > ((int64_t)1 << 30) || batch * q_len >= ((int64_t)1 << 31) / heads ||
        !grid_fits(batch * q_len * heads, 256))
        return CK_E_INVALID_ARG;
    const int64_t group = heads / kv_heads;
    int rc = plan_side(batch, q_len * group, kv_heads, kv_cap, merge, 0, &p->own);
    if (rc != CK_OK) return rc;
    p->ws_bytes = p->own.end;
    if (merge && batch > 0) {
        rc = plan_side(1, batch * group, kv_heads, prefix_cap, true, p->own.end, &p->prefix);
        if (rc != CK_OK) return rc;
        p->ws_bytes = p->prefix.end;
    }
    return CK_OK;
}

template <int DT>
int launch_side(const DecodeArgs &a, const Side &p, hipStream_t s) {
    const dim3 grid((unsigned)p.groups), block(kThreads);
    if (p.blocks == 1) hipLaunchKernelGGL((kv4_decode_kernel<DT, 1>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((kv4_decode_kernel<DT, 2>), grid, block, 0, s, a);
    CK_RETURN_LAUNCH();
}

template <int DT>
int launch(const DecodeArgs &own, const DecodeArgs *prefix, const Plan &p, const FoldArgs &f, hipStream_t s) {
    if (prefix) {
        const int rc = launch_side<DT>(*prefix, p.prefix, s);
        if (rc != CK_OK) return rc;
    }
    const int rc = launch_side<DT>(own, p.own, s);
    if (rc != CK_OK) return rc;
    if (f.rows >= kFoldRows)
        hipLaunchKernelGGL((kv4_combine_kernel<DT, 1>), dim3((unsigned)ceil_div(f.rows, 8)), dim3(256), 0, s, f);
    else
        hipLaunchKernelGGL((kv4_combine_kernel<DT, 8>), dim3((unsigned)f.rows), dim3(256), 0, s, f);
    CK_RETURN_LAUNCH();
}

struct Pool {
    const void *cache;
    const int32_t *bt;
    const int64_t *lens;
    int64_t cols, num_blocks;
};
int check_pool(const Pool &p) {
    if (p.num_blocks < 0 || p.num_blocks > ((int64_t)1 << 31)) return CK_E_INVALID_ARG;
    if (!p.lens || (p.cols > 0 && (!p.bt || (p.num_blocks > 0 && !p.cache)))) return CK_E_NULL_PTR;
    return aligned_to(p.cache, 16) && aligned_to(p.bt, 4) && aligned_to(p.lens, 8) ? CK_OK : CK_E_INVALID_ARG;
}

void fill(DecodeArgs *a, FoldSide *f, const Pool &pool, const Side &p, int64_t batch, char *ws) {
    a->cache = static_cast<const uint8_t *>(pool.cache);
    a->bt = pool.bt;
    a->lens = pool.lens;
    a->bt_cols = pool.cols;
    a->num_blocks = pool.num_blocks;
    a->batch = (int)batch;
    a->rows = (int)p.rows;
    a->tiles = (int)p.tiles;
    a->waves = (int)p.waves;
    a->part_o = reinterpret_cast<float *>(ws + p.off_o);
    a->part_ml = reinterpret_cast<float2 *>(ws + p.off_ml);
    a->sums = reinterpret_cast<int32_t *>(ws + p.off_sums);
    *f = FoldSide{a->part_o, a->part_ml, a->sums, a->batch, a->waves, a->tiles, (int)(16 * p.blocks), (int)p.slot_rows};
}

int run(const void *q, const Pool &pool, const Pool *prefix, int64_t batch, int64_t q_len, int64_t heads,
        int64_t kv_heads, int64_t block_size, int dtype, float scale, void *out, float *lse, void *workspace,
        int64_t workspace_bytes, hipStream_t s) {
    auto tokens_of = [](int64_t cols) { return cols < 0 ? -1 : (cols > ((int64_t)1 << 30) ? (int64_t)1 << 30 : cols) * kPage; };
    Plan p;
    int rc = make_plan(batch, q_len, heads, kv_heads, tokens_of(pool.cols), prefix != nullptr,
                       prefix ? tokens_of(prefix->cols) : 0, &p);
    if (rc != CK_OK) return rc;
    if (block_size != kPage || (dtype != CK_DTYPE_BF16 && dtype != CK_DTYPE_F16)) return CK_E_UNSUPPORTED;
    // the kernels work with scale log2(e)
    if (!(scale > 0.f) || !std::isfinite(scale * kLog2e)) return CK_E_INVALID_ARG;
    if (batch == 0) return CK_OK;
    if (!q || !out || !lse) return CK_E_NULL_PTR;
    if ((rc = check_pool(pool)) != CK_OK || (prefix && (rc = check_pool(*prefix)) != CK_OK)) return rc;
    if (!aligned_to(q, 16) || !aligned_to(out, 16) || !aligned_to(lse, 4) || !aligned_to(workspace, 16))
        return CK_E_INVALID_ARG;
    if (!workspace || workspace_bytes < p.ws_bytes) return CK_E_WORKSPACE;

    DecodeArgs a = {}, b = {};
    FoldArgs f = {};
    char *ws = static_cast<char *>(workspace);
    a.q = static_cast<const uint16_t *>(q);
    a.heads = (int)heads;
    a.kv_heads = (int)kv_heads;
    a.group = (int)(heads / kv_heads);
    a.merge = prefix != nullptr;
    a.scale_log2 = scale * kLog2e;
    a.out = static_cast<uint16_t *>(out);
    a.lse = lse;
    b = a;
    a.q_len = (int)q_len;
    a.causal = q_len > 1;
    fill(&a, &f.own, pool, p.own, batch, ws);
    if (prefix) {  // one request, the batch's tokens in it, none hidden from another
        b.q_len = (int)batch;
        fill(&b, &f.prefix, *prefix, p.prefix, 1, ws);
    }
    f.q_len = (int)q_len;
    f.heads = a.heads;
    f.kv_heads = a.kv_heads;
    f.group = a.group;
    f.rows = batch * q_len * heads;
    f.merge = a.merge;
    f.out = a.out;
    f.lse = lse;
    return dtype == CK_DTYPE_BF16 ? launch<CK_DTYPE_BF16>(a, prefix ? &b : nullptr, p, f, s)
                                  : launch<CK_DTYPE_F16>(a, prefix ? &b : nullptr, p, f, s);
}

}  // namespace
}  // namespace ck

using namespace ck;

extern "C" int ck_kv4_decode_plan(int64_t batch, int64_t q_len, int64_t num_heads, int64_t kv_heads, int64_t kv_cap,
                                  int64_t *workspace_bytes) {
    if (!workspace_bytes) return CK_E_NULL_PTR;
    Plan p;
    int rc = make_plan(batch, q_len, num_heads, kv_heads, kv_cap, false, 0, &p);
    if (rc == CK_OK) *workspace_bytes = p.ws_bytes;
    return rc;
}

extern "C" int ck_kv4_decode(const void *q, const void *cache, const int32_t *block_table, int64_t bt_cols,
                             const int64_t *kv_seqlens, int64_t batch, int64_t q_len, int64_t num_heads,
                             int64_t kv_heads, int64_t num_blocks, int64_t block_size, int dtype, float scale, void *out,
                             float *lse, void *workspace, int64_t workspace_bytes, void *stream) {
    const Pool pool{cache, block_table, kv_seqlens, bt_cols, num_blocks};
    return run(q, pool, nullptr, batch, q_len, num_heads, kv_heads, block_size, dtype, scale, out, lse, workspace,
               workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int ck_kv4_cascade_decode_plan(int64_t batch, int64_t num_heads, int64_t kv_heads, int64_t prefix_cap,
                                          int64_t suffix_cap, int64_t *workspace_bytes) {
    if (!workspace_bytes) return CK_E_NULL_PTR;
    Plan p;
    int rc = make_plan(batch, 1, num_heads, kv_heads, suffix_cap, true, prefix_cap, &p);
    if (rc == CK_OK) *workspace_bytes = p.ws_bytes;
    return rc;
}

extern "C" int ck_kv4_cascade_decode(const void *q, const void *prefix_cache, const int32_t *prefix_block_table,
                                     int64_t prefix_bt_cols, const int64_t *prefix_kv_seqlen,
                                     int64_t prefix_num_blocks, const void *suffix_cache,
                                     const int32_t *suffix_block_table, int64_t suffix_bt_cols,
                                     const int64_t *suffix_kv_seqlens, int64_t suffix_num_blocks, int64_t batch,
                                     int64_t num_heads, int64_t kv_heads, int64_t block_size, int dtype, float scale,
                                     void *out, float *lse, void *workspace, int64_t workspace_bytes, void *stream) {
    const Pool suffix{suffix_cache, suffix_block_table, suffix_kv_seqlens, suffix_bt_cols, suffix_num_blocks};
    const Pool prefix{prefix_cache, prefix_block_table, prefix_kv_seqlen, prefix_bt_cols, prefix_num_blocks};
    return run(q, suffix, &prefix, batch, 1, num_heads, kv_heads, block_size, dtype, scale, out, lse, workspace,
               workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}
