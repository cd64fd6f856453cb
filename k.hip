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
#include "latent_common.h"

namespace ck {
namespace {
__device__ unsigned long long g_st[4096*16];
#define ST(k) do { if (threadIdx.x % 64 == 0 && (threadIdx.x >> 6) == 0) g_st[blockIdx.x * 16 + (k)] = wall_clock64(); } while (0)
using namespace kv4;

typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kGroups = 512;  // workgroups: two per CU
constexpr int kGroupsWide = 256;  // of many rows: one per CU
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
    int tile_rows;
    int waves;   // shares of the list (waves', or with many rows workgroups'), per row tile
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

// The arguments, read where they are used: held in scalar registers throughout they would spill.
typedef const __attribute__((address_space(4))) DecodeArgs *KernArgs;
__device__ __forceinline__ KernArgs args_again(KernArgs a) {
    asm volatile("" : "+s"(a));
    return a;
}
// The lane, so that what depends on it is computed where it is used.
__device__ __forceinline__ int lane_again(int lane) {
    asm volatile("" : "+v"(lane));
    return lane;
}

__device__ __forceinline__ int len_of(KernArgs a, int b) {
    const int64_t cap = a->bt_cols * kPage;
    int64_t n = a->lens[b];
    if (n > cap) n = cap;
    return n < 0 || a->num_blocks <= 0 ? 0 : (int)n;
}
__device__ __forceinline__ int units_of(int len) { return (len + kUnit - 1) / kUnit; }

// starts[t]: units (of one kv head) before thread t's requests, t's share of the batch. Returns their number in
// all; the first workgroup leaves those before each request for the fold.
template <int T>
__device__ __forceinline__ int requests_per_thread(KernArgs a) { return (a->batch + T - 1) / T; }
template <int T>
__device__ __forceinline__ int list_starts(KernArgs a, int *starts, int *scan, int tid) {
    const int per = requests_per_thread<T>(a), b0 = min(tid * per, a->batch), b1 = min(b0 + per, a->batch);
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += units_of(len_of(a, b));
    const int incl = (int)wave_scan((uint32_t)mine, 0x7fffffffu);
    if ((tid & 63) == 63) scan[tid >> 6] = incl;
    __syncthreads();
    int start = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) {
        if (w < tid >> 6) start += scan[w];
        total += scan[w];
    }
    starts[tid] = start;
    if (blockIdx.x == 0) {
        int at = start;
        for (int b = b0; b < b1; ++b) {
            a->sums[b] = at;
            at += units_of(len_of(a, b));
        }
        if (tid == 0) a->sums[a->batch] = total;
    }
    __syncthreads();
    return total;
}
// The request that holds place u of the list, its first place and its length.
struct Found {
    int b, at, len;
};
template <int T>
__device__ __forceinline__ Found find_request(KernArgs a, const int *starts, int u) {
    int x = 0;  // the last thread whose requests begin at or before u
#pragma unroll
    for (int step = T / 2; step > 0; step >>= 1)
        if (starts[x + step] * a->kv_heads <= u) x += step;
    Found f;
    f.b = min(x * requests_per_thread<T>(a), a->batch - 1);
    f.at = starts[x] * a->kv_heads;
    f.len = len_of(a, f.b);
    while (f.b + 1 < a->batch && f.at + units_of(f.len) * a->kv_heads <= u) {  // of the thread's
        f.at += units_of(f.len) * a->kv_heads;
        f.len = len_of(a, ++f.b);
    }
    return f;
}
// A unit's place in memory; bit 0 (addresses are 16-byte aligned) marks a page outside the pool.
__device__ __forceinline__ uint64_t unit_address(KernArgs a, int b, int h, int i) {
    const int page = a->bt[(int64_t)b * a->bt_cols + (i >> 1)];
    const bool ok = page >= 0 && page < a->num_blocks;
    return (uint64_t)(uintptr_t)a->cache + (ok ? (((uint64_t)(uint32_t)page * a->kv_heads + h) * 2 + (i & 1)) * kUnitBytes : 1);
}
__device__ __forceinline__ uint64_t of_lane(uint64_t x, int lane) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)x, lane);
}

// A unit as a wave's lanes hold it: lane (g, n) has group g of keys 8 (n / 4) + n % 4 + {0, 4, 32, 36}
// and their scales, dims 8 n + 2 q, + 1 of values 8 g .. + 7 and 32 + 8 g .. + 7, and these tokens' scales of dim
// group n / 4.
struct Unit {
    u32x4 k[4], v[4], vs;
    uint32_t ks;
    __device__ __forceinline__ u32x4 keys(int t) const { return k[t]; }
    __device__ __forceinline__ u32x4 values(int q) const { return v[q]; }
};
// A unit in LDS, its pieces in the lanes' order: what is needed is read where it is.
struct UnitInLds {
    const CK_LDS char *at;  // the lane's
    u32x4 vs;
    uint32_t ks;
    __device__ __forceinline__ u32x4 keys(int t) const { return *reinterpret_cast<const CK_LDS u32x4 *>(at + 1024 * t); }
    __device__ __forceinline__ u32x4 values(int q) const { return *reinterpret_cast<const CK_LDS u32x4 *>(at + kVAt + 1024 * q); }
};
// The same in the compiler's eyes new: what one of two ways through computes from it is not made before them, for
// both.
__device__ __forceinline__ u32x4 again(u32x4 x) {
    asm volatile("" : "+v"(x));
    return x;
}
constexpr int kSlotBytes = 9216;  // a unit in LDS: 9 moves of 1 KB, the last of which its scales half fill
constexpr int kPieces = 9;
// Lane offsets of a unit's moves: of the keys (tile t at + 0, 256, 2048, 2304), of what lies in the lanes' order, and
// of the scales (the upper lanes' are out of range).
struct MoveOffsets {
    int keys, linear, last;
    __device__ __forceinline__ explicit MoveOffsets(int lane)
        : keys((8 * ((lane & 15) >> 2) + (lane & 3)) * 64 + 16 * (lane >> 4)), linear(16 * lane),
          last(lane < 32 ? 16 * lane : kUnitBytes) {}
};
// The unit at `at` (unit_address) to LDS; from a page outside the pool, zeros.
__device__ __forceinline__ void move_unit(uint64_t at, const MoveOffsets &off, const CK_LDS char *slot) {
    const ck_rsrc_t r = {(int)(uint32_t)(at & ~1ull), (int)((uint32_t)(at >> 32) & 0xffffu), at & 1 ? 0 : kUnitBytes,
                         (int)kRsrcFlags};
    const int base = scalar((int)(uint32_t)(uintptr_t)slot);
    static_for<kPieces>([&](auto p) __attribute__((always_inline)) {
        constexpr int P = p;
        if constexpr (P < 4) lat::dma_tile<1024 * P>(r, off.keys, (P >> 1) * 2048 + (P & 1) * 256, base);
        else lat::dma_tile<1024 * P>(r, P < 8 ? off.linear : off.last, 1024 * P, base);
    });
}
__device__ __forceinline__ UnitInLds unit_in(const CK_LDS char *slot, int lane) {
    UnitInLds u;
    u.at = slot + 16 * lane;
    u.ks = *reinterpret_cast<const CK_LDS uint32_t *>(slot + kKsAt + 4 * lane);
    u.vs = *reinterpret_cast<const CK_LDS u32x4 *>(slot + kVsAt + ((lane & 15) >> 2) * 64 + 16 * (lane >> 4));
    return u;
}

__device__ __forceinline__ void load_unit(Unit &u, uint64_t at, int lane) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<char *>((uintptr_t)(at & ~1ull)), (short)0,
                                                                       at & 1 ? 0 : kUnitBytes, kRsrcFlags);
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

// How a wave of NB row blocks computes. One row block is bound by memory: P enters the second product as two
// bf16 terms, within 2^-17 of fp32, an fp16 query the first as two bf16 terms, which hold all of it. More row blocks
// are bound by arithmetic: where a unit's scales lie in [2^-23, 2^8] fp16 holds every value, and P is one fp16
// number, 2^7 p (fp16's normal range ends at 2^-14; with the largest score at most 2^kSlack past the reference
// point 2^7 p stays below 65504), half a step off, 2^-12; so does an fp16 query's key. Units of other scales are
// computed as above. 24 x 3 x 64 heads over 5000 tokens (fp16): FILL.
template <int DT, int NB>
struct Form {
    static constexpr bool kHalf = NB > 1;
    static constexpr int kTerms = DT == CK_DTYPE_F16 && !kHalf ? 2 : 1;  // of the query, as it is held
    static constexpr float kBias = kHalf ? 7.f : 0.f;
};

// The rows of a wave: row 16 i + n in lanes (g, n).
template <int DT, int NB>
struct Rows {
    u32x4 q[NB][Form<DT, NB>::kTerms][4];  // dims 32 g + 8 c .. + 7
    f32x4 o[NB][8];  // O^T: dims 32 g + 8 r + block of the row
    float m[NB];     // the sum's reference point (log2; the same for all g) is m - kBias
    float l[NB];     // this lane's share of the sum
};
template <int DT, int NB>
__device__ __forceinline__ void clear(Rows<DT, NB> &s) {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int k = 0; k < 8; ++k) s.o[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
        s.m[i] = -INFINITY;
        s.l[i] = 0.f;
    }
}

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 x, u32x4 y, f32x4 c) { return Elem<CK_DTYPE_BF16>::mfma16(x, y, c); }
__device__ __forceinline__ f32x4 mfma_f16(u32x4 x, u32x4 y, f32x4 c) { return Elem<CK_DTYPE_F16>::mfma16(x, y, c); }

// fp16 numbers as two bf16 terms.
__device__ __forceinline__ void two_terms(u32x4 x, u32x4 &hi, u32x4 &lo) {
    using E = Elem<CK_DTYPE_F16>;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        hi[e] = pack_bf16x2(E::lo(x[e]), E::hi(x[e]));
        lo[e] = pack_bf16x2(E::lo(x[e]) - bf16_lo(hi[e]), E::hi(x[e]) - bf16_hi(hi[e]));
    }
}

// Nonzero where a scale byte of w is outside [104, 135] (2^-23 to 2^8).
constexpr uint32_t kMidScales = 0x68686868;
__device__ __forceinline__ uint32_t past_half(uint32_t w) { return ((w + 0x18181818) ^ 0x80808080) & 0xe0e0e0e0; }

// Scores of a unit's 16 tokens t, HALF: of fp16 numbers.
template <bool HALF, int DT, int NB>
__device__ __forceinline__ void add_scores(const Rows<DT, NB> &s, const u32x4 &codes, float scale, f32x4 (&sc)[NB][4], int t) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t w = codes[c];
        u32x4 a;
        if constexpr (HALF) a = u32x4{pair_f16<0>(w, scale), pair_f16<1>(w, scale), pair_f16<2>(w, scale), pair_f16<3>(w, scale)};
        else a = u32x4{pair_bf16<0>(w, scale), pair_bf16<1>(w, scale), pair_bf16<2>(w, scale), pair_bf16<3>(w, scale)};
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if constexpr (HALF) {
                sc[i][t] = mfma_f16(a, s.q[i][0][c], sc[i][t]);
            } else if constexpr (DT == CK_DTYPE_F16 && Form<DT, NB>::kTerms == 1) {
                u32x4 hi, lo;
                two_terms(s.q[i][0][c], hi, lo);
                sc[i][t] = mfma_bf16(a, hi, sc[i][t]);
                sc[i][t] = mfma_bf16(a, lo, sc[i][t]);
            } else {
#pragma unroll
                for (int x = 0; x < Form<DT, NB>::kTerms; ++x) sc[i][t] = mfma_bf16(a, s.q[i][x][c], sc[i][t]);
            }
        }
    }
    __builtin_amdgcn_sched_barrier(0);
}
template <bool HALF, int DT, int NB>
__device__ __forceinline__ void add_scores(const Rows<DT, NB> &s, const u32x4 (&k)[4], uint32_t ks, f32x4 (&sc)[NB][4]) {
    add_scores<HALF>(s, k[0], scale_of<0>(ks), sc, 0);
    add_scores<HALF>(s, k[1], scale_of<1>(ks), sc, 1);
    add_scores<HALF>(s, k[2], scale_of<2>(ks), sc, 2);
    add_scores<HALF>(s, k[3], scale_of<3>(ks), sc, 3);
}

// P of row blocks I0 .. I0 + N - 1 over a unit, its sums, and O^T += V^T P^T; vs: the values' scales.
template <bool HALF, int I0, int N, int DT, int NB>
__device__ __forceinline__ void add_values(Rows<DT, NB> &s, const u32x4 (&v)[4], u32x4 vs, const f32x4 (&sc)[NB][4], float scale_log2) {
    constexpr int kParts = HALF ? 1 : 2;
    u32x4 p[N][kParts][2];  // [term][half of the tokens]
    asm volatile("" : "+s"(scale_log2));  // not the other form's exponentials
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int i = I0 + k;
        const float sub = s.m[i] == -INFINITY ? 0.f : s.m[i] - Form<DT, NB>::kBias;
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = exp2_fast(fmaf(sc[i][e >> 1][2 * (e & 1)], scale_log2, -sub));
            const float y = exp2_fast(fmaf(sc[i][e >> 1][2 * (e & 1) + 1], scale_log2, -sub));
            sum += x;
            sum += y;
            if constexpr (HALF) {
                p[k][0][e >> 2][e & 3] = Elem<CK_DTYPE_F16>::pack2(x, y);
            } else {
                const uint32_t h = pack_bf16x2(x, y);
                p[k][0][e >> 2][e & 3] = h;
                p[k][kParts - 1][e >> 2][e & 3] = pack_bf16x2(x - bf16_lo(h), y - bf16_hi(h));
            }
        }
        s.l[i] += sum;
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float f[8];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            f[4 * w] = scale_of<0>(vs[2 * h + w]);
            f[4 * w + 1] = scale_of<1>(vs[2 * h + w]);
            f[4 * w + 2] = scale_of<2>(vs[2 * h + w]);
            f[4 * w + 3] = scale_of<3>(vs[2 * h + w]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            u32x4 even, odd;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const uint32_t c = v[q][2 * h + w];
                uint32_t t[4];
                if constexpr (HALF) {
                    t[0] = pair_f16<0>(c, f[4 * w]), t[1] = pair_f16<1>(c, f[4 * w + 1]);
                    t[2] = pair_f16<2>(c, f[4 * w + 2]), t[3] = pair_f16<3>(c, f[4 * w + 3]);
                } else {
                    t[0] = pair_bf16<0>(c, f[4 * w]), t[1] = pair_bf16<1>(c, f[4 * w + 1]);
                    t[2] = pair_bf16<2>(c, f[4 * w + 2]), t[3] = pair_bf16<3>(c, f[4 * w + 3]);
                }
                even[2 * w] = __builtin_amdgcn_perm(t[1], t[0], 0x05040100);
                odd[2 * w] = __builtin_amdgcn_perm(t[1], t[0], 0x07060302);
                even[2 * w + 1] = __builtin_amdgcn_perm(t[3], t[2], 0x05040100);
                odd[2 * w + 1] = __builtin_amdgcn_perm(t[3], t[2], 0x07060302);
            }
#pragma unroll
            for (int x = 0; x < kParts; ++x)
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    f32x4 &lo = s.o[I0 + k][2 * q], &hi = s.o[I0 + k][2 * q + 1];
                    if constexpr (HALF) {
                        lo = mfma_f16(even, p[k][x][h], lo);
                        hi = mfma_f16(odd, p[k][x][h], hi);
                    } else {
                        lo = mfma_bf16(even, p[k][x][h], lo);
                        hi = mfma_bf16(odd, p[k][x][h], hi);
                    }
                }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// The first n bytes of w, the others `rest`.
__device__ __forceinline__ uint32_t first_bytes(uint32_t w, int n, uint32_t rest) {
    const uint32_t mask = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
    return (w & mask) | (rest & ~mask);
}

// The values' scales of a unit that not every row sees whole. Those of tokens from `left` on go, and values that
// are not numbers would reach rows that do not see them (0 times them is none): their scales become
// ordinary ones, and rows that do see one get it added. A lane (g, n) has the dims of group g of its rows' O.
template <int NB>
__device__ __forceinline__ void hide_values(f32x4 (&o)[NB][8], u32x4 &vs, const int (&sees)[NB], int left, int g) {
    int first_bad = kUnit;
#pragma unroll
    for (int w = 3; w >= 0; --w) {
        const int t0 = 32 * (w >> 1) + 8 * g + 4 * (w & 1);
        vs[w] = first_bytes(vs[w], left - t0, kMidScales);
#pragma unroll
        for (int b = 3; b >= 0; --b) {
            if (((vs[w] >> (8 * b)) & 0xff) != kBad) continue;
            first_bad = t0 + b;
            vs[w] ^= (kBad ^ (kMidScales & 0xff)) << (8 * b);
        }
    }
    if (__builtin_expect(!__builtin_amdgcn_ballot_w64(first_bad < kUnit), 1)) return;
    first_bad = (int)over_groups((float)first_bad, [](float x, float y) { return fminf(x, y); });
    first_bad = __shfl(first_bad, 4 * g);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        if (first_bad >= sees[i]) continue;
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[i][k][r] = NAN;
    }
}

// One unit. Where tail: tokens from sees[i] on are hidden from row block i's row, those from `left` on
// (counted from the unit's first) hold anything.
template <int DT, int NB, class U>
__device__ __forceinline__ void compute(Rows<DT, NB> &s, const U &u, float scale_log2, int lane, bool tail,
                                        const int (&sees)[NB], int left) {
    constexpr bool kHalf = Form<DT, NB>::kHalf, kHalfKeys = kHalf && DT == CK_DTYPE_F16;
    u32x4 k[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) k[t] = u.keys(t);
    f32x4 sc[NB][4];
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) sc[i][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (kHalfKeys && __builtin_expect(!__builtin_amdgcn_ballot_w64(past_half(u.ks) != 0), 1)) add_scores<true>(s, k, u.ks, sc);
    else add_scores<false>(s, k, u.ks, sc);
    u32x4 vs = u.vs, v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = u.values(q);
    if (__builtin_expect(tail, 0)) {
        const int g = lane_again(lane) >> 4;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int n = sees[i] - 8 * g;  // token of sc[i][t][r]: 32 (t / 2) + 8 g + 4 (t % 2) + r
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (32 * (e >> 3) + (e & 7) >= n) sc[i][e >> 2][e & 3] = -INFINITY;
        }
        hide_values<NB>(s.o, vs, sees, left, g);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        float most = max3(sc[i][0][0], sc[i][0][1], sc[i][0][2]);
#pragma unroll
        for (int e = 3; e < 15; e += 2) most = max3(most, sc[i][e >> 2][e & 3], sc[i][(e + 1) >> 2][(e + 1) & 3]);
        most = fmaxf(most, sc[i][3][3]) * scale_log2;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(most > s.m[i] + kSlack) != 0, 0)) {
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
    }
    if (kHalf && __builtin_expect(!__builtin_amdgcn_ballot_w64((past_half(vs[0]) | past_half(vs[1]) | past_half(vs[2]) | past_half(vs[3])) != 0), 1))
        add_values<true, 0, NB>(s, v, vs, sc, scale_log2);
    else
        add_values<false, 0, NB>(s, v, again(vs), sc, scale_log2);
}

template <int DT, int NB>
__global__ __launch_bounds__(kThreads, 2) void kv4_decode_kernel(DecodeArgs) {
    const KernArgs args = (KernArgs)__builtin_amdgcn_kernarg_segment_ptr();
    KernArgs a = args_again(args);
    __shared__ int starts[kThreads], scan[kWaves];
    __shared__ __attribute__((aligned(16))) char ring[NB > 1 ? kWaves * 2 * kSlotBytes : 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6);
    constexpr int kRows = 16 * NB;
    constexpr bool kQAhead = NB == 1;  // the next item's queries are loaded ahead

    const int total = scalar(list_starts<kThreads>(a, starts, scan, tid));

    // ---- this wave's share ---------------------------------------------------------------------------
    // neighbouring shares on different CUs, so that few units spread over all of them
    const int w = scalar(wave * (int)gridDim.x + (int)blockIdx.x);
    const Cut cut = list_cut(total * a->kv_heads, a->waves);
    if (w >= cut.chunks) return;
    const int lo = scalar(cut_lo(cut, w)), hi = scalar(cut_lo(cut, w + 1));
    const int slot_rows = min(kRows, a->rows);

    const MoveOffsets off(lane);
    Rows<DT, NB> s;
    u32x4 next_q[NB][4];
    int tok[NB];  // of row block i's row, among the request's
#pragma unroll
    for (int i = 0; i < NB; ++i) tok[i] = (16 * i + (lane & 15)) / a->group;

    auto load_q = [&](int item) {
        const KernArgs a = args_again(args);
        const int b = scalar(item / a->kv_heads), h = item - b * a->kv_heads;
        const int x = lane_again(lane), n16 = x & 15, g4 = x >> 4;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int r = 16 * i + n16;
            const uint16_t *p = a->q + (((int64_t)b * a->q_len + tok[i]) * a->heads + h * a->group + (r - tok[i] * a->group)) * kD + 32 * g4;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                next_q[i][c] = u32x4{0, 0, 0, 0};
                if (r < a->rows) next_q[i][c] = *reinterpret_cast<const u32x4 *>(p + 8 * c);
            }
        }
    };
    auto open_item = [&](int item) {
        if constexpr (!kQAhead) load_q(item);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                constexpr int kTerms = Form<DT, NB>::kTerms;
                if constexpr (kTerms == 1) s.q[i][0][c] = next_q[i][c];
                else two_terms(next_q[i][c], s.q[i][0][c], s.q[i][kTerms - 1][c]);
            }
        }
        clear(s);
    };
    auto close_item = [&](int item, bool before, bool after) {
        const KernArgs a = args_again(args);
        const int b = scalar(item / a->kv_heads), h = item - b * a->kv_heads;
        const int x = lane_again(lane), n16 = x & 15, g4 = x >> 4;
        const bool whole = !before && !after && !a->merge;
        const int64_t slot = part_slot(before, after, w, a->waves, item);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int r = 16 * i + n16;
            const float l = over_groups(s.l[i], [](float x, float y) { return x + y; }), m = s.m[i] - Form<DT, NB>::kBias;
            if (r >= a->rows) continue;
            if (whole) {
                using E = Elem<DT>;
                const int64_t row = ((int64_t)b * a->q_len + tok[i]) * a->heads + h * a->group + (r - tok[i] * a->group);
                const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    u32x4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = E::pack2(s.o[i][2 * e][d] * inv, s.o[i][2 * e + 1][d] * inv);
                    *reinterpret_cast<u32x4 *>(a->out + row * kD + 32 * g4 + 8 * d) = x;
                }
                if (g4 == 0) a->lse[row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
            } else {
                const int at = 16 * i + n16;
                float *p = a->part_o + slot * slot_rows * kD;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // dims 32 g + 4 j + e: 8 (j / 2) + block 4 (j % 2) + e
                    const f32x4 x = {s.o[i][4 * (j & 1)][j >> 1], s.o[i][4 * (j & 1) + 1][j >> 1],
                                     s.o[i][4 * (j & 1) + 2][j >> 1], s.o[i][4 * (j & 1) + 3][j >> 1]};
                    *reinterpret_cast<f32x4 *>(p + ((j * slot_rows + at) * 4 + g4) * 4) = x;
                }
                if (g4 == 0) a->part_ml[slot * slot_rows + at] = make_float2(m, l);
            }
        }
    };

    // ---- the units, 64 described at a time: one a lane ---------------------------------------------------
    int item = -1;
    bool before = false, goes_on = false;  // the open item: begun in an earlier share; its last unit not seen yet
    for (int base = lo; base < hi; base += 64) {
        a = args_again(args);
        const int n = min(64, hi - base);
        int d_item = 0, d_first = 0, d_len = 0;
        uint64_t d_at = 0;
        if (lane < n) {
            const int u = base + lane;
            const Found f = find_request<kThreads>(a, starts, u);
            const int each = units_of(f.len), h = (u - f.at) / each, i = u - f.at - h * each;
            d_item = f.b * a->kv_heads + h;
            d_first = i * kUnit;
            d_len = f.len;
            d_at = unit_address(a, f.b, h, i);
        }
        // One row block: the next unit in registers; more: in the wave's other half of its ring.
        Unit next;
        CK_LDS char *slots = (CK_LDS char *)ring + (NB > 1 ? wave * 2 * kSlotBytes : 0);
        auto fetch = [&](int j) {
            const uint64_t at = of_lane(d_at, j);
            if constexpr (NB > 1) move_unit(at, off, slots + (j & 1) * kSlotBytes);
            else load_unit(next, at, lane);
        };
        fetch(0);
        if (const int first = __builtin_amdgcn_readlane(d_item, 0); kQAhead && first != item) load_q(first);
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
            const Unit in_registers = next;
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
                fetch(j + 1);
                if (const int then = __builtin_amdgcn_readlane(d_item, j + 1); kQAhead && then != it) load_q(then);
            }
            const int left = len - first, first_sees = a->causal ? left - a->q_len + 1 : left;
            int sees[NB];
#pragma unroll
            for (int i = 0; i < NB; ++i) sees[i] = a->causal ? first_sees + tok[i] : left;
            if constexpr (NB > 1) {
                if (j + 1 < n) wait_vmcnt<kPieces>();
                else wait_vmcnt<0>();
                asm volatile("" ::: "memory");
                compute<DT, NB>(s, unit_in(slots + (j & 1) * kSlotBytes, lane), a->scale_log2, lane, first_sees < kUnit, sees, left);
            } else {
                compute<DT, NB>(s, in_registers, a->scale_log2, lane, first_sees < kUnit, sees, left);
            }
        }
    }
    close_item(item, before, goes_on);
}

// ---- many rows ---------------------------------------------------------------------------------------------
// The same for items of more than 32 rows, on workgroups of 8 waves with a CU to themselves, two waves per SIMD that
// fill each other's waits. A row tile is 32 rows each of 2, 4 or 8 row waves; 4, 2 or 1 such sets take an item's units
// in turn, and their parts are joined in LDS, so that few go to memory. All waves read the units from a ring in
// LDS: 8 units (70 KB) are under way (buffer -> LDS DMA in the operands' order, a unit a wave), one barrier a unit.
// The shares of the list are workgroups'.
constexpr int kWideThreads = 512, kWideWaves = kWideThreads / 64;
constexpr int kAhead = kWideWaves;  // units under way: unit u is moved by wave u % 8
constexpr int kSlots = 15;  // of units under way, computed by up to 4 sets, and some
constexpr int kWidePart = 32 * kD * 4;  // a wave's O, in the ring's place
constexpr int kWideMl = kSlots * kSlotBytes;
constexpr int kWideStarts = kWideMl + kWideWaves * 32 * 8;
constexpr int kWideLds = kWideStarts + (kWideThreads + kWideWaves) * 4;
static_assert(kSlots >= kAhead + 4 && kWideWaves * kWidePart <= kWideMl && kWideLds <= 160 * 1024, "LDS");

template <int DT>
__global__ __launch_bounds__(kWideThreads, 2) void kv4_wide_kernel(DecodeArgs) {
 ST(0);
    const KernArgs args = (KernArgs)__builtin_amdgcn_kernarg_segment_ptr();
    KernArgs a = args_again(args);
    constexpr int NB = 2;
    using E = Elem<DT>;
    extern __shared__ __attribute__((aligned(16))) char wide_raw[];
    CK_LDS char *smem = (CK_LDS char *)wide_raw;
    int *starts = reinterpret_cast<int *>(wide_raw + kWideStarts);
    const int tid = threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6);
    const int total = scalar(list_starts<kWideThreads>(a, starts, starts + kWideThreads, tid));
    const int share = scalar((int)blockIdx.x / a->tiles), tile = scalar((int)blockIdx.x - share * a->tiles);
    const Cut cut = list_cut(total * a->kv_heads, a->waves);
    if (share >= cut.chunks) return;
    ST(1);
    int cur = scalar(cut_lo(cut, share));
    const int hi = scalar(cut_lo(cut, share + 1));
    const int row_waves = a->tile_rows >> 5, sets = kWideWaves / row_waves;  // powers of two
    const int set = wave / row_waves, row0 = a->tile_rows * tile + 32 * (wave - set * row_waves);

    int tok[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) tok[i] = (row0 + 16 * i + (lane & 15)) / a->group;
    const MoveOffsets off(lane);

    Rows<DT, NB> s;
    while (cur < hi) {
        a = args_again(args);
        const Found f = find_request<kWideThreads>(a, starts, cur);
        const int b = scalar(f.b), len = scalar(f.len), each = units_of(len), in = cur - scalar(f.at);
        const int h = scalar(in / each), i0 = in - h * each, i1 = min(each, i0 + hi - cur);
        const int item = b * a->kv_heads + h;
        const bool before = i0 > 0, after = i1 < each;
        cur += i1 - i0;
        {
            const int x = lane_again(lane), n16 = x & 15, g = x >> 4;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int r = row0 + 16 * i + n16;
                const uint16_t *p = a->q + (((int64_t)b * a->q_len + tok[i]) * a->heads + h * a->group + (r - tok[i] * a->group)) * kD + 32 * g;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    s.q[i][0][c] = u32x4{0, 0, 0, 0};
                    if (r < a->rows) s.q[i][0][c] = *reinterpret_cast<const u32x4 *>(p + 8 * c);
                }
            }
            clear(s);
        }
        for (int c0 = i0; c0 < i1; c0 += 64 * kAhead) {
            const int n = min(64 * kAhead, i1 - c0);
            // this wave moves units c0 + wave + 8 x; lane x has the address
            const uint64_t d_at = unit_address(a, b, h, min(c0 + wave + kAhead * lane, i1 - 1));
            auto move = [&](int u) {
                if (u < n) move_unit(of_lane(d_at, u / kAhead), off, smem + u % kSlots * kSlotBytes);
            };
            move(wave);
#pragma unroll 1
            for (int t = 0; t < n; t += sets) {
                // a wave has one unit under way: that of this step has landed before the barrier, the next one
                // goes into a slot that all waves have left by it
                const int mine = t + ((wave - t) & (kAhead - 1));  // the first unit from t on that is this wave's
                if (mine < t + sets) wait_vmcnt<0>();
                __syncthreads();
                if (mine < t + sets) move(mine + kAhead);
                const int u = t + set;
                if (u >= n) continue;
                const UnitInLds x = unit_in(smem + u % kSlots * kSlotBytes, lane);
                const int left = len - (c0 + u) * kUnit, first_sees = a->causal ? left - a->q_len + 1 : left;
                int sees[NB];
#pragma unroll
                for (int i = 0; i < NB; ++i) sees[i] = a->causal ? min(first_sees + tok[i], left) : left;
                compute<DT, NB>(s, x, a->scale_log2, lane, first_sees < kUnit, sees, left);
            }
            __syncthreads();
 ST(7);
        }

        // ---- the sets' parts, joined -------------------------------------------------------------------------
        {
            const int x = lane_again(lane), n16 = x & 15, g = x >> 4;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const float sum = over_groups(s.l[i], [](float x, float y) { return x + y; });
                const int at = 16 * i + n16;
                CK_LDS char *p = smem + wave * kWidePart + (at * 4 + g) * 16;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    *reinterpret_cast<CK_LDS f32x4 *>(p + j * 32 * 64) =
                        f32x4{s.o[i][4 * (j & 1)][j >> 1], s.o[i][4 * (j & 1) + 1][j >> 1], s.o[i][4 * (j & 1) + 2][j >> 1],
                              s.o[i][4 * (j & 1) + 3][j >> 1]};
                if (g == 0)
                    *reinterpret_cast<CK_LDS f32x2 *>(smem + kWideMl + (wave * 32 + at) * 8) = f32x2{s.m[i] - Form<DT, NB>::kBias, sum};
            }
        }
        __syncthreads(); ST(8);
        a = args_again(args);
        const bool whole = !before && !after && !a->merge;
        const int slot_rows = min(a->tile_rows, a->rows);
        const int64_t slot = part_slot(before, after, share, a->waves, item) * a->tiles + tile;
        // a thread takes dims 32 g + 4 j .. + 3 of a row, j of every second (fourth, ...) eighth
        const int y = 64 * wave + lane_again(lane);
        for (int at = y >> 2; at < a->tile_rows; at += kWideThreads / 4) {
            const int g = y & 3, r = a->tile_rows * tile + at;
            const CK_LDS char *part = smem + (at >> 5) * kWidePart + ((at & 31) * 4 + g) * 16;
            float top = -INFINITY, sum = 0.f;
            for (int w = 0; w < sets; ++w)
                top = fmaxf(top, (*reinterpret_cast<const CK_LDS f32x2 *>(smem + kWideMl + (w * a->tile_rows + at) * 8))[0]);
            f32x4 z[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int w = 0; w < sets; ++w) {
                const f32x2 ml = *reinterpret_cast<const CK_LDS f32x2 *>(smem + kWideMl + (w * a->tile_rows + at) * 8);
                const float by = ml[0] == -INFINITY ? 0.f : exp2_fast(ml[0] - top);
                sum = fmaf(ml[1], by, sum);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const f32x4 v = *reinterpret_cast<const CK_LDS f32x4 *>(part + w * row_waves * kWidePart + j * 32 * 64);
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[j][e] = fmaf(v[e], by, z[j][e]);
                }
            }
            if (r >= a->rows) continue;
            if (whole) {
                const int t = r / a->group;
                const int64_t row = ((int64_t)b * a->q_len + t) * a->heads + h * a->group + (r - t * a->group);
                const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    *reinterpret_cast<uint2 *>(a->out + row * kD + 32 * g + 4 * j) =
                        make_uint2(E::pack2(z[j][0] * inv, z[j][1] * inv), E::pack2(z[j][2] * inv, z[j][3] * inv));
                if (g == 0) a->lse[row] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * kLn2;
            } else {
                float *to = a->part_o + slot * slot_rows * kD + (at * 4 + g) * 4;
#pragma unroll
                for (int j = 0; j < 8; ++j) *reinterpret_cast<f32x4 *>(to + j * slot_rows * 16) = z[j];
                if (g == 0) a->part_ml[slot * slot_rows + at] = make_float2(top, sum);
            }
        }
        __syncthreads(); ST(9);
    }
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
    int64_t rows, blocks, tile_rows, tiles, groups, waves, slot_rows, slots;  // blocks 0: the form for many rows
    int64_t off_sums, off_ml, off_o, end;
};

int plan_side(int64_t batch, int64_t rows, int64_t kv_heads, int64_t kv_cap, bool merge, int64_t at, Side *p) {
    p->rows = rows;
    p->blocks = rows <= 16 ? 1 : rows <= 32 ? 2 : 0;
    // many rows: 32 of 2, 4 or 8 waves, of the two largest that which leaves fewer empty
    p->tile_rows = p->blocks ? 16 * p->blocks : rows <= 64 ? 64 : ceil_div(rows, 128) % 2 ? 128 : 256;
    p->tiles = ceil_div(rows, p->tile_rows);
    if (p->blocks == 0) {  // shares of workgroups
        p->waves = p->tiles < kGroupsWide ? kGroupsWide / p->tiles : 1;
        p->groups = p->waves * p->tiles;
    } else {
        p->groups = kGroups;
        p->waves = p->groups * kWaves;
    }
    if (!grid_fits(p->groups, kThreads)) return CK_E_INVALID_ARG;
    // the list's places are 32-bit, and its shares' numbers
    if (batch * kv_heads >= (int64_t)1 << 31 || batch * kv_heads * ceil_div(kv_cap, kUnit) >= (int64_t)1 << 31)
        return CK_E_INVALID_ARG;
    p->slot_rows = rows < p->tile_rows ? rows : p->tile_rows;
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
    else if (p.blocks == 2) hipLaunchKernelGGL((kv4_decode_kernel<DT, 2>), grid, block, 0, s, a);
    else {
        static std::atomic<uint64_t> lds_set{0};
        const int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(&kv4_wide_kernel<DT>), kWideLds, lds_set);
        if (rc != CK_OK) return rc;
        hipLaunchKernelGGL((kv4_wide_kernel<DT>), grid, dim3(kWideThreads), kWideLds, s, a);
    }
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
    a->tile_rows = (int)p.tile_rows;
    a->waves = (int)p.waves;
    a->part_o = reinterpret_cast<float *>(ws + p.off_o);
    a->part_ml = reinterpret_cast<float2 *>(ws + p.off_ml);
    a->sums = reinterpret_cast<int32_t *>(ws + p.off_sums);
    *f = FoldSide{a->part_o, a->part_ml, a->sums, a->batch, a->waves, a->tiles, a->tile_rows, (int)p.slot_rows};
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

extern "C" int st_read(void *dst) { return (int)hipMemcpyFromSymbol(dst, HIP_SYMBOL(ck::g_st), sizeof(unsigned long long) * 4096 * 16); }
