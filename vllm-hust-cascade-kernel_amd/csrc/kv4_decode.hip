// kv4_decode.hip - decode attention over a paged K/V cache in 4 bits (gfx950), alone or with a prefix that all
// sequences share.
//
// Row (token i, head h) of request b, k_j and v_j the dequantised cache of its kv head:
//   s_j = scale q . k_j, j < len_b - q_len + 1 + i
//   o = sum_j softmax(s)_j v_j,  lse = log sum_j exp(s_j)
// A row that sees no token gets o = 0, lse = -inf.
//
// A token and kv head are 136 bytes and 512 flops a row: memory bounds a call up to some 16 rows a kv head
// (tokens of a request times query heads of the kv head), arithmetic beyond.
// * S^T = K Q^T on 16x16x32 products: lane (g, n) holds group g of a token's key, four code conversions (two
//   values each, the scale in the instruction) make an operand. O^T = V^T P^T: lane (g, n) holds dims 8 n .. + 7 of
//   tokens 8 g .. + 7; two conversions give (token, dim pair) words, two byte permutations turn them to (dim, token
//   pair). P is in its operand's place as it leaves the scores. The pool's order is that of these operands, so that a
//   lane loads 16 bytes at a time and nothing is exchanged.
// * The softmax's reference point m of a row moves only when a score passes the one it was set by by 2^kSlack (any
//   point gives the same result), so that O is hardly ever rescaled.
// * The units (64 tokens, 8704 bytes that lie together) of all requests and kv heads form one list, cut evenly
//   over a grid that fills the chip once, so ragged lengths balance. An item (request and kv head) inside one share is
//   written as it is; parts of a cut one go to the workspace, and kv4_combine_kernel folds them.
// * Up to 32 rows a wave computes alone (kv4_decode_kernel): up to 16 with units in registers, the next one's loads
//   under way while one is computed; up to 32 with a ring of two units in LDS. More rows take kv4_wide_kernel.
// * Shared prefix: the batch is one request's rows over the prefix. Where the suffixes have up to 16 rows each, one
//   launch takes both lists, a wave its share of the prefix and then of the suffixes; one fold for all parts.
//   us a call, one launch / two: 8 x 32 heads on 2000 + 200 tokens 16.5 / 18.7, 64 x 32 on 8000 + 200 35.7 / 41.5,
//   on 500 + 2000 44.6 / 47.9, 256 x 32 on 8000 + 300 73 / 79.
//
// Measured (kernel + fold in us; query / kv heads): 64 requests of 2048 to 8192 tokens, 32 / 8, 72 + 6, 4.9 TB/s; 16 of 16384
// to 65536, 64 / 8, 160 + 7, 5.3 TB/s; 5 of 5000 to 20011, 20 / 20 in fp16, 32 + 5; one of 1300, 32 / 8, 6 + 4, chains of
// round trips (lengths, table, unit, fold) and two launches. 24 requests of 1250 to 5000, 3 tokens, 64 / 8 in fp16 (24
// rows): 29 + 8, 12 of them vector instructions, 25 MB of parts written and read. 17 / 24 / 32 rows in the form for
// 32 against the one for 64, us a call: 24 requests of 1000 tokens, 8 kv heads, 23 / 25 / 26 against 30 / 30 / 32; 64 of 4000
// 70 / 74 / 78 against 90 / 94 / 97; 4 of 500 11 / 11 / 12 against 16 / 17 / 17. One of 16000 would be sooner in the form for 64, whose
// shares end with the kv heads: 25 / 26 / 28 against 20 / 20 / 21.
#include <cmath>
#include <type_traits>

#include "kv4_common.h"
#include "kv4_map.h"
#include "latent_common.h"

namespace ck {
namespace {

using namespace kv4;

typedef __attribute__((__vector_size__(2 * sizeof(float)))) float f32x2;

// 1 / x within a step, for weights that are to sum up to 1; of a sum of nothing 0.
__device__ __forceinline__ float one_over(float x) { return x == 0.f ? 0.f : __builtin_amdgcn_rcpf(x); }

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kGroups = 512;      // workgroups: two per CU, so two waves a SIMD, as many as the registers allow
constexpr int kGroupsWide = 256;  // of many rows: one per CU, which its LDS fills
// Up to how many rows a row's parts are folded by 8, 4 and 2 groups of lanes. us with 8 / 4 / 2 / 1: 32 rows of 21 parts
// 4.2 / 4.8 / 5.4 / 6.4, 256 of 36 4.6 / 5.3 / 6.6 / 9.6, 1024 of 17 7.6 / 6.8 / 7.3 / 9.5, 2048 of 10 10.0 / 7.1 / 7.4 / 9.2
// (of 5: 8.9 / 6.7 / 5.5 / 5.4), 4608 of 11 14.3 / 8.9 / 8.2 / 8.3, 7488 of 6 19.8 / 14.6 / 11.7 / 9.0.
constexpr int kFoldRows[3] = {512, 2048, 6144};
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
    int group;  // query heads per kv head
    int rows;   // q_len * group: of an item
    int tiles;  // row tiles of an item
    int waves;  // at most so many shares of the list (waves', or with many rows workgroups'), per row tile
    int pieces;  // many rows of one request: at most so many shares of a kv head, or 0
    int causal;
    int merge;  // every part goes to the workspace
    float scale_log2;
    uint16_t *out;
    float *lse;
    // Parts, each the mean over its tokens: [slot][tile][8][tile's rows][4 g][4], dims 32 g + 4 j + e
    float *part_o;
    float2 *part_ml;  // [slot][tile][tile's rows]: reference point (log2), sum of p
    int32_t *sums;    // [batch + 1]: units before each request (of one kv head)
    Shares *shares;   // how the list is cut, behind them; both for the fold
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

// starts[t]: units (of one kv head) before thread t's requests, t's share of the batch, len0[t] the first one's
// length. Returns the units in all; the first workgroup leaves those before each request for the fold.
template <int T>
__device__ __forceinline__ int requests_per_thread(KernArgs a) { return (a->batch + T - 1) / T; }
template <int T>
__device__ __forceinline__ int list_starts(KernArgs a, int *starts, int *len0, int *scan, int tid) {
    const int per = requests_per_thread<T>(a), b0 = min(tid * per, a->batch), b1 = min(b0 + per, a->batch);
    int mine = 0;
    for (int b = b0; b < b1; ++b) {
        const int len = len_of(a, b);
        if (b == b0) len0[tid] = len;
        mine += units_of(len);
    }
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
// x: the last thread whose requests begin at or before u.
template <int T>
__device__ __forceinline__ Found find_from(KernArgs a, const int *starts, const int *len0, int u, int x) {
    Found f;
    f.b = min(x * requests_per_thread<T>(a), a->batch - 1);
    f.at = starts[x] * a->kv_heads;
    f.len = len0[x];
    while (f.b + 1 < a->batch && f.at + units_of(f.len) * a->kv_heads <= u) {  // of the thread's
        f.at += units_of(f.len) * a->kv_heads;
        f.len = len_of(a, ++f.b);
    }
    return f;
}
template <int T>
__device__ __forceinline__ Found find_request(KernArgs a, const int *starts, const int *len0, int u) {  // u a lane
    int x = 0;
#pragma unroll
    for (int step = T / 2; step > 0; step >>= 1)
        if (starts[x + step] * a->kv_heads <= u) x += step;
    return find_from<T>(a, starts, len0, u, x);
}
template <int T>
__device__ __forceinline__ Found find_request_of_wave(KernArgs a, const int *starts, const int *len0, int u, int lane) {
    constexpr int kEach = T / 64;
    const int some = __popcll(__builtin_amdgcn_ballot_w64(starts[kEach * lane] * a->kv_heads <= u)) - 1;
    const int more = __popcll(__builtin_amdgcn_ballot_w64(lane < kEach && starts[kEach * some + lane % kEach] * a->kv_heads <= u)) - 1;
    return find_from<T>(a, starts, len0, u, scalar(kEach * some + more));
}
// The list of a call's units for a workgroup of T threads; SINGLE: of one request (a prefix), which needs no table.
template <int T, bool SINGLE>
struct List {
    const int *starts, *len0;
    int total;  // units of one kv head
    int len;    // of the one request
    // All threads come here (a barrier).
    __device__ __forceinline__ List(KernArgs a, int *starts_at, int *len0_at, int *scan, int tid) : starts(starts_at), len0(len0_at) {
        if constexpr (SINGLE) {
            len = scalar(len_of(a, 0));
            total = units_of(len);
            if (blockIdx.x == 0 && tid < 2) a->sums[tid] = tid * total;
        } else {
            len = 0;
            total = scalar(list_starts<T>(a, starts_at, len0_at, scan, tid));
        }
    }
    __device__ __forceinline__ List(const int *starts_at, const int *len0_at, int units) : starts(starts_at), len0(len0_at), total(units), len(0) {}
    __device__ __forceinline__ Found find(KernArgs a, int u) const {  // u a lane
        if constexpr (SINGLE) return Found{0, 0, len};
        else return find_request<T>(a, starts, len0, u);
    }
    __device__ __forceinline__ Found find_of_wave(KernArgs a, int u, int lane) const {
        if constexpr (SINGLE) return Found{0, 0, len};
        else return find_request_of_wave<T>(a, starts, len0, u, lane);
    }
};
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
// Where a lane's keys lie in a unit in LDS, those of tile t at + 2048 (t / 2) + 256 (t % 2).
__device__ __forceinline__ int keys_in_lds(int lane) {
    const int n = lane & 15;
    return (8 * (n >> 2) + (n & 3)) * 64 + 16 * ((lane >> 4) ^ (n >> 2));
}
// A unit in LDS: what is needed is read where it is.
struct UnitInLds {
    const CK_LDS char *k_at, *at;  // the lane's
    u32x4 vs;
    uint32_t ks;
    __device__ __forceinline__ u32x4 keys(int t) const {
        return *reinterpret_cast<const CK_LDS u32x4 *>(k_at + 2048 * (t >> 1) + 256 * (t & 1));
    }
    __device__ __forceinline__ u32x4 values(int q) const { return *reinterpret_cast<const CK_LDS u32x4 *>(at + kVAt + 1024 * q); }
};
// The same in the compiler's eyes new: what one of two ways through computes from it is not made before them, for
// both.
__device__ __forceinline__ u32x4 again(u32x4 x) {
    asm volatile("" : "+v"(x));
    return x;
}
// A unit's way to LDS: 10 moves without a register between, 16 bytes a lane of the codes and 4 of the scales. All lie as
// in memory, but a token's four groups of key codes are exchanged by (token / 8) % 4: the 16 lanes that read one
// group of 16 tokens, 4 tokens in a row of 8, then touch every bank once.
constexpr int kPieces = 10;
template <int IMM>
__device__ __forceinline__ void dma_words(const ck_rsrc_t &r, int voff, int soff, int base) {
    asm volatile("s_add_i32 m0, %0, %c1\n\ts_nop 0\n\tbuffer_load_dword %2, %3, %4 offen lds"
                 :
                 : "s"(base), "i"(IMM), "v"(voff), "s"(r), "s"(soff)
                 : "memory", "m0", "scc");
}
// The unit at `at` (unit_address) to a slot of kUnitBytes; from a page outside the pool, zeros (a range of nothing).
__device__ __forceinline__ void move_unit(uint64_t at, const CK_LDS char *slot, int lane) {
    const ck_rsrc_t r = {(int)(uint32_t)(at & ~1ull), (int)((uint32_t)(at >> 32) & 0xffffu), at & 1 ? 0 : kUnitBytes,
                         (int)kRsrcFlags};
    const int base = scalar((int)(uint32_t)(uintptr_t)slot);
    const int keys = (lane >> 2) * 64 + 16 * ((lane & 3) ^ (lane >> 5));  // tokens 16 P + lane / 4
    static_for<8>([&](auto p) __attribute__((always_inline)) {
        constexpr int P = p;
        lat::dma_tile<1024 * P>(r, P >= 4 ? 16 * lane : P % 2 ? keys ^ 32 : keys, 1024 * P, base);
    });
    dma_words<kKsAt>(r, 4 * lane, kKsAt, base);
    dma_words<kVsAt>(r, 4 * lane, kVsAt, base);
}
__device__ __forceinline__ UnitInLds unit_in(const CK_LDS char *slot, int lane) {
    UnitInLds u;
    u.k_at = slot + keys_in_lds(lane);
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
// point 2^7 p stays below 65504), half a step off: 2^-11 of p, and 2^-32 of the row's largest weight (2^7 p is 2^7 there at the
// least, fp16's smallest steps are 2^-24) however small p is. An fp16 query's keys are fp16 numbers too, exactly. Units of
// other scales are computed as above. 24 x 3 x 64 heads over 5000 tokens (fp16): 36.7 -> 27.9 us, the units in LDS instead of
// registers among it.
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
    float m[NB];     // the sum's reference point (log2; the same for all g), kBias below a score
    float l[NB];     // this lane's share of the sum
    uint32_t bad;    // bit i: row i sees a value that is not a number in this lane's dims
    uint32_t far;    // bit d: O's dims 32 d .. + 31 are lowered (the same in all lanes)
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
    s.bad = 0;
    s.far = 0;
}
// Gives O what hide_values() has put off.
template <int NB>
__device__ __forceinline__ void add_bad(f32x4 (&o)[NB][8], uint32_t bad) {
    if (__builtin_expect(!__builtin_amdgcn_ballot_w64(bad != 0), 1)) return;
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[i][k][r] = (bad >> i) & 1 ? NAN : o[i][k][r];
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
        const float sub = s.m[i] == -INFINITY ? 0.f : s.m[i];
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

// Values up to the largest that are written, 6 * 2^125 = 1.5 * 2^127: their mean is finite, a sum of them need not be. Below a
// scale of 2^65 (byte kFar) the sum p v of 2^30 tokens, p at most 2^(kSlack + 7) = 2^15, stays below 6 * 2^64 * 2^45 < 2^112.
// A wave that meets a larger scale in an item holds O of that group of 32 dims times 2^-48 from then on, and lowers
// the group's scales: 1.5 * 2^(127 - 48 + 45) = 1.5 * 2^124 at most. Scale bytes below 48 become 0, which is 2^-127: values of
// less than 6 * 2^-80 are off by less than 6 * 2^-79, 2^-76. Parts are joined as means, with weights that sum up to 1, by which no
// sum passes the values.
constexpr int kFar = 192, kLowered = 48;
constexpr float kLower = 0x1p-48f, kRaise = 0x1p48f;
// Nonzero where a scale byte of w is kFar and more.
__device__ __forceinline__ uint32_t far_bytes(uint32_t w) { return w & (w << 1) & 0x80808080; }
// The groups of dims in which some lane's tokens have such a scale, the lanes n / 4 each; any: some of this lane's.
__device__ __forceinline__ uint32_t far_groups(bool any) {
    const uint64_t b = __builtin_amdgcn_ballot_w64(any);
    uint32_t x = (uint32_t)(b >> 32) | (uint32_t)b;
    x |= x >> 16;  // lanes n
    return ((x & 0xf) != 0 ? 1 : 0) | ((x & 0xf0) != 0 ? 2 : 0) | ((x & 0xf00) != 0 ? 4 : 0) | ((x & 0xf000) != 0 ? 8 : 0);
}
// The scales of four tokens in a lowered group (255 stays what it is); a lane (g, n) has those of group n / 4.
__device__ __forceinline__ uint32_t lowered(uint32_t w) {
    uint32_t to = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const uint32_t e = (w >> (8 * b)) & 0xff;
        to |= (e == kBad ? kBad : max(e, (uint32_t)kLowered) - kLowered) << (8 * b);
    }
    return to;
}
__device__ __forceinline__ bool has_lowered(uint32_t far, int lane) { return (far >> ((lane & 15) >> 2)) & 1; }
// What a lane's O of group g is to be multiplied by.
__device__ __forceinline__ float by_group(uint32_t groups, int lane, float by) { return (groups >> (lane >> 4)) & 1 ? by : 1.f; }

// Moves the reference points of rows whose scores pass them by 2^(kSlack + kBias) (most: the lane's largest) to 2^kBias
// below the largest; no score of these passes them by as much again. lower: what else O is multiplied by.
template <int NB>
__device__ __forceinline__ void move_points(f32x4 (&o)[NB][8], float (&m)[NB], float (&l)[NB], const float (&most)[NB], float lower) {
    constexpr float kBias = Form<CK_DTYPE_BF16, NB>::kBias;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const float all = over_groups(most[i], [](float x, float y) { return fmaxf(x, y); });
        const float to = all > m[i] + (kSlack + kBias) ? all - kBias : m[i];
        const float by = to == m[i] ? 1.f : exp2_fast(m[i] - to), o_by = by * lower;
        l[i] *= by;
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[i][k][r] *= o_by;
        m[i] = to;
    }
}

// The first n bytes of w, the others `rest`.
__device__ __forceinline__ uint32_t first_bytes(uint32_t w, int n, uint32_t rest) {
    const uint32_t mask = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
    return (w & mask) | (rest & ~mask);
}

// The values' scales of a half unit that not every row sees whole (sees and left counted from its first token; x, y those
// of tokens 8 g .. + 7). Those of tokens from `left` on go, and values that are not numbers would reach rows that
// do not see them (0 times them is none): their scales become ordinary ones, and rows that do see one are marked.
// A lane (g, n) has the dims of group g of its rows' O. A row may see more tokens than the unit has (kUnit stands
// for no such token).
template <int NB>
__device__ __forceinline__ void hide_values(uint32_t &bad, uint32_t &x, uint32_t &y, const int (&sees)[NB], int left, int g) {
    int first_bad = kUnit;
#pragma unroll
    for (int w = 1; w >= 0; --w) {
        uint32_t &s = w ? y : x;
        const int t0 = 8 * g + 4 * w;
        s = first_bytes(s, left - t0, kMidScales);
#pragma unroll
        for (int b = 3; b >= 0; --b) {
            if (((s >> (8 * b)) & 0xff) != kBad) continue;
            first_bad = t0 + b;
            s ^= (kBad ^ (kMidScales & 0xff)) << (8 * b);
        }
    }
    if (__builtin_expect(!__builtin_amdgcn_ballot_w64(first_bad < kUnit), 1)) return;
    first_bad = (int)over_groups((float)first_bad, [](float x, float y) { return fminf(x, y); });
    first_bad = __shfl(first_bad, 4 * g);
#pragma unroll
    for (int i = 0; i < NB; ++i) bad |= first_bad < min(sees[i], kUnit) ? 1u << i : 0;
}

// One unit. Where tail: tokens from sees[i] on are hidden from row block i's row, those from `left` on
// (counted from the unit's first) hold anything.
template <int DT, int NB, class U>
__device__ __forceinline__ void compute(Rows<DT, NB> &s, const U &u, float scale_log2, int lane, bool tail,
                                        const int (&sees)[NB], int left) {
    constexpr float kBias = Form<DT, NB>::kBias;
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
        int sees2[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) sees2[i] = sees[i] - 32;
        uint32_t x[4] = {vs[0], vs[1], vs[2], vs[3]};
        hide_values<NB>(s.bad, x[0], x[1], sees, left, g);
        hide_values<NB>(s.bad, x[2], x[3], sees2, left - 32, g);
        vs = u32x4{x[0], x[1], x[2], x[3]};
    }
    const bool half = kHalf && s.far == 0 &&
                      __builtin_expect(!__builtin_amdgcn_ballot_w64((past_half(vs[0]) | past_half(vs[1]) | past_half(vs[2]) | past_half(vs[3])) != 0), 1);
    uint32_t more = 0;  // groups of dims to be lowered
    if (!half) {
        const bool any = (far_bytes(vs[0]) | far_bytes(vs[1]) | far_bytes(vs[2]) | far_bytes(vs[3])) != 0;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(any) != 0, 0)) more = far_groups(any) & ~s.far;
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        float most = max3(sc[i][0][0], sc[i][0][1], sc[i][0][2]);
#pragma unroll
        for (int e = 3; e < 15; e += 2) most = max3(most, sc[i][e >> 2][e & 3], sc[i][(e + 1) >> 2][(e + 1) & 3]);
        most = fmaxf(most, sc[i][3][3]) * scale_log2;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(most > s.m[i] + (kSlack + kBias)) != 0 || more != 0, 0)) {
            const float all = over_groups(most, [](float x, float y) { return fmaxf(x, y); });
            const float m = all > s.m[i] + (kSlack + kBias) ? all - kBias : s.m[i];
            float f = m == s.m[i] ? 1.f : exp2_fast(s.m[i] - m);
            s.l[i] *= f;
            f *= by_group(more, lane_again(lane), kLower);
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r) s.o[i][k][r] *= f;
            s.m[i] = m;
        }
    }
    s.far |= more;
    if (__builtin_expect(half, 1)) {
        add_values<true, 0, NB>(s, v, vs, sc, scale_log2);
    } else {
        u32x4 x = again(vs);
        if (__builtin_expect(s.far != 0, 0) && has_lowered(s.far, lane_again(lane))) {
#pragma unroll
            for (int w = 0; w < 4; ++w) x[w] = lowered(x[w]);
        }
        add_values<false, 0, NB>(s, v, x, sc, scale_log2);
    }
}

// What a wave makes of its share w of the list; more than one row block: through its ring of two units in LDS.
template <int DT, int NB, class L>
__device__ __forceinline__ void decode_share(const KernArgs args, const L &list, CK_LDS char *ring, int w, int lane) {
    KernArgs a = args_again(args);
    constexpr int kRows = 16 * NB;
    constexpr bool kQAhead = NB == 1;  // the next item's queries are loaded ahead
    const int total = list.total;
    const Shares cut = list_shares(total * a->kv_heads, a->waves, 1, 0, 0);
    if (w >= cut.count) return;
    if (w == 0 && lane == 0) *a->shares = cut;
    const int lo = scalar(share_lo(cut, w)), hi = scalar(share_lo(cut, w + 1));
    const int slot_rows = min(kRows, a->rows);

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
        add_bad<NB>(s.o, s.bad);
        const bool whole = !before && !after && !a->merge;
        const int64_t slot = part_slot(before, after, w, a->waves, item);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int r = 16 * i + n16;
            const float l = over_groups(s.l[i], [](float x, float y) { return x + y; }), m = s.m[i];
            const float inv = (l == 0.f ? 0.f : 1.0f / l) * by_group(s.far, x, kRaise);
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) s.o[i][k][e] *= inv;
            if (r >= a->rows) continue;
            if (whole) {
                using E = Elem<DT>;
                const int64_t row = ((int64_t)b * a->q_len + tok[i]) * a->heads + h * a->group + (r - tok[i] * a->group);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    u32x4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = E::pack2(s.o[i][2 * e][d], s.o[i][2 * e + 1][d]);
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
            const Found f = list.find(a, u);
            const int each = units_of(f.len), h = (u - f.at) / each, i = u - f.at - h * each;
            d_item = f.b * a->kv_heads + h;
            d_first = i * kUnit;
            d_len = f.len;
            d_at = unit_address(a, f.b, h, i);
        }
        // One row block: the next unit in registers; more: in the wave's other half of its ring.
        Unit next;
        auto fetch = [&](int j) {
            const uint64_t at = of_lane(d_at, j);
            if constexpr (NB > 1) move_unit(at, ring + (j & 1) * kUnitBytes, lane_again(lane));
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
                compute<DT, NB>(s, unit_in(ring + (j & 1) * kUnitBytes, lane), a->scale_log2, lane, first_sees < kUnit, sees, left);
            } else {
                compute<DT, NB>(s, in_registers, a->scale_log2, lane, first_sees < kUnit, sees, left);
            }
        }
    }
    close_item(item, before, goes_on);
}

// The arguments of a call's lists lie one behind the other: the suffixes', or a prefix's (a request of NB row
// blocks) and then the suffixes' (of one), whose shares a wave takes one after the other.
struct PairArgs {
    DecodeArgs prefix, own;
};
template <int DT, int NB, bool PAIR>
__global__ __launch_bounds__(kThreads, 2) void kv4_decode_kernel(std::conditional_t<PAIR, PairArgs, DecodeArgs>) {
    const KernArgs args = (KernArgs)__builtin_amdgcn_kernarg_segment_ptr();
    __shared__ int starts[kThreads], len0[kThreads], scan[kWaves];
    __shared__ __attribute__((aligned(16))) char ring[NB > 1 ? kWaves * 2 * kUnitBytes : 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6);
    // neighbouring shares on different CUs, so that few units spread over all of them
    const int w = scalar(wave * (int)gridDim.x + (int)blockIdx.x);
    CK_LDS char *mine = (CK_LDS char *)ring + (NB > 1 ? wave * 2 * kUnitBytes : 0);
    const List<kThreads, PAIR> list(args, starts, len0, scan, tid);
    if constexpr (PAIR) {
        const List<kThreads, false> own(args + 1, starts, len0, scan, tid);
        decode_share<DT, NB>(args, list, mine, w, lane);
        decode_share<DT, 1>(args + 1, own, mine, w, lane);
    } else {
        decode_share<DT, NB>(args, list, mine, w, lane);
    }
}

// ---- many rows ---------------------------------------------------------------------------------------------
// The same for items of more than 32 rows, on workgroups of 8 waves with a CU to themselves, two per SIMD, which fill
// each other's waits. A workgroup takes a row tile of 64 rows, whose query is in LDS (O alone takes half of a wave's
// registers); its waves take an item's units in turn, each through a double buffer of its own in LDS, so that
// nothing holds them together: with a ring that all read, and a barrier for every 4 units, 117 x 64 heads on 16001 tokens
// took 108 to 118 us. Their parts are joined through LDS, so that few go to memory. A wave works in halves of 32 tokens,
// 64 products and 273 vector instructions each (codes 64 and their permutations 32, exponentials 32, their arguments,
// sums and conversions 84); these bound it, at 950 TFLOP/s over a long prefix, and the start and the joint where a
// workgroup has few units. Where a half's last tokens are hidden, only scores and scales are changed in the loop; a half
// that holds nothing is passed over (the one and the other cost 16001 tokens 3 us of 106 outside it).
// The shares of the list are workgroups', neighbours on one XCD, so that the row tiles of a share meet in its L2.
// us a call with the fold: 117 x 64 heads on 16001 tokens and suffixes (fp16) 100, 64 x 32 on 8192 39.
constexpr int kWideThreads = 512, kWideWaves = kWideThreads / 64;
constexpr int kWideQ = kWideWaves * 2 * kUnitBytes;  // [NB][4] operands of 1 KB, behind the waves' buffers
constexpr int kWideStarts = kWideQ + 4 * 4 * 1024;
constexpr int kWideLds = kWideStarts + (2 * kWideThreads + kWideWaves) * 4;
constexpr int kWidePart = (4 * 8 + 2) * 1024;  // a wave's O, m and l as its lanes hold them, in the buffers' and the query's place
static_assert(kWideWaves / 2 * kWidePart <= kWideStarts && kWideLds <= 160 * 1024, "LDS");

// A half unit (tokens 32 h .. + 31) as a wave's lanes hold it.
struct Half {
    u32x4 k[2];
    uint32_t ks, v[4][2], vs[2];
};
typedef __attribute__((__vector_size__(2 * sizeof(unsigned)))) unsigned u32x2;
__device__ __forceinline__ void read_keys(Half &x, const CK_LDS char *slot, int h, int lane) {
    const CK_LDS char *k_at = slot + keys_in_lds(lane) + 2048 * h;
    x.k[0] = *reinterpret_cast<const CK_LDS u32x4 *>(k_at);
    x.k[1] = *reinterpret_cast<const CK_LDS u32x4 *>(k_at + 256);
    x.ks = *reinterpret_cast<const CK_LDS uint16_t *>(slot + kKsAt + 4 * lane + 2 * h);
    const u32x2 s = *reinterpret_cast<const CK_LDS u32x2 *>(slot + kVsAt + ((lane & 15) >> 2) * 64 + 16 * (lane >> 4) + 8 * h);
    x.vs[0] = s[0], x.vs[1] = s[1];
}
__device__ __forceinline__ void read_values(Half &x, const CK_LDS char *slot, int h, int lane) {
    const CK_LDS char *at = slot + 16 * lane;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const u32x2 y = *reinterpret_cast<const CK_LDS u32x2 *>(at + kVAt + 1024 * d + 8 * h);
        x.v[d][0] = y[0], x.v[d][1] = y[1];
    }
}

// The order of a part of a loop: N times a product and V vector instructions, which run beside it.
template <int N, int V>
__device__ __forceinline__ void mix() {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, V, 0);
    }
}

// Scores of a half; q: the lane's place in the query's operands.
template <bool HALF, int DT, int NB>
__device__ __forceinline__ void half_scores(f32x4 (&sc)[NB][2], const Half &x, const CK_LDS char *q) {
#pragma unroll
    for (int i = 0; i < NB; ++i) sc[i][0] = sc[i][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    // the query's operands of the next dims come while these are multiplied; as two terms there are no registers for it
    constexpr int kAhead = DT != CK_DTYPE_F16 || HALF ? 1 : 0;
    u32x4 y[1 + kAhead][NB];
    auto read_q = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NB; ++i) y[c & kAhead][i] = *reinterpret_cast<const CK_LDS u32x4 *>(q + (4 * i + c) * 1024);
    };
    if (kAhead) read_q(0);
    const float f[2] = {scale_of<0>(x.ks), scale_of<1>(x.ks)};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (c + kAhead < 4) read_q(c + kAhead);
        __builtin_amdgcn_sched_barrier(0);
        u32x4 a[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const uint32_t w = x.k[t][c];
            if constexpr (HALF) a[t] = u32x4{pair_f16<0>(w, f[t]), pair_f16<1>(w, f[t]), pair_f16<2>(w, f[t]), pair_f16<3>(w, f[t])};
            else a[t] = u32x4{pair_bf16<0>(w, f[t]), pair_bf16<1>(w, f[t]), pair_bf16<2>(w, f[t]), pair_bf16<3>(w, f[t])};
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const u32x4 &z = y[c & kAhead][i];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                if constexpr (HALF) {
                    sc[i][t] = mfma_f16(a[t], z, sc[i][t]);
                } else if constexpr (DT == CK_DTYPE_F16) {
                    u32x4 hi, lo;
                    two_terms(z, hi, lo);
                    sc[i][t] = mfma_bf16(a[t], hi, sc[i][t]);
                    sc[i][t] = mfma_bf16(a[t], lo, sc[i][t]);
                } else {
                    sc[i][t] = mfma_bf16(a[t], z, sc[i][t]);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}
// The largest score of a row block's lane.
__device__ __forceinline__ float largest(const f32x4 (&s)[2]) {
    float x = max3(s[0][0], s[0][1], s[0][2]);
    x = max3(x, s[0][3], s[1][0]);
    x = max3(x, s[1][1], s[1][2]);
    return max3(x, s[1][3], s[1][3]);  // fmaxf would first make its operands canonical
}

// P of row blocks I0 .. I0 + N - 1 over a half, its sums, and O^T += V^T P^T.
template <bool HALF, int I0, int N, int NB>
__device__ __forceinline__ void half_values(f32x4 (&o)[NB][8], float (&l)[NB], const float (&m)[NB], const Half &x,
                                            const f32x4 (&sc)[NB][2], float scale_log2) {
    constexpr int kParts = HALF ? 1 : 2;
    u32x4 p[N][kParts];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int i = I0 + k;
        const float sub = !HALF && m[i] == -INFINITY ? 0.f : m[i];  // HALF: no such row
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = exp2_fast(fmaf(sc[i][e >> 1][2 * (e & 1)], scale_log2, -sub));
            const float b = exp2_fast(fmaf(sc[i][e >> 1][2 * (e & 1) + 1], scale_log2, -sub));
            sum[0] += a;
            sum[1] += b;
            if constexpr (HALF) {
                p[k][0][e] = Elem<CK_DTYPE_F16>::pack2(a, b);
            } else {
                p[k][0][e] = pack_bf16x2(a, b);
                p[k][kParts - 1][e] = pack_bf16x2(a - bf16_lo(p[k][0][e]), b - bf16_hi(p[k][0][e]));
            }
        }
        l[i] += sum[0] + sum[1];
        __builtin_amdgcn_sched_barrier(0);
    }
    float f[8];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        f[4 * w] = scale_of<0>(x.vs[w]);
        f[4 * w + 1] = scale_of<1>(x.vs[w]);
        f[4 * w + 2] = scale_of<2>(x.vs[w]);
        f[4 * w + 3] = scale_of<3>(x.vs[w]);
    }
    constexpr int kAhead = HALF ? 1 : 0;  // the next dims' operands are made beside the products
    u32x4 even[1 + kAhead], odd[1 + kAhead];
    auto operands = [&](int d) __attribute__((always_inline)) {
        u32x4 &a = even[d & kAhead], &b = odd[d & kAhead];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const uint32_t c = x.v[d][w];
            uint32_t t[4];
            if constexpr (HALF) {
                t[0] = pair_f16<0>(c, f[4 * w]), t[1] = pair_f16<1>(c, f[4 * w + 1]);
                t[2] = pair_f16<2>(c, f[4 * w + 2]), t[3] = pair_f16<3>(c, f[4 * w + 3]);
            } else {
                t[0] = pair_bf16<0>(c, f[4 * w]), t[1] = pair_bf16<1>(c, f[4 * w + 1]);
                t[2] = pair_bf16<2>(c, f[4 * w + 2]), t[3] = pair_bf16<3>(c, f[4 * w + 3]);
            }
            a[2 * w] = __builtin_amdgcn_perm(t[1], t[0], 0x05040100);
            b[2 * w] = __builtin_amdgcn_perm(t[1], t[0], 0x07060302);
            a[2 * w + 1] = __builtin_amdgcn_perm(t[3], t[2], 0x05040100);
            b[2 * w + 1] = __builtin_amdgcn_perm(t[3], t[2], 0x07060302);
        }
    };
    if (kAhead) {
        operands(0);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        if (kAhead == 0) operands(d);
        else if (d < 3) operands(d + 1);
#pragma unroll
        for (int e = 0; e < kParts; ++e)
#pragma unroll
            for (int k = 0; k < N; ++k) {
                f32x4 &lo = o[I0 + k][2 * d], &hi = o[I0 + k][2 * d + 1];
                lo = HALF ? mfma_f16(even[d & kAhead], p[k][e], lo) : mfma_bf16(even[d & kAhead], p[k][e], lo);
                hi = HALF ? mfma_f16(odd[d & kAhead], p[k][e], hi) : mfma_bf16(odd[d & kAhead], p[k][e], hi);
            }
        if constexpr (kAhead) mix<2 * N, 2>();
        __builtin_amdgcn_sched_barrier(0);
    }
}

// How many of a half's tokens a lane's row of block i sees.
__device__ __forceinline__ int sees_of(int i, int n16, int left, int first_sees, int row0, int group) {
    return first_sees < left ? min(first_sees + (row0 + 16 * i + n16) / group, left) : left;
}
// Scores of tokens that a row does not see: -inf.
template <int NB>
__device__ __forceinline__ void hide_scores(f32x4 (&sc)[NB][2], int lane, int left, int first_sees, int row0, int group) {
    const int y = lane_again(lane);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int n = sees_of(i, y & 15, left, first_sees, row0, group) - 8 * (y >> 4);  // token of sc[i][t][r]: 8 g + 4 t + r
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e >= n) sc[i][e >> 2][e & 3] = -INFINITY;
    }
}
// Ordinary scales in the place of those behind `left`, which may be any.
template <int DT>
__device__ __forceinline__ void end_half(Half &x, int left, int lane) {
    const int y = lane_again(lane), n16 = y & 15, t = 8 * (n16 >> 2) + (n16 & 3);
#pragma unroll
    for (int w = 0; w < 2; ++w) x.vs[w] = first_bytes(x.vs[w], left - 8 * (y >> 4) - 4 * w, kMidScales);
    if constexpr (DT == CK_DTYPE_F16) {
        if (t >= left) x.ks = (x.ks & 0xff00) | (kMidScales & 0xff);
        if (t + 4 >= left) x.ks = (x.ks & 0xff) | (kMidScales & 0xff00);
    }
}

// Any half: of any scales, with scores past a reference point, with rows that have seen nothing yet. row0, group: of the
// wave's rows, where several tokens of a request are causal among themselves (first_sees < left). An fp16 query's keys are
// made as in the usual half where their scales allow it: of random scores 117 x 64 heads on 16001 tokens then take 103 us
// instead of 115, as each wave moves its points a few times.
template <int DT, int NB>
__device__ __forceinline__ void any_half(f32x4 (&o)[NB][8], float (&m)[NB], float (&l)[NB], uint32_t &bad, uint32_t &far,
                                         const CK_LDS char *q, const CK_LDS char *slot, int h, float scale_log2, int lane, int left, int first_sees,
                                         int row0, int group) {
    Half x;
    read_keys(x, slot, h, lane);
    read_values(x, slot, h, lane);
    f32x4 sc[NB][2];
    if (DT == CK_DTYPE_F16 && __builtin_amdgcn_ballot_w64(past_half(x.ks | (kMidScales & 0xffff0000)) != 0) == 0)
        half_scores<true, DT, NB>(sc, x, q);
    else
        half_scores<false, DT, NB>(sc, x, q);
    if (first_sees < 32) {
        hide_scores<NB>(sc, lane, left, first_sees, row0, group);
        const int y = lane_again(lane);
        int sees[NB];
#pragma unroll
        for (int i = 0; i < NB; ++i) sees[i] = sees_of(i, y & 15, left, first_sees, row0, group);
        hide_values<NB>(bad, x.vs[0], x.vs[1], sees, left, y >> 4);
    }
    float most[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) most[i] = largest(sc[i]) * scale_log2;
    const uint32_t more = far_groups((far_bytes(x.vs[0]) | far_bytes(x.vs[1])) != 0) & ~far;
    far |= more;
    move_points<NB>(o, m, l, most, by_group(more, lane_again(lane), kLower));
    if (has_lowered(far, lane_again(lane))) x.vs[0] = lowered(x.vs[0]), x.vs[1] = lowered(x.vs[1]);
    static_for<NB>([&](auto i) __attribute__((always_inline)) {
        // a row block at a time, and nothing kept from one for the next: there are no registers for more
        asm volatile("" : "+v"(x.vs[0]), "+v"(x.vs[1]));
#pragma unroll
        for (int d = 0; d < 4; ++d) asm volatile("" : "+v"(x.v[d][0]), "+v"(x.v[d][1]));
        half_values<false, int(i), 1, NB>(o, l, m, x, sc, scale_log2);
    });
}

template <int DT, bool PAIR>
__global__ __launch_bounds__(kWideThreads, 2) void kv4_wide_kernel(std::conditional_t<PAIR, PairArgs, DecodeArgs>) {
    using E = Elem<DT>;
    constexpr int NB = 4, kTileRows = 16 * NB, kParts = kWideWaves / 2;
    constexpr float kBias = Form<DT, NB>::kBias;
    const KernArgs args = (KernArgs)__builtin_amdgcn_kernarg_segment_ptr();
    KernArgs a = args_again(args);
    extern __shared__ __attribute__((aligned(16))) char wide_raw[];
    CK_LDS char *smem = (CK_LDS char *)wide_raw;
    int *starts = reinterpret_cast<int *>(wide_raw + kWideStarts), *len0 = starts + kWideThreads, *scan = len0 + kWideThreads;
    const int tid = threadIdx.x, lane = tid & 63, wave = scalar(tid >> 6);
    const List<kWideThreads, PAIR> list(a, starts, len0, scan, tid);
    int own_total = 0;
    if constexpr (PAIR) own_total = List<kWideThreads, false>(args + 1, starts, len0, scan, tid).total;
    const int block = scalar((int)xcd_remap(blockIdx.x, gridDim.x));
    const int share = scalar(block / a->tiles), tile = block - share * a->tiles;
    const Shares cut = list_shares(list.total * a->kv_heads, a->waves, list_least(a->batch), list.total, a->pieces);
    if (block == 0 && tid == 0) *a->shares = cut;
    int cur = share < cut.count ? scalar(share_lo(cut, share)) : 0;
    const int hi = share < cut.count ? scalar(share_lo(cut, share + 1)) : 0;
    const int row0 = kTileRows * tile;
    CK_LDS char *buffer = smem + wave * 2 * kUnitBytes;

    f32x4 o[NB][8];
    float m[NB], l[NB];
    uint32_t bad, far;
    while (cur < hi) {
        a = args_again(args);
        const Found f = list.find_of_wave(a, cur, lane);
        const int b = scalar(f.b), len = scalar(f.len), each = units_of(len), in = cur - scalar(f.at);
        const int h = scalar(in / each), i0 = in - h * each, i1 = min(each, i0 + hi - cur);
        const int item = b * a->kv_heads + h;
        const bool before = i0 > 0, after = i1 < each, causal = a->causal;
        const int q_len = a->q_len, group = a->group;
        const float scale_log2 = a->scale_log2;
        int fewer = causal ? q_len - 1 : 0;  // keys that the request's first row does not see
        asm volatile("" : "+s"(fewer));      // nor loaded again for every half
        cur += i1 - i0;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
#pragma unroll
            for (int k = 0; k < 8; ++k) o[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
            m[i] = -INFINITY;
            l[i] = 0.f;
        }
        bad = far = 0;
        bool fresh = true;  // nothing has been added to O
        // The first unit, and the query's operands, some of each wave. Units of this wave: c0 + 8 k, lane k has the
        // address.
        const int w0 = i0 + wave;
        uint64_t d_at = 0;
        if (w0 < i1) d_at = unit_address(a, b, h, min(w0 + kWideWaves * lane, i1 - 1));
        {
            const int x = lane_again(lane), n16 = x & 15, g = x >> 4;
            u32x4 y[NB * 4 / kWideWaves];
#pragma unroll
            for (int e = 0; e < NB * 4 / kWideWaves; ++e) {
                const int piece = e * kWideWaves + wave, c = piece & 3;  // (i, c)
                const int r = kTileRows * tile + 16 * (piece >> 2) + n16, t = r / a->group;
                y[e] = u32x4{0, 0, 0, 0};
                if (r < a->rows)
                    y[e] = *reinterpret_cast<const u32x4 *>(
                        a->q + (((int64_t)b * q_len + t) * a->heads + h * a->group + (r - t * a->group)) * kD + 32 * g + 8 * c);
            }
            if (w0 < i1) move_unit(of_lane(d_at, 0), buffer, lane_again(lane));
#pragma unroll
            for (int e = 0; e < NB * 4 / kWideWaves; ++e)
                *reinterpret_cast<CK_LDS u32x4 *>(smem + kWideQ + (e * kWideWaves + wave) * 1024 + 16 * x) = y[e];
        }
        const CK_LDS char *q = smem + kWideQ + 16 * lane;
        __syncthreads();
        for (int c0 = w0; c0 < i1; c0 += 64 * kWideWaves) {
            const int n = min(64, (i1 - c0 + kWideWaves - 1) / kWideWaves);
            auto slot_of = [&](int k) { return buffer + (k & 1) * kUnitBytes; };
            if (c0 != w0) {
                d_at = unit_address(a, b, h, min(c0 + kWideWaves * lane, i1 - 1));
                move_unit(of_lane(d_at, 0), slot_of(0), lane_again(lane));
            }
            int k = 0, half = 0;
            // The first loop takes halves of fp16's scales with no score past a reference point; nothing else changes O in
            // it, or the compiler would hold O twice and copy it.
            for (;;) {
                int left, first_sees;
                const CK_LDS char *slot;
#pragma unroll 1
                for (;;) {
                    if (half == 0) {
                        if (k + 1 < n) {
                            move_unit(of_lane(d_at, k + 1), slot_of(k + 1), lane_again(lane));
                            wait_vmcnt<kPieces>();
                        } else {
                            wait_vmcnt<0>();
                        }
                        asm volatile("" ::: "memory");
                    }
                    slot = slot_of(k);
                    left = len - (c0 + kWideWaves * k) * kUnit - 32 * half;
                    first_sees = left - fewer;
                    const bool tail = first_sees < 32;
                    Half x;
                    read_keys(x, slot, half, lane);
                    if (__builtin_expect(tail, 0)) end_half<DT>(x, left, lane);
                    uint32_t past = past_half(x.vs[0]) | past_half(x.vs[1]) | far;
                    if constexpr (DT == CK_DTYPE_F16) past |= past_half(x.ks | (kMidScales & 0xffff0000));
                    f32x4 sc[NB][2];
                    half_scores<DT == CK_DTYPE_F16, DT, NB>(sc, x, q);
                    read_values(x, slot, half, lane);
                    __builtin_amdgcn_sched_barrier(0);
                    if (__builtin_expect(__builtin_amdgcn_ballot_w64(past != 0) != 0, 0)) break;
                    if (__builtin_expect(tail, 0)) hide_scores<NB>(sc, lane, left, first_sees, row0, group);
                    bool moves = false;
#pragma unroll
                    for (int i = 0; i < NB; ++i) moves |= !(fmaf(largest(sc[i]), scale_log2, -m[i]) <= kSlack + kBias);  // NaN too
                    if (__builtin_expect(__builtin_amdgcn_ballot_w64(moves) != 0, 0)) {
                        if (!fresh) break;
                        bool none = false;
#pragma unroll
                        for (int i = 0; i < NB; ++i) {  // nothing to scale yet
                            m[i] = over_groups(largest(sc[i]), [](float x, float y) { return fmaxf(x, y); }) * scale_log2 - kBias;
                            none |= !(m[i] > -INFINITY);
                        }
                        if (__builtin_expect(__builtin_amdgcn_ballot_w64(none) != 0, 0)) break;
                    }
                    fresh = false;
                    half_values<true, 0, NB, NB>(o, l, m, x, sc, scale_log2);
                    half = left > 32 ? half ^ 1 : 0;  // the second holds nothing
                    if (half == 0 && ++k == n) break;
                }
                if (k == n) break;
                fresh = false;
                any_half<DT, NB>(o, m, l, bad, far, q, slot, half, scale_log2, lane, left, first_sees, row0, group);
                half = left > 32 ? half ^ 1 : 0;
                if (half == 0 && ++k == n) break;
            }
        }

        add_bad<NB>(o, bad);
        if (lane == 0) scan[wave] = (int)far;

        // ---- the waves' parts, joined: waves 4 to 7's into those of 0 to 3, means from then on; then a wave takes half the
        // dims of a row block
        __syncthreads();
        CK_LDS char *part = smem + (wave & (kParts - 1)) * kWidePart + 16 * lane_again(lane);
        auto ml_at = [](int i) { return 4 * 8 * 1024 + 1024 * (i >> 1) + 8 * (i & 1); };
        auto leave = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
#pragma unroll
                for (int k = 0; k < 8; ++k) *reinterpret_cast<CK_LDS f32x4 *>(part + (8 * i + k) * 1024) = o[i][k];
                *reinterpret_cast<CK_LDS f32x2 *>(part + ml_at(i)) = f32x2{m[i], l[i]};
            }
        };
        if (wave >= kParts) leave();
        __syncthreads();
        if (wave < kParts) {
            const float up0 = by_group(far, lane_again(lane), kRaise);
            const float up1 = by_group((uint32_t)scalar(scan[wave + kParts]), lane_again(lane), kRaise);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const f32x2 ml = *reinterpret_cast<const CK_LDS f32x2 *>(part + ml_at(i));
                const float top = fmaxf(m[i], ml[0]);
                float f0 = m[i] == -INFINITY ? 0.f : exp2_fast(m[i] - top);
                float f1 = ml[0] == -INFINITY ? 0.f : exp2_fast(ml[0] - top);
                l[i] = over_groups(l[i] * f0 + ml[1] * f1, [](float x, float y) { return x + y; });
                m[i] = top;
                const float inv = one_over(l[i]);
                f0 *= inv * up0;
                f1 *= inv * up1;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const f32x4 y = *reinterpret_cast<const CK_LDS f32x4 *>(part + (8 * i + k) * 1024);
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[i][k][r] = fmaf(o[i][k][r], f0, y[r] * f1);
                    if (k % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
            }
            leave();
        }
        __syncthreads();
        {
            a = args_again(args);
            const int x = lane_again(lane), n16 = x & 15, g = x >> 4, i = wave >> 1, k0 = 4 * (wave & 1);
            const CK_LDS char *p = smem + 16 * x;
            float top = -INFINITY, sum = 0.f;
            f32x2 ml[kParts];
#pragma unroll
            for (int w = 0; w < kParts; ++w) {
                ml[w] = *reinterpret_cast<const CK_LDS f32x2 *>(p + w * kWidePart + ml_at(i));
                top = fmaxf(top, ml[w][0]);
            }
#pragma unroll
            for (int w = 0; w < kParts; ++w) {
                ml[w][1] *= ml[w][0] == -INFINITY ? 0.f : exp2_fast(ml[w][0] - top);
                sum += ml[w][1];
            }
            const float inv = one_over(sum);
            f32x4 y[4];
#pragma unroll
            for (int w = 0; w < kParts; ++w) {
                const float f = ml[w][1] * inv;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const f32x4 z = *reinterpret_cast<const CK_LDS f32x4 *>(p + w * kWidePart + (8 * i + k0 + k) * 1024);
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[k][r] = w ? fmaf(z[r], f, y[k][r]) : z[r] * f;
                }
            }
            const bool whole = !before && !after && !a->merge;
            const int at = 16 * i + n16, r = kTileRows * tile + at;
            if (r < a->rows) {
                // dims 32 g + 8 d + k0 .. + 3
                if (whole) {
                    const int t = r / a->group;
                    const int64_t row = ((int64_t)b * q_len + t) * a->heads + h * a->group + (r - t * a->group);
#pragma unroll
                    for (int d = 0; d < 4; ++d)
                        *reinterpret_cast<uint2 *>(a->out + row * kD + 32 * g + 8 * d + k0) =
                            make_uint2(E::pack2(y[0][d], y[1][d]), E::pack2(y[2][d], y[3][d]));
                    if (g == 0 && k0 == 0) a->lse[row] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * kLn2;
                } else {
                    const int slot_rows = min(kTileRows, a->rows);
                    const int64_t slot = part_slot(before, after, share, a->waves, item) * a->tiles + tile;
                    float *to = a->part_o + slot * slot_rows * kD + (at * 4 + g) * 4;
#pragma unroll
                    for (int d = 0; d < 4; ++d)
                        *reinterpret_cast<f32x4 *>(to + (2 * d + (wave & 1)) * slot_rows * 16) = f32x4{y[0][d], y[1][d], y[2][d], y[3][d]};
                    if (g == 0 && k0 == 0) a->part_ml[slot * slot_rows + at] = make_float2(top, sum);
                }
            }
        }
        if (cur < hi) __syncthreads();
    }
    if constexpr (PAIR) {
        const List<kWideThreads, false> own(starts, len0, own_total);
        decode_share<DT, 1>(args + 1, own, nullptr, scalar(wave * (int)gridDim.x + (int)blockIdx.x), lane);
    }
}

// ---- the fold of cut items, and of a prefix with its suffixes ---------------------------------------------
struct FoldSide {
    const float *part_o;
    const float2 *part_ml;
    const int32_t *sums;
    const Shares *shares;
    int waves, tiles, tile_rows, slot_rows;
};
struct FoldArgs {
    FoldSide own, prefix;
    int q_len, heads, kv_heads, group;
    int rows;   // batch * q_len * heads
    int merge;  // with a prefix, and every part there
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
    const int before = f.sums[b], each = f.sums[b + 1] - before;
    const Shares cut = *f.shares;
    const int tile = r / f.tile_rows, at = r - tile * f.tile_rows;
    p.item = b * kv_heads + h;
    p.waves = f.waves;
    p.o_step = (int64_t)f.tiles * f.slot_rows * kD;
    p.ml_step = (int64_t)f.tiles * f.slot_rows;
    p.o = f.part_o + ((int64_t)tile * f.slot_rows * kD + at * 16);
    p.ml = f.part_ml + ((int64_t)tile * f.slot_rows + at);
    p.c0 = p.count = 0;
    if (each > 0) {
        const ShareRange r = shares_of(cut, h, before * kv_heads + h * each, each);
        p.c0 = r.first;
        p.count = r.count;
    }
    return p;
}

// 32 lanes hold a row's dims, lane (j, g) dims 32 g + 4 j .. + 3; PG such groups share its parts. O is the mean over the
// parts so far, their weights made to sum up to 1 for each batch.
template <int DT, int PG>
__global__ __launch_bounds__(256) void kv4_combine_kernel(FoldArgs a) {
    constexpr int kBlockRows = 8 / PG;
    const int group = threadIdx.x >> 5, lane = threadIdx.x & 31, pg = group % PG, g4 = lane & 3, j = lane >> 2;
    const int row = (int)blockIdx.x * kBlockRows + group / PG;  // below 2^24
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    bool done = row >= a.rows;  // or written by the wave that had all of it
    if (!done) {
        const int t = row / a.heads, head = row - t * a.heads, b = t / a.q_len, tok = t - b * a.q_len;
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
                const float old = (m == -INFINITY ? 0.f : exp2_fast(m - top)) * l;
                l = old;
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    if (i0 + i * PG >= p.count) continue;
                    ml[i].y *= ml[i].x == -INFINITY ? 0.f : exp2_fast(ml[i].x - top);
                    l += ml[i].y;
                }
                const float inv = one_over(l);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] *= old * inv;
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    if (i0 + i * PG >= p.count) continue;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = fmaf(po[i][e], ml[i].y * inv, o[e]);
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
        __shared__ f32x4 part[8][32];
        __shared__ float2 part_ml[8];
        part[group][lane] = o;
        if (lane == 0) part_ml[group] = make_float2(m, l);
        __syncthreads();
        if (pg > 0) return;  // the others of the row: group + 1 .. + PG - 1
        float top = m;
#pragma unroll
        for (int i = 1; i < PG; ++i) top = fmaxf(top, part_ml[group + i].x);
        l = 0.f;
        float f[PG];
#pragma unroll
        for (int i = 0; i < PG; ++i) {
            const float2 ml = part_ml[group + i];
            f[i] = (ml.x == -INFINITY ? 0.f : exp2_fast(ml.x - top)) * ml.y;
            l += f[i];
        }
        const float inv = one_over(l);
        o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < PG; ++i) {
            const f32x4 x = part[group + i][lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f[i] * inv, o[e]);
        }
        m = top;
    }
    if (done) return;
    using E = Elem<DT>;
    const uint2 x = make_uint2(E::pack2(o[0], o[1]), E::pack2(o[2], o[3]));
    *reinterpret_cast<uint2 *>(a.out + (int64_t)row * kD + 32 * g4 + 4 * j) = x;
    if (lane == 0) a.lse[row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
}

int64_t ceil_div(int64_t x, int64_t y) { return (x + y - 1) / y; }
int64_t pad256(int64_t n) { return (n + 255) & ~(int64_t)255; }

// One list over the waves (a call's requests, or its prefix) and its part of the workspace.
struct Side {
    int64_t rows, blocks, tile_rows, tiles, groups, waves, slot_rows, slots;
    bool wide;  // the form for many rows
    int64_t off_sums, off_ml, off_o, end;
};

// waves: the shares of a list whose launch another one sizes, or 0
int plan_side(int64_t batch, int64_t rows, int64_t kv_heads, int64_t kv_cap, bool merge, int64_t at, int64_t waves, Side *p) {
    p->rows = rows;
    p->wide = rows > 32;
    // 16 rows in the form for 16 / for 32, us a call: one request of 1300 tokens (8 kv heads) 10.3 / 11.0, 24 of 1000 20.0 /
    // 21.9, 64 of 4000 59.4 / 68.7; the form for 32 against that for 64 is at the top
    p->blocks = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    p->tile_rows = 16 * p->blocks;
    p->tiles = ceil_div(rows, p->tile_rows);
    if (p->wide) {  // shares of workgroups
        p->waves = p->tiles < kGroupsWide ? kGroupsWide / p->tiles : 1;
        p->groups = p->waves * p->tiles;
    } else {
        p->groups = kGroups;
        p->waves = waves ? waves : p->groups * kWaves;
    }
    if (!grid_fits(p->groups, kThreads)) return CK_E_INVALID_ARG;
    // the list's places are 32-bit, and its shares' numbers
    if (batch * kv_heads >= (int64_t)1 << 31 || batch * kv_heads * ceil_div(kv_cap, kUnit) >= (int64_t)1 << 31)
        return CK_E_INVALID_ARG;
    p->slot_rows = rows < p->tile_rows ? rows : p->tile_rows;
    p->slots = (2 * p->waves + (merge ? batch * kv_heads : 0)) * p->tiles;
    p->off_sums = at;
    p->off_ml = p->off_sums + pad256((batch + 1) * 4 + (int64_t)sizeof(Shares));
    p->off_o = p->off_ml + pad256(p->slots * p->slot_rows * 8);
    p->end = p->off_o + p->slots * p->slot_rows * kD * 4;
    return CK_OK;
}

struct Plan {
    Side own, prefix;
    bool paired;  // prefix and suffixes in one launch, of as many waves for both
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
    int rc;
    int64_t at = 0, waves = 0;
    p->paired = false;
    if (merge && batch > 0) {
        rc = plan_side(1, batch * group, kv_heads, prefix_cap, true, at, 0, &p->prefix);
        if (rc != CK_OK) return rc;
        at = p->prefix.end;
        p->paired = group <= 16;
        if (p->paired) waves = p->prefix.groups * (p->prefix.wide ? kWideWaves : kWaves);
    }
    rc = plan_side(batch, q_len * group, kv_heads, kv_cap, merge, at, waves, &p->own);
    if (rc != CK_OK) return rc;
    p->ws_bytes = p->own.end;
    return CK_OK;
}

template <int DT, bool PAIR, class A>
int launch_wide(const A &a, dim3 grid, hipStream_t s) {
    static std::atomic<uint64_t> lds_set{0};
    const int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(&kv4_wide_kernel<DT, PAIR>), kWideLds, lds_set);
    if (rc != CK_OK) return rc;
    hipLaunchKernelGGL((kv4_wide_kernel<DT, PAIR>), grid, dim3(kWideThreads), kWideLds, s, a);
    CK_RETURN_LAUNCH();
}

template <int DT, bool PAIR, class A>
int launch_side(const A &a, const Side &p, hipStream_t s) {
    const dim3 grid((unsigned)p.groups), block(kThreads);
    if (p.wide) return launch_wide<DT, PAIR>(a, grid, s);
    if (p.blocks == 1) hipLaunchKernelGGL((kv4_decode_kernel<DT, 1, PAIR>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((kv4_decode_kernel<DT, 2, PAIR>), grid, block, 0, s, a);
    CK_RETURN_LAUNCH();
}

template <int DT>
int launch(const DecodeArgs &own, const DecodeArgs *prefix, const Plan &p, const FoldArgs &f, hipStream_t s) {
    int rc = CK_OK;
    if (prefix && p.paired) {
        rc = launch_side<DT, true>(PairArgs{*prefix, own}, p.prefix, s);
    } else {
        if (prefix) rc = launch_side<DT, false>(*prefix, p.prefix, s);
        if (rc == CK_OK) rc = launch_side<DT, false>(own, p.own, s);
    }
    if (rc != CK_OK) return rc;
    auto fold = [&](auto groups) {
        constexpr int PG = groups;
        hipLaunchKernelGGL((kv4_combine_kernel<DT, PG>), dim3((unsigned)ceil_div(f.rows, 8 / PG)), dim3(256), 0, s, f);
    };
    if (f.rows <= kFoldRows[0]) fold(std::integral_constant<int, 8>{});
    else if (f.rows <= kFoldRows[1]) fold(std::integral_constant<int, 4>{});
    else if (f.rows <= kFoldRows[2]) fold(std::integral_constant<int, 2>{});
    else fold(std::integral_constant<int, 1>{});
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

void fill(DecodeArgs *a, FoldSide *f, const Pool &pool, const Side &p, int64_t batch, int64_t kv_heads, char *ws) {
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
    a->shares = reinterpret_cast<Shares *>(a->sums + batch + 1);
    a->pieces = p.wide && batch == 1 ? (int)(p.waves / kv_heads) : 0;
    *f = FoldSide{a->part_o, a->part_ml, a->sums, a->shares, a->waves, a->tiles, (int)p.tile_rows, (int)p.slot_rows};
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
    fill(&a, &f.own, pool, p.own, batch, kv_heads, ws);
    if (prefix) {  // one request, the batch's tokens in it, none hidden from another
        b.q_len = (int)batch;
        fill(&b, &f.prefix, *prefix, p.prefix, 1, kv_heads, ws);
    }
    f.q_len = (int)q_len;
    f.heads = a.heads;
    f.kv_heads = a.kv_heads;
    f.group = a.group;
    f.rows = (int)(batch * q_len * heads);
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
