// latent_decode.hip - attention in the absorbed form over a paged latent cache (gfx950),
// alone or with a prefix that all sequences share.
//
// Row (token i, head h) of request b, cache rows x_j = [c_j (512) | r_j (64)]:
//   s_j = scale q . x_j (576 dims), j < len_b - q_len + 1 + i
//   o = sum_j softmax(s)_j c_j (512 dims),  lse = log sum_j exp(s_j)
// A row that sees no token gets o = 0, lse = -inf.
//
// One cache row serves every head as key and as value: 1152 bytes feed 2176 flops per row of
// a query. Memory bounds calls of few rows, the matrix cores those of 64 rows and more; the form
// below reads a tile of 32 tokens once for up to 128 (token, head) rows.
// * A workgroup per CU, 4 waves, one per SIMD with all its 512 registers: a wave holds 32 rows of one
//   token (fewer heads leave rows empty, and an item of up to 32 rows three waves; a tile takes its
//   time all the same). Q is in 144 vector registers, O in the 256 accumulation registers; the wave
//   computes scores, softmax and O by itself, so that nothing crosses waves. Against 8 waves of 64 rows that divide
//   scores and O (P through LDS): 128 heads 640 -> 552 us at 117 sequences on 16001 shared tokens.
// * Tiles stream through a ring of 4 slots (37 KB, buffer -> LDS DMA), two in flight.
// * S^T = X Q^T and O^T = C^T P^T on 16x16x32 products: a key fragment is a 16-byte row read, C^T
//   comes from the same tile through ds_read_b64_tr_b16, P is in the operand's place as it leaves.
// * A step has one barrier and is one run of code without branches: P of tile t and the DMAs of tile
//   t + 3 are made in the shadow of tile t + 1's scores, the largest of those in that of tile t's
//   products. 3450 cycles for 128 rows x 32 tokens, of which the products alone take 2180.
// * The softmax's reference point m of a row is not its running maximum but a value that moves
//   only when some score passes it by 2^kSlack (any point gives the same result; p stays at or
//   below 2^kSlack), so that O is hardly ever rescaled (768 instructions).
// * Tiles of all requests form one list (each item with some empty places for what opening and
//   closing it costs), cut into equal chunks, one per workgroup (and per 128-row tile of a request),
//   so ragged lengths balance. A request inside one chunk is written as it is; parts of a cut one
//   go to the workspace as they are, with m and l, and latent_combine_kernel folds them.
// * Shared prefix: the flattened rows of the batch (sequence, head) form 128-row units over splits
//   of the prefix, which read each prefix tile once per 128 rows. The number of splits is chosen on
//   the device, so that the list of suffix tiles fills what the units leave; the combine folds
//   prefix and suffix parts in fp32.
// P is rounded to the cache's 16-bit type before the second product (its sum l is not): the
// relative error of o stays near that of o's own rounding.
// Measured, inputs changing from call to call: 48 x 16 heads over 12000 tokens (fp16, ragged) 92 us,
// 4.8 TB/s; 64 x 128 heads over 6000 103 us, 660 TFLOP/s (a fifth of it writes and folds the parts);
// 117 x 128 heads on 16001 shared tokens 475 us, 1.13 PFLOP/s (454 on the same inputs each time); 1 x 16
// heads over 1300 17 us, all latency; 24 x 7 x 16 heads over 5000 60 us, as 7 groups of 32 rows in two teams.
#include <algorithm>
#include <cmath>

#include "latent_common.h"
#include "latent_map.h"

namespace ck {
namespace {

using namespace lat;

typedef __attribute__((__vector_size__(2 * sizeof(unsigned)))) unsigned u32x2;

constexpr int kTok = 32;                      // tokens per tile
constexpr int kTilesPerPage = kPage / kTok;
constexpr int kTileBytes = kTok * kRowBytes;  // 36864
// A tile in LDS: 32 rows of the latent, 66 16-byte chunks apart, then 32 of the rotated
// dims, 8 chunks apart. A 16-byte read is served in groups of 16 lanes that are 8 rows of one
// chunk and the 8 others of the next one, a transpose read in groups of 8 rows x 2 chunks: with
// rows 2 bank groups apart both touch every bank group once, without any swizzle (and so with
// one address register). The rotated dims' rows, which a DMA writes without gaps, are XORed.
constexpr int kPitch = kR * 2 + 32;
constexpr int kRopeAt = kTok * kPitch;
constexpr int kSlotBytes = kRopeAt + kTok * kP * 2;
constexpr int kSlots = 4;
constexpr int kThreads = 256;  // 4 waves, one per SIMD, each with all of its 512 registers
constexpr int kWaveRows = 32;   // query rows per wave, two blocks of 16
constexpr int kRows = 128;      // query rows per workgroup
constexpr int kWaves = kThreads / 64;
constexpr int kPieces = 9;    // DMAs per wave and tile: 8 rows of the latent, and their rotated dims
constexpr int kPhase = 256;   // tiles described in LDS at a time
constexpr int kGroups = 256;  // workgroups: one per CU
// Least places of the list per chunk: short requests over more CUs against parts to fold. 2 against
// 4, us: 1 x 16 heads over 1300 tokens 17.2 / 18.9, 7 x 32 over 900 18.9 / 21.9, 2 x 128 over 3000
// 30.9 / 30.2.
constexpr int kMinPlaces = 2;
// Blocks of 16 rows from which on the fold gives a wave all parts. In that form / the other, us a call:
// 64 blocks 24 / 22 (64 x 16 heads over 600) to 66 / 48 (8 x 128 over 12000), 128 blocks 29 / 30 to 65 / 61,
// 256 blocks 39 / 42 to 48 / 47 (32 x 128 over 3000), 384 blocks 50 / 55 to 136 / 136, 512 blocks 61 / 68 to 157 / 159
// (shared prefix, 64 x 128: 115 / 111). Where they meet grows with the parts, from 128 blocks to 384.
constexpr int kFoldBlocks = 256;
constexpr int kFoldThreads = 256;
constexpr float kSlack = 8.f;

constexpr int kLdsZero = kSlots * kSlotBytes;  // a row of zeros
constexpr int kLdsDesc = kLdsZero + kPitch;
constexpr int kLdsPlace = kLdsDesc + kPhase * 16;
constexpr int kLdsScan = kLdsPlace + kPhase * 8;
constexpr int kLdsStart = kLdsScan + 64;  // each thread's place in the list
constexpr int kLdsLen = kLdsStart + kThreads * 4;  // and its first request's length
constexpr int kLds = kLdsLen + kThreads * 4;
static_assert(kPhase == kThreads, "a tile per thread");
static_assert(kLds <= 160 * 1024, "LDS");

// XOR of the 8 chunks of row r's rotated dims (128 bytes: bit 0 of r is the bank half).
__device__ __forceinline__ int swz(int r) {
    return ((r & 2) << 1) | ((((r >> 2) ^ (r >> 3)) & 1) << 1) | ((r >> 3) & 1);
}

struct DecodeArgs {
    const uint16_t *q;      // [batch * q_len, heads, 576]
    const uint16_t *cache;
    const int32_t *bt;
    const int64_t *lens;
    int64_t bt_cols;
    int64_t num_blocks;
    int batch;
    int q_len;
    int heads;
    int rows;     // per request: q_len * heads
    int head_groups;  // 32-row groups of a token's heads, one per wave: its rows see the same tokens
    int teams;    // row tiles of a request given to workgroups of their own
    int listed;   // row tiles of a request listed one after another (teams == 1)
    int chunks;   // workgroups per team
    float scale_log2;
    void *out;    // [batch * q_len, heads, 512]
    float *lse;   // [batch * q_len * heads]
    // Parts, not normalised, are kept by blocks of 16 rows as the lanes hold them, [128 x 4 dims][16 rows][4]:
    // neighbouring lanes then store and load neighbouring bytes. Lanes in different rows (2 KB
    // apart) took a cycle each, 16000 of them for a workgroup's 256 KB.
    float *part_o;    // [slots][slot_rows / 16][128][16][4]
    float2 *part_ml;  // [slots][slot_rows]: reference point (log2) and sum of p
    int32_t *sums;    // [batch + 2]: the list's places before each request and in all; the prefix's splits
    int slot_rows;
    int merge;        // 1: every part goes to the workspace (a prefix is folded in)
    // shared prefix (merge == 1)
    const uint16_t *pcache;
    const int32_t *pbt;
    const int64_t *plen;
    int64_t pcols;
    int64_t pblocks;
    int prows;    // batch * heads
    int prows_up;  // in whole row tiles
    int pmtiles;
    int most_splits;
    float *ppart_o;    // [splits][prows_up / 16][128][16][4]
    float2 *ppart_ml;  // [splits][prows_up]
};

__device__ __forceinline__ int64_t clamp_len(int64_t n, int64_t cols, int64_t num_blocks) {
    const int64_t cap = cols * kPage;
    if (n > cap) n = cap;
    return n < 0 || num_blocks <= 0 ? 0 : n;
}
__device__ __forceinline__ int tiles_of(int64_t len) { return (int)((len + kTok - 1) / kTok); }
__device__ __forceinline__ int places_of(int64_t len) { return len > 0 ? tiles_of(len) + kItemPlaces : 0; }

// op over the four lanes n, 16 + n, 32 + n, 48 + n, in each of them: exchanging the odd rows of
// 16 lanes (then the upper half) of x with the even ones (the lower half) of x leaves one
// operand in each result.
template <class Op>
__device__ __forceinline__ float over_groups(float x, Op &&op) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Of a row's 32 dims, x its dims 4 g .. + 3 and y its dims 16 + 4 g .. + 3 in lane group g:
// 8 neighbouring ones, from dim 16 (g & 1) + 8 (g >> 1) on, rounded once to 16 bits.
template <int DT>
__device__ __forceinline__ u32x4 eight_dims(f32x4 x, f32x4 y) {
    using E = Elem<DT>;
    const auto lo = __builtin_amdgcn_permlane16_swap(E::pack2(x[0], x[1]), E::pack2(y[0], y[1]), false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap(E::pack2(x[2], x[3]), E::pack2(y[2], y[3]), false, false);
    return u32x4{lo[0], hi[0], lo[1], hi[1]};
}

typedef const __attribute__((address_space(4))) DecodeArgs *KernArgs;
__device__ __forceinline__ KernArgs args_again(KernArgs a) {
    asm volatile("" : "+s"(a));
    return a;
}

// ---- O: the accumulation registers -----------------------------------------------------------
// O^T of a wave's 32 rows is 512 dims x 32 rows of fp32, all 256 accumulation registers of a
// lane: block (db, i) of 16 dims x 16 rows is a[8 db + 4 i .. + 3]. The compiler cannot hold
// values there that vector instructions also touch (it moves them to vector registers, which
// Q fills), so O is kept out of its sight: only the statements below name these registers. It
// has no use of its own for them, as long as it spills nothing (the build checks that).
// acc_ready stands between the last write of an operand and the first product, acc_done
// between the last product and a read (a product takes 4 passes of 4 cycles).
constexpr int acc_at(int db, int i) { return 8 * db + 4 * i; }

__device__ __forceinline__ void acc_zero() {
    // 16 products of zeros: a register at a time is twice the time and 2 KB of code
    u32x4 zero = {0, 0, 0, 0};
    asm volatile("s_nop 7" : "+v"(zero));
    static_for<16>([zero](auto n) __attribute__((always_inline)) {
        asm volatile("v_mfma_f32_32x32x16_bf16 a[%c0:%c1], %2, %2, 0" ::"i"(16 * int(n)), "i"(16 * int(n) + 15), "v"(zero));
    });
    asm volatile("" ::: "a255");  // all of them belong to the kernel
}
__device__ __forceinline__ void acc_ready(u32x4 &x, u32x4 &y) { asm volatile("s_nop 7" : "+v"(x), "+v"(y)); }
__device__ __forceinline__ void acc_done() { asm volatile("s_nop 15\n\ts_nop 15"); }
template <int DT, int DB, int I>
__device__ __forceinline__ void acc_mfma(u32x4 a, u32x4 b) {
    constexpr int n = acc_at(DB, I);
    if constexpr (DT == CK_DTYPE_BF16)
        asm volatile("v_mfma_f32_16x16x32_bf16 a[%c0:%c1], %2, %3, a[%c0:%c1]" ::"i"(n), "i"(n + 3), "v"(a), "v"(b));
    else
        asm volatile("v_mfma_f32_16x16x32_f16 a[%c0:%c1], %2, %3, a[%c0:%c1]" ::"i"(n), "i"(n + 3), "v"(a), "v"(b));
}
template <int N>
__device__ __forceinline__ float acc_read1() {
    float x;
    asm volatile("v_accvgpr_read_b32 %0, a%c1" : "=v"(x) : "i"(N));
    return x;
}
template <int DB, int I>
__device__ __forceinline__ f32x4 acc_read() {
    constexpr int n = acc_at(DB, I);
    return f32x4{acc_read1<n>(), acc_read1<n + 1>(), acc_read1<n + 2>(), acc_read1<n + 3>()};
}
// Blocks (DB, I) to 16 bytes a lane at base + at + 1024 * (DB - DB0), for DB0 .. DB0 + 3.
template <int DB0, int I>
__device__ __forceinline__ void acc_store4(const float *base, int at) {
    static_for<4>([base, at](auto k) __attribute__((always_inline)) {
        constexpr int n = acc_at(DB0 + k, I);
        asm volatile("global_store_dwordx4 %0, a[%c1:%c2], %3 offset:%c4" ::"v"(at), "i"(n), "i"(n + 3), "s"(base), "i"(1024 * k)
                     : "memory");
    });
}
// Rows of block i times f_i.
__device__ __forceinline__ void acc_scale(float f0, float f1) {
    static_for<256>([&](auto n) __attribute__((always_inline)) {
        const float x = acc_read1<n>() * ((n / 4) % 2 ? f1 : f0);
        asm volatile("v_accvgpr_write_b32 a%c0, %1" ::"i"(int(n)), "v"(x));
    });
}

template <int DT>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(1, 1))) void latent_decode_kernel(DecodeArgs) {
    using E = Elem<DT>;
    // The arguments, read where they are used: held in scalar registers throughout they would
    // spill, into vector registers that Q and O need.
    const KernArgs first_args = args_again((KernArgs)__builtin_amdgcn_kernarg_segment_ptr());
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    CK_LDS char *smem = (CK_LDS char *)smem_raw;
    CK_LDS int *desc = (CK_LDS int *)(smem + kLdsDesc);  // {page, item, first token, length}
    CK_LDS u32x2 *place = (CK_LDS u32x2 *)(smem + kLdsPlace);  // a described tile's bytes into its pool
    CK_LDS int *scan = (CK_LDS int *)(smem + kLdsScan);
    CK_LDS int *bad = scan + kWaves;  // the last phase with an invalid page
    const int wave = scalar((int)threadIdx.x >> 6);
    const int lane = __lane_id();
    const int first_tid = 64 * wave + lane;

    const uint32_t lw = xcd_remap(blockIdx.x, gridDim.x);
    const int wg = scalar((int)(lw / first_args->teams)), team = (int)lw - wg * first_args->teams;

    // ---- the list: this thread's requests, their first tile, the total --------------------
    auto first_request = [](KernArgs a, int t) {
        return min(t * ((a->batch + kThreads - 1) / kThreads), a->batch);  // batch is at most 2^24
    };
    auto len_of = [](KernArgs a, int b) { return (int)clamp_len(a->lens[b], a->bt_cols, a->num_blocks); };
    CK_LDS int *starts = (CK_LDS int *)(smem + kLdsStart), *len0 = (CK_LDS int *)(smem + kLdsLen);
    int total = 0;
    const int64_t plen = first_args->merge ? *first_args->plen : 0;
    {
        int mine = 0;
        const int b0 = first_request(first_args, first_tid), b1 = first_request(first_args, first_tid + 1);
        for (int b = b0; b < b1; ++b) {
            const int len = len_of(first_args, b);
            if (b == b0) len0[first_tid] = len;
            mine += places_of(len) * first_args->listed;
        }
        const int incl = (int)wave_scan((uint32_t)mine, 0x7fffffffu);
        if (lane == 63) scan[wave] = incl;
        if (first_tid == 0) *bad = 0;
        __syncthreads();
        int start = incl - mine;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) {
            if (i < wave) start += scan[i];
            total += scan[i];
        }
        starts[first_tid] = start;
        total = scalar(total);
    }

    // ---- this workgroup's share ------------------------------------------------------------
    int ptiles = 0, unit_tiles = 0, units = 0, splits = 0;
    if (first_args->merge) {
        ptiles = scalar(tiles_of(clamp_len(plen, first_args->pcols, first_args->pblocks)));
        if (ptiles > 0) {
            // a choice per lane
            const Split mine = split_choice(lane & (kSplitChoices - 1), first_args->pmtiles, ptiles, total, kGroups,
                                            min(first_args->most_splits, ptiles));
            auto of = [&](int i) {
                return Split{__builtin_amdgcn_readlane(mine.splits, i),
                             __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine.end), i))};
            };
            Split best = of(0);
#pragma unroll
            for (int i = 1; i < kSplitChoices; ++i)
                if (better(of(i), best)) best = of(i);
            splits = best.splits;
            unit_tiles = scalar((ptiles + splits - 1) / splits);
            units = first_args->pmtiles * splits;
        }
    }
    const ListMap map = list_map(total, first_args->chunks, kMinPlaces, units, unit_tiles + kItemPlaces);
    const int chunk = scalar(wg < map.ra ? wg : wg - map.ra + map.a.chunks);
    const bool has_list = scalar((int)(wg < map.ra ? wg < map.a.chunks : wg - map.ra < map.b.chunks));
    const int lo = has_list ? scalar(list_lo(map, chunk)) : 0, hi = has_list ? scalar(list_lo(map, chunk + 1)) : 0;

    // ---- per-lane addresses ------------------------------------------------------------------
    for (int i = first_tid; i < kPitch / 4; i += kThreads) ((CK_LDS int *)(smem + kLdsZero))[i] = 0;

    // The lane again, for addresses that are not to be held over the steps: there are no registers
    // for them beside Q (O has the accumulation registers).
    struct Lane {
        int id, g, n16;
        __device__ __forceinline__ explicit Lane(int l) {
            asm volatile("" : "+v"(l));
            id = l;
            g = l >> 4;
            n16 = l & 15;
        }
    };
    // Those that are: of a key's latent part and rotated part (first 32 dims; the others ^ 64),
    // of a value's, and of the DMAs (rows 8 wave .. + 7 of the latent, one each, and their rotated
    // dims together).
    const int k_addr = (lane & 15) * kPitch + (lane >> 4) * 16;
    const int r_addr = kRopeAt + (lane & 15) * (kP * 2) + (((lane >> 4) ^ swz(lane & 15)) & 7) * 16;
    const int v_row = 4 * (lane >> 4) + ((lane & 15) >> 2), v_addr = v_row * kPitch + (lane & 3) * 8;
    const int rope_row = 8 * wave + (lane >> 3);
    const int rope_off = rope_row * kRowBytes + kR * 2 + ((lane & 7) ^ swz(rope_row)) * 16;

    // ---- a segment: an item's tiles in this workgroup -----------------------------------------
    struct Segment {
        int64_t row0;  // row i of the wave is row row0 + i of q, i < rows_n
        int rows_n;
        int limit;     // tokens that the wave's rows see
        int item;
        int began_before;
    };
    Segment seg = {0, 0, 0, -1, 0};
    const float scale_log2 = first_args->scale_log2;
    u32x4 qf[2][18];
    bool fresh = false;  // O is zero
    float m_row[2], sub[2], l_part[2];  // per row: reference point, what scores are lowered by, sum of p

    CK_LDS int *mark = (CK_LDS int *)smem;  // in the ring's place: [kPhase] each
    CK_LDS int *seg_item = mark + kPhase, *seg_at = seg_item + kPhase, *seg_len = seg_at + kPhase;
    int unit = wg, phase = 0;
    int at_prefix = 0, at_list = lo;  // within the unit; in the list
    for (;;) {
        const KernArgs a = args_again(first_args);
        const int tid = 64 * wave + Lane(lane).id;  // again: its places in the tables are not to be held either
        // ---- describe the next tiles, at most kPhase: a prefix unit's, then the list's -------
        const bool in_prefix = unit < units;
        ++phase;
        auto describe = [&](int i, int page, int64_t blocks, int item, int tile, int len) {
            const bool ok = page >= 0 && page < blocks;
            const int64_t at = ok ? (int64_t)page * kPageBytes + (tile % kTilesPerPage) * kTileBytes : 0;
            *reinterpret_cast<CK_LDS u32x4 *>(desc + 4 * i) =
                u32x4{ok ? 1u : 0u, (unsigned)item, (unsigned)(tile * kTok), (unsigned)len};
            place[i] = u32x2{(unsigned)at, (unsigned)(at >> 32)};
            if (!ok) *bad = phase;
        };
        int n, sp = 0;
        int64_t prefix_row0 = 0;
        bool last;
        const char *cache;
        if (in_prefix) {
            // row tiles inner: workgroups side by side read the same prefix tiles
            sp = scalar(unit / a->pmtiles);
            const int mt = unit - sp * a->pmtiles;
            const int p_lo = sp * unit_tiles + at_prefix, p_hi = min((sp + 1) * unit_tiles, ptiles);
            n = max(0, min(kPhase, p_hi - p_lo));
            last = p_lo + n >= p_hi;
            cache = reinterpret_cast<const char *>(a->pcache);
            prefix_row0 = (int64_t)mt * kRows + kWaveRows * wave;  // rows of all sequences, one after another
            if (tid < n) {
                const int tile = p_lo + tid;
                describe(tid, a->pbt[tile / kTilesPerPage], a->pblocks, unit, tile, (int)min(a->plen[0], a->pcols * kPage));
            }
            at_prefix += n;
            if (last) {
                unit += a->chunks;
                at_prefix = 0;
            }
            if (n == 0) continue;  // past a short prefix's end: the combine counts the splits the same way
        } else if (at_list < hi) {
            const int ph = at_list, places = min(kPhase, hi - ph);
            last = ph + places >= hi;
            at_list += places;
            cache = reinterpret_cast<const char *>(a->cache);
            mark[tid] = 0;
            __syncthreads();
            int at = starts[tid];
            const int b0 = first_request(a, tid), b1 = first_request(a, tid + 1);
            for (int b = b0; b < b1 && at < ph + places; ++b) {
                const int len = b == b0 ? len0[tid] : len_of(a, b);
                const int each = places_of(len);
                for (int m = 0; m < a->listed; ++m, at += each) {
                    if (each > 0 && at < ph + places && at + each > ph) {
                        const int i = max(at, ph) - ph;
                        mark[i] = 1;
                        seg_item[i] = b * a->listed + m;
                        seg_at[i] = max(at, ph) - at;
                        seg_len[i] = len;
                    }
                }
            }
            __syncthreads();
            // Place i's item is that of the last mark at or before it. Each mark past the first is
            // followed by kItemPlaces empty places, which the tiles close up over.
            const Lane l(lane);
            int item_at = 0, last_at = 0, marks = 0, all_marks = 0;  // marks: up to this place
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const uint64_t all = __builtin_amdgcn_ballot_w64(mark[64 * w + l.id] != 0);
                const uint64_t mine = w < wave ? all : w == wave ? all & (~0ull >> (63 - l.id)) : 0;
                if (mine) item_at = 64 * w + 63 - __clzll(mine);
                if (all) last_at = 64 * w + 63 - __clzll(all);
                marks += __popcll(mine);
                all_marks += __popcll(all);
            }
            const int skipped = kItemPlaces - min(kItemPlaces, seg_at[0]);  // of the first mark
            n = scalar(places - kItemPlaces * (all_marks - 1) - skipped + max(0, kItemPlaces - (seg_at[last_at] + places - last_at)));
            const int off = seg_at[item_at] + tid - item_at;
            if (tid < places && off >= kItemPlaces) {
                const int it = seg_item[item_at], tile = off - kItemPlaces;
                describe(tid - kItemPlaces * (marks - 1) - skipped,
                         a->bt[(int64_t)(it / a->listed) * a->bt_cols + tile / kTilesPerPage], a->num_blocks, it, tile, seg_len[item_at]);
            }
        } else {
            break;
        }
        __syncthreads();
        if (n == 0) continue;  // empty places

        // ---- the tiles ------------------------------------------------------------------------
        struct Tile {
            int ok, item, first, len;  // ok: of a page in the pool
        };
        auto tile_at = [&](int t) {  // past the last, it again
            const u32x4 d = *reinterpret_cast<const CK_LDS u32x4 *>(desc + 4 * min(t, n - 1));
            return Tile{scalar((int)d[0]), scalar((int)d[1]), scalar((int)d[2]), scalar((int)d[3])};
        };
        const bool all_ok = scalar(*bad) != phase;
        // This wave's moves of tile t into its slot. A resource without bytes moves nothing but
        // zeros, so that every step issues the same number.
        struct Moves {
            ck_rsrc_t r;
            int base;
        };
        auto place_at = [&](int t) { return place[min(t, n - 1)]; };
        auto moves_of = [&](u32x2 at, int t, bool ok) {
            const uint64_t from = (uint64_t)(uintptr_t)cache + (((uint64_t)(uint32_t)scalar((int)at[1]) << 32) | (uint32_t)scalar((int)at[0]));
            Moves m;
            m.r[0] = (int)(uint32_t)from;
            m.r[1] = (int)((uint32_t)(from >> 32) & 0xffffu);
            m.r[2] = t < n && ok ? kTileBytes : 0;
            m.r[3] = 0x00020000;
            m.base = scalar((int)(uintptr_t)smem + (t & (kSlots - 1)) * kSlotBytes + 8 * wave * kPitch);
            return m;
        };
        const int rows_at = scalar(8 * wave * kRowBytes);
        auto move = [&](const Moves &m, auto j) __attribute__((always_inline)) {
            if constexpr (j < 8) dma_tile<j * kPitch>(m.r, lane * 16, rows_at + j * kRowBytes, m.base);
            else dma_tile<kRopeAt>(m.r, rope_off, 0, m.base - 8 * wave * kPitch + wave * 1024);
        };
        // An invalid page reads as zeros: this wave's part of it, once the DMAs are through.
        auto blank = [&](int t) {
            CK_LDS char *dst = smem + (t & (kSlots - 1)) * kSlotBytes + Lane(lane).id * 16;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                *reinterpret_cast<CK_LDS u32x4 *>(dst + (8 * wave + j) * kPitch) = u32x4{0, 0, 0, 0};
            *reinterpret_cast<CK_LDS u32x4 *>(dst + kRopeAt + wave * 1024) = u32x4{0, 0, 0, 0};
        };

        // The segment that tile d begins or goes on with.
        auto segment_of = [&](const Tile &d) {
            const KernArgs a = args_again(first_args);
            Segment x = {prefix_row0, 0, d.len, d.item, d.first > 0};
            if (in_prefix) {
                x.rows_n = (int)max((int64_t)0, min((int64_t)kWaveRows, a->prows - prefix_row0));
                if (x.rows_n == 0) x.row0 = 0;
                return x;
            }
            const int b = scalar(d.item / a->listed);
            const int group = (a->teams > 1 ? team : d.item - b * a->listed) * 4 + wave;  // of the request
            const int tok = scalar(group / a->head_groups), head = kWaveRows * (group - tok * a->head_groups);
            x.rows_n = tok < a->q_len ? min(kWaveRows, a->heads - head) : 0;
            x.row0 = x.rows_n > 0 ? ((int64_t)b * a->q_len + tok) * a->heads + head : 0;
            x.limit = max(0, min(d.len, d.len - a->q_len + 1 + tok));
            return x;
        };
        // Q comes in pieces of 256 contiguous bytes for 16 lanes (an operand's own place, 64 lanes in
        // 16 rows, costs a cycle a lane: 9200 of them for a workgroup's 128 rows) and is turned
        // into operands through LDS: piece (m, e), rows 4 e .. + 3, dims 128 m .. + 127, waits in the
        // registers of operand (e / 4, 4 m + e % 4); the rotated dims in 8 rows x 128 bytes.
        auto load_q = [&](const Segment &x) {  // a row past the last repeats it: it is not stored
            const KernArgs a = args_again(first_args);
            const Lane l(lane);
            const int end = x.rows_n - 1;
            const uint16_t *q = a->q + x.row0 * kRow;
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    qf[e >> 2][4 * m + (e & 3)] =
                        *reinterpret_cast<const u32x4 *>(q + min(4 * e + l.g, end) * kRow + 128 * m + 8 * l.n16);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                qf[e >> 1][16 + (e & 1)] =
                    *reinterpret_cast<const u32x4 *>(q + min(8 * e + (l.id >> 3), end) * kRow + kR + 8 * (l.id & 7));
        };
        // Through the wave's own 8 rows of the slot of tile t, which nothing moves to or reads now.
        auto turn_q = [&](int t) {
            const Lane l(lane);
            CK_LDS char *at = smem + (t & (kSlots - 1)) * kSlotBytes + 8 * wave * kPitch;
            auto piece = [&](int row, int chunk) {  // of [32][16] chunks: the 16 of a row XORed
                return reinterpret_cast<CK_LDS u32x4 *>(at + row * 256 + ((chunk ^ row) & 15) * 16);
            };
#pragma unroll
            for (int m = 0; m < 4; ++m) {
#pragma unroll
                for (int e = 0; e < 8; ++e) *piece(4 * e + l.g, l.n16) = qf[e >> 2][4 * m + (e & 3)];
#pragma unroll
                for (int e = 0; e < 8; ++e) qf[e >> 2][4 * m + (e & 3)] = *piece(16 * (e >> 2) + l.n16, 4 * (e & 3) + l.g);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) *piece(8 * e + (l.id >> 3), l.id & 7) = qf[e >> 1][16 + (e & 1)];
#pragma unroll
            for (int e = 0; e < 4; ++e) qf[e >> 1][16 + (e & 1)] = *piece(16 * (e >> 1) + l.n16, 4 * (e & 1) + l.g);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // before the next move there
        };
        auto start = [&]() {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                m_row[i] = -INFINITY;
                sub[i] = -E::kBias;
                l_part[i] = 0.f;
            }
            acc_zero();
            fresh = true;
        };

        // S^T = X Q^T of tile t: tokens 4 g + r and 16 + 4 g + r of rows n16 and 16 + n16.
        // between(f) is placed after the f-th pair of products: what fits in their shadow.
        f32x4 s[2][2];  // [16 tokens][16 rows]
        float v[2];     // the rows' largest score in the lane
        auto scores = [&](int t, f32x4 (&x)[2][2], auto &&between) __attribute__((always_inline)) {
            const CK_LDS char *tile = smem + (t & (kSlots - 1)) * kSlotBytes;
            auto kfrag = [&](int f) {
                const int kk = f >> 1;
                const CK_LDS char *at = kk < 16 ? tile + k_addr + kk * 64 + (f & 1) * 16 * kPitch
                                                : tile + (r_addr ^ ((kk & 1) << 6)) + (f & 1) * 16 * kP * 2;
                return *reinterpret_cast<const CK_LDS u32x4 *>(at);
            };
            constexpr int kAhead = 4, kHeld = kAhead + 1;
            u32x4 kf[kHeld];
#pragma unroll
            for (int f = 0; f < 4; ++f) x[f >> 1][f & 1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int f = 0; f < kAhead; ++f) kf[f] = kfrag(f);
            __builtin_amdgcn_sched_barrier(0);
            static_for<36>([&](auto f) __attribute__((always_inline)) {
                x[f & 1][0] = E::mfma16(kf[f % kHeld], qf[0][f >> 1], x[f & 1][0]);
                if (f + kAhead < 36) kf[(f + kAhead) % kHeld] = kfrag(f + kAhead);
                __builtin_amdgcn_sched_barrier(0);
                x[f & 1][1] = E::mfma16(kf[f % kHeld], qf[1][f >> 1], x[f & 1][1]);
                between(f);
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        auto hide = [&](int sees) {  // scores of tokens that the rows do not see
            if (sees < kTok) {
                const Lane l(lane);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (16 * h + 4 * l.g + r >= sees) s[h][0][r] = s[h][1][r] = -INFINITY;
            }
        };
        auto largest = [&](const f32x4 (&x)[2][2], int i) {
            v[i] = max3(max3(max3(x[0][i][0], x[0][i][1], x[0][i][2]), x[0][i][3], x[1][i][0]), x[1][i][1],
                        fmaxf(x[1][i][2], x[1][i][3])) * scale_log2;
        };
        auto nothing = [](int) {};
        // Whether a score passes its row's reference point by more than 2^kSlack.
        auto moves = [&]() {
            return __builtin_amdgcn_ballot_w64(v[0] > m_row[0] + kSlack || v[1] > m_row[1] + kSlack) != 0;
        };
        u32x4 pf[2];  // P^T of a tile: the scores' token order is the operand's
        auto p_of = [&](int e) __attribute__((always_inline)) {  // two of the lane's 16 probabilities
            const int i = e / 4, h = e / 2 % 2, r = e % 2;
            const float p0 = exp2_fast(fmaf(s[h][i][2 * r], scale_log2, -sub[i]));
            const float p1 = exp2_fast(fmaf(s[h][i][2 * r + 1], scale_log2, -sub[i]));
            l_part[i] += p0;
            l_part[i] += p1;
            pf[i][2 * h + r] = E::pack2(p0, p1);
        };
        // O^T += C^T P^T of a tile whose rows 4 g + n16 / 4 (+ 16) are at v0 (v1).
        auto products = [&](const CK_LDS char *v0, const CK_LDS char *v1, auto &&between) __attribute__((always_inline)) {
            constexpr int kAhead = 4, kHeld = kAhead + 1;
            uint2 va[kHeld], vb[kHeld];
#pragma unroll
            for (int db = 0; db < kAhead; ++db) {
                va[db] = lds_read_tr16(v0 + db * 32);
                vb[db] = lds_read_tr16(v1 + db * 32);
            }
            __builtin_amdgcn_sched_barrier(0);
            acc_ready(pf[0], pf[1]);
            static_for<32>([&](auto db) __attribute__((always_inline)) {
                constexpr int at = (db + kAhead) % kHeld;
                const uint2 x = va[db % kHeld], y = vb[db % kHeld];
                const u32x4 c = {x.x, x.y, y.x, y.y};
                acc_mfma<DT, db, 0>(c, pf[0]);
                if (db + kAhead < 32) va[at] = lds_read_tr16(v0 + (db + kAhead) * 32);
                __builtin_amdgcn_sched_barrier(0);
                acc_mfma<DT, db, 1>(c, pf[1]);
                if (db + kAhead < 32) vb[at] = lds_read_tr16(v1 + (db + kAhead) * 32);
                between(db);
                __builtin_amdgcn_sched_barrier(0);
            });
        };

        // ---- the phase's first tiles ------------------------------------------------------------
        {
            const Tile d = tile_at(0);
            const bool opens = d.item != seg.item;
            if (opens) seg = segment_of(d);
            auto move_tile = [&](int t) {
                const Moves m = moves_of(place_at(t), t, tile_at(t).ok);
                static_for<kPieces>([&](auto j) __attribute__((always_inline)) { move(m, j); });
            };
            move_tile(0);
            if (seg.rows_n > 0) load_q(seg);  // in each phase, so that it is not held while the tiles are described
            if (opens) start();
            wait_vmcnt<0>();
            if (seg.rows_n > 0) turn_q(3);
            move_tile(1);
            move_tile(2);
            if (!d.ok) blank(0);
            __syncthreads();
            if (seg.rows_n > 0) {
                scores(0, s, nothing);
                hide(seg.limit - d.first);
                largest(s, 0);
                largest(s, 1);
            }
        }
        bool stored = false;  // the last step ended with stores, not to be waited for yet
        for (int t = 0; t < n; ++t) {
            // ---- a step in general ----------------------------------------------------------------
            // Tile t + 1 is in, in every wave; tile t + 3 takes the place of tile t - 1. The scores
            // of tile t are there.
            const Tile d0 = tile_at(t), d1 = tile_at(t + 1);
            if (!stored) wait_vmcnt<kPieces>();  // such a step waited for it before its stores
            if (!d1.ok) blank(t + 1);
            __syncthreads();
            stored = false;
            const bool goes_on = d0.first + kTok < d0.len;
            const bool ends = !goes_on || (last && t + 1 == n);
            const bool carries = !ends && t + 1 < n;  // tile t + 1 is the segment's too
            const bool opens = ends && t + 1 < n;     // tile t + 1 opens another
            Segment next = seg;
            if (opens) {  // Q's registers are free since the scores of tile t
                next = segment_of(d1);
                if (next.rows_n > 0) load_q(next);
            }
            if (seg.rows_n > 0) {
                if (moves()) {
                    float scale[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float m_new = fmaxf(m_row[i], over_groups(v[i], [](float x, float y) { return fmaxf(x, y); }));
                        scale[i] = m_new == -INFINITY ? 1.f : exp2_fast(m_row[i] - m_new);
                        m_row[i] = m_new;
                        sub[i] = (m_new == -INFINITY ? 0.f : m_new) - E::kBias;
                        l_part[i] *= scale[i];
                    }
                    if (!fresh) acc_scale(scale[0], scale[1]);
                }
                fresh = false;
                static_for<8>([&](auto e) __attribute__((always_inline)) { p_of(e); });
                // Tokens that the rows do not see (past the length they may hold anything) are read
                // as zeros: 0 * inf must not reach O.
                const int sees = seg.limit - d0.first;
                const CK_LDS char *at = smem + (t & (kSlots - 1)) * kSlotBytes + v_addr;
                products(v_row < sees ? at : smem + kLdsZero, v_row + 16 < sees ? at + 16 * kPitch : smem + kLdsZero, nothing);
            }
            // Q, and tile t + 2: before the moves and stores below. Whether the step opens a segment
            // or not: at Q's use in the plain steps the compiler would wait otherwise.
            wait_vmcnt<0>();
            if (opens && next.rows_n > 0) turn_q(t + 3);
            {
                const Moves m = moves_of(place_at(t + 3), t + 3, tile_at(t + 3).ok);
                static_for<kPieces>([&](auto j) __attribute__((always_inline)) { move(m, j); });
            }
            if (carries && seg.rows_n > 0) {
                scores(t + 1, s, nothing);
                hide(seg.limit - d1.first);
                largest(s, 0);
                largest(s, 1);
            }

            // ---- the segment's end ------------------------------------------------------------------
            if (ends) {
                const KernArgs a = args_again(first_args);
                float *po = nullptr;  // the wave's first row of its part
                float2 *pl = nullptr;
                if (in_prefix) {
                    const int64_t row = sp * (int64_t)a->prows_up + seg.row0;
                    po = a->ppart_o + row * kR;
                    pl = a->ppart_ml + row;
                } else if (a->merge || seg.began_before || goes_on) {
                    const int64_t slot = seg.began_before || goes_on ? part_slot(seg.began_before, chunk, a->teams, team)
                                                                     : (int64_t)2 * a->chunks * a->teams + seg.item;
                    const int64_t row = slot * a->slot_rows + kWaveRows * wave;
                    po = a->part_o + row * kR;
                    pl = a->part_ml + row;
                }
                const Lane l(lane);
                acc_done();
                static_for<2>([&](auto i) __attribute__((always_inline)) {
                    const float sum = over_groups(l_part[i], [](float x, float y) { return x + y; });
                    const int row = 16 * i + l.n16;
                    const bool is_row = row < seg.rows_n;
                    if (po != nullptr) {  // as it is: the fold divides
                        if (is_row) {
                            static_for<8>([&](auto q) __attribute__((always_inline)) {
                                acc_store4<4 * q, i>(po + 16 * i * kR + 1024 * q, 16 * l.id);
                            });
                            if (l.g == 0) pl[row] = make_float2(m_row[i], sum);
                        }
                    } else {
                        // 0 where no token was seen (or every score was -inf)
                        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
                        const float lse2 = sum == 0.f ? -INFINITY : m_row[i] - E::kBias + log2f(sum);
                        uint16_t *out = static_cast<uint16_t *>(a->out) + (seg.row0 + row) * kR + 16 * (l.g & 1) + 8 * (l.g >> 1);
                        static_for<16>([&](auto p) __attribute__((always_inline)) {
                            const u32x4 o = eight_dims<DT>(acc_read<2 * p, i>() * inv, acc_read<2 * p + 1, i>() * inv);
                            if (is_row) *reinterpret_cast<u32x4 *>(out + 32 * p) = o;
                        });
                        if (is_row && l.g == 0) a->lse[seg.row0 + row] = lse2 * kLn2;
                    }
                });
                asm volatile("s_nop 7" ::: "memory");  // the stores have read O
                stored = seg.rows_n > 0;
                seg.item = -1;
                if (opens) {
                    seg = next;
                    start();
                    if (seg.rows_n > 0) {
                        scores(t + 1, s, nothing);
                        hide(seg.limit - d1.first);
                        largest(s, 0);
                        largest(s, 1);
                    }
                }
            }

            // ---- plain steps: whole tiles of one segment, no reference point moves ---------------------
            // One run of code without branches (one between products costs as much as two of them),
            // and as few other instructions as the products' shadow holds: alone on its SIMD, a
            // wave issues one in four cycles, three beside each product. P of tile t is made and tile
            // t + 3 is moved beside the scores of tile t + 1, the largest of those is taken
            // beside the products of tile t.
            if (!carries || stored || seg.rows_n == 0 || !all_ok || moves()) continue;
            // the last step whose tile and next are seen whole
            const int end = min(n - 1, t + 1 + max(0, (seg.limit - d1.first) / kTok - 1));
            bool moved = false;
            while (t + 1 < end && !moved) {
                ++t;
                const u32x2 at3 = place_at(t + 3);
                wait_vmcnt<kPieces>();
                __syncthreads();
                f32x4 s2[2][2];
                Moves m;
                scores(t + 1, s2, [&](auto f) __attribute__((always_inline)) {
                    if constexpr (f == 0) m = moves_of(at3, t + 3, true);
                    if constexpr (f >= 4 && f < 31 && f % 3 == 1) move(m, std::integral_constant<int, f / 3 - 1>{});
                    if constexpr (f >= 2 && f < 34 && f % 4 == 2) p_of((f - 2) / 4);
                });
                const CK_LDS char *tile = smem + (t & (kSlots - 1)) * kSlotBytes + v_addr;
                products(tile, tile + 16 * kPitch, [&](auto db) __attribute__((always_inline)) {
                    if constexpr (db == 4) largest(s2, 0);
                    if constexpr (db == 8) largest(s2, 1);
                    if constexpr (db == 12) moved = moves();
                    if constexpr (db >= 16 && db < 20) s[(db - 16) / 2][db % 2] = s2[(db - 16) / 2][db % 2];
                });
            }
        }
        wait_vmcnt<0>();  // the empty moves too
        __syncthreads();  // the tables and the ring are free
    }

    if (wg == 0 && team == 0) {
        const KernArgs a = args_again(first_args);
        const int tid = 64 * wave + Lane(lane).id;
        int at = starts[tid];
        for (int b = first_request(a, tid); b < first_request(a, tid + 1); ++b) {
            a->sums[b] = at;
            at += places_of(len_of(a, b)) * a->listed;
        }
        if (tid == 0) {
            a->sums[a->batch] = total;
            a->sums[a->batch + 1] = splits;
        }
    }
}

// Folds the parts of every row that has some, in list order and after the prefix's, and
// writes rows that see nothing. A workgroup takes 16 heads of a token, a lane one row and 4 dims
// of each 16, the part's own layout; kAhead parts are loaded independently of each other. Where
// the blocks fill the CUs (SHARE false) a wave has 8 x 16 dims of all parts; where they do not, the
// dims go over 8 workgroups and the parts over 4 waves, which are joined through LDS.
template <int DT, bool SHARE>
__global__ __launch_bounds__(kFoldThreads) void latent_combine_kernel(DecodeArgs a) {
    constexpr int kDb = SHARE ? 4 : 8, kAhead = SHARE ? 4 : 2, kStep = SHARE ? 4 : 1;
    const int lane = __lane_id(), g = lane >> 4, n16 = lane & 15, wave = scalar((int)threadIdx.x >> 6);
    const int head_blocks = (a.heads + 15) / 16;
    const int token = scalar((int)(blockIdx.x / head_blocks)), hb = (int)blockIdx.x - token * head_blocks;
    const int b = scalar(token / a.q_len), tok = token - b * a.q_len;
    const int db0 = SHARE ? blockIdx.y * kDb : wave * kDb;
    const int head = 16 * hb + n16;
    const int group = tok * a.head_groups + hb / 2, mt = group / 4;
    const int row = (group - 4 * mt) * kWaveRows + 16 * (hb & 1) + n16;
    const int team = a.teams > 1 ? mt : 0, m = a.teams > 1 ? 0 : mt;
    const int places = scalar((a.sums[b + 1] - a.sums[b]) / a.listed);

    int ptiles = 0, unit_tiles = 0, splits = 0, units = 0;
    if (a.merge) {
        ptiles = tiles_of(clamp_len(*a.plen, a.pcols, a.pblocks));
        if (ptiles > 0) {
            const int dealt = a.sums[a.batch + 1];
            unit_tiles = scalar((ptiles + dealt - 1) / dealt);
            units = a.pmtiles * dealt;
            splits = scalar((ptiles + unit_tiles - 1) / unit_tiles);  // that hold tiles
        }
    }
    int c0 = 0, parts = 0;
    bool whole = false;
    if (places > 0) {
        const ListMap map = list_map(a.sums[a.batch], a.chunks, kMinPlaces, units, unit_tiles + kItemPlaces);
        const int at = a.sums[b] + m * places;
        c0 = scalar(list_chunk(map, at + kItemPlaces));
        parts = scalar(list_chunk(map, at + places - 1)) - c0 + 1;
        whole = parts == 1;
        if (whole && !a.merge) return;  // written by its workgroup
    }
    const int total = splits + parts;
    const int64_t prow = (int64_t)b * a.heads + min(head, a.heads - 1);  // of the prefix's rows
    const float *prefix_o = a.ppart_o + ((prow >> 4) * 128 + 4 * db0 + g) * 64 + (prow & 15) * 4;
    float mx = -INFINITY, sum = 0.f;
    f32x4 acc[kDb] = {};
    for (int p0 = SHARE ? wave : 0; p0 < total; p0 += kStep * kAhead) {
        float2 ml[kAhead];
        f32x4 o[kAhead][kDb];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int p = min(p0 + j * kStep, total - 1);  // past the last part: it again, not added
            const float *po;
            if (p < splits) {
                ml[j] = a.ppart_ml[(int64_t)p * a.prows_up + prow];
                po = prefix_o + (int64_t)p * a.prows_up * kR;
            } else {
                const int c = c0 + p - splits;
                const int64_t slot = whole ? (int64_t)2 * a.chunks * a.teams + b * a.listed + m : part_slot(c > c0, c, a.teams, team);
                ml[j] = a.part_ml[slot * a.slot_rows + row];
                po = a.part_o + (slot * a.slot_rows + row - n16) * kR + db0 * 256 + 4 * lane;
            }
#pragma unroll
            for (int d = 0; d < kDb; ++d) o[j][d] = *reinterpret_cast<const f32x4 *>(po + d * 256);
        }
        float mb = mx;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (p0 + j * kStep < total) mb = fmaxf(mb, ml[j].x);
        }
        const float mu = mb == -INFINITY ? 0.f : mb;
        const float f = exp2_fast(mx - mu);
        mx = mb;
        sum *= f;
#pragma unroll
        for (int d = 0; d < kDb; ++d) acc[d] *= f;
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            if (p0 + j * kStep < total) {
                const float w = exp2_fast(ml[j].x - mu);  // 0 of a part that saw nothing, which holds zeros
                sum = fmaf(ml[j].y, w, sum);
#pragma unroll
                for (int d = 0; d < kDb; ++d) acc[d] += o[j][d] * w;
            }
    }
    const int64_t r = (int64_t)token * a.heads + head;
    uint16_t *out = static_cast<uint16_t *>(a.out) + r * kR;
    if constexpr (SHARE) {
        __shared__ f32x4 part[4][kDb][64];
        __shared__ float part_mx[4][16], part_sum[4][16];
#pragma unroll
        for (int d = 0; d < kDb; ++d) part[wave][d][lane] = acc[d];
        if (g == 0) {
            part_mx[wave][n16] = mx;
            part_sum[wave][n16] = sum;
        }
        __syncthreads();
        // a wave each of the four 16 dims
        mx = fmaxf(fmaxf(part_mx[0][n16], part_mx[1][n16]), fmaxf(part_mx[2][n16], part_mx[3][n16]));
        const float mu = mx == -INFINITY ? 0.f : mx;
        sum = 0.f;
        f32x4 x = {};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = exp2_fast(part_mx[w][n16] - mu);  // a wave without a part: zeros
            sum += part_sum[w][n16] * f;
            x += part[w][wave][lane] * f;
        }
        x *= sum == 0.f ? 0.f : 1.0f / sum;
        using E = Elem<DT>;
        if (head < a.heads)
            *reinterpret_cast<uint2 *>(out + 16 * (db0 + wave) + 4 * g) = make_uint2(E::pack2(x[0], x[1]), E::pack2(x[2], x[3]));
    } else {
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
#pragma unroll
        for (int d = 0; d < kDb; d += 2) {
            const u32x4 x = eight_dims<DT>(acc[d] * inv, acc[d + 1] * inv);
            if (head < a.heads) *reinterpret_cast<u32x4 *>(out + 16 * (db0 + d + (g & 1)) + 8 * (g >> 1)) = x;
        }
    }
    if (db0 == 0 && wave == 0 && g == 0 && head < a.heads)
        a.lse[r] = sum == 0.f ? -INFINITY : (mx - Elem<DT>::kBias + log2f(sum)) * kLn2;
}

int64_t ceil_div(int64_t x, int64_t y) { return (x + y - 1) / y; }
int64_t pad256(int64_t n) { return (n + 255) & ~(int64_t)255; }

// Sizes of a call: the list's and the prefix's partition, and the workspace.
struct LatentPlan {
    int64_t rows, head_groups, mtiles, teams, listed, chunks, slot_rows, slots;
    int64_t prows, prows_up, pmtiles, psplits;
    int64_t off_ml, off_o, off_pml, off_po, ws_bytes;
};

int make_plan(int64_t batch, int64_t q_len, int64_t heads, int64_t kv_cap, bool merge, int64_t prefix_cap,
              LatentPlan *p) {
    if (batch < 0 || q_len < 1 || heads < 1 || kv_cap < 0 || prefix_cap < 0) return CK_E_INVALID_ARG;
    if (batch > (1 << 24) || q_len > (1 << 24) || heads > (1 << 16) || kv_cap > ((int64_t)1 << 30) ||
        prefix_cap > ((int64_t)1 << 30) || batch * q_len >= ((int64_t)1 << 31) / heads ||
        !grid_fits(batch * q_len * ceil_div(heads, 16), kFoldThreads))
        return CK_E_INVALID_ARG;
    p->rows = q_len * heads;
    p->head_groups = ceil_div(heads, kWaveRows);
    const int64_t groups = q_len * p->head_groups;
    p->mtiles = ceil_div(groups, 4);
    p->teams = merge ? 1 : p->mtiles;
    p->listed = merge ? p->mtiles : 1;
    p->chunks = p->teams >= kGroups ? 1 : kGroups / p->teams;
    // the list's places and the sums are 32-bit
    if (batch * p->listed * (ceil_div(kv_cap, kTok) + kItemPlaces) >= (int64_t)1 << 31) return CK_E_INVALID_ARG;
    p->slot_rows = kWaveRows * (groups < 4 ? groups : 4);
    p->slots = 2 * p->chunks * p->teams + (merge ? batch * p->listed : 0);
    p->prows = merge ? batch * heads : 0;
    p->pmtiles = ceil_div(p->prows, kRows);
    p->prows_up = p->pmtiles * kRows;
    p->psplits = 0;
    if (merge && p->pmtiles > 0) {
        p->psplits = p->pmtiles >= 2 * kGroups ? 1 : 2 * kGroups / p->pmtiles;  // two rounds
        const int64_t most = ceil_div(prefix_cap, 2 * kTok);  // of two tiles at least
        if (p->psplits > most) p->psplits = most < 1 ? 1 : most;
    }
    int64_t at = pad256((batch + 2) * 4);
    p->off_ml = at;
    at += pad256(p->slots * p->slot_rows * 8);
    p->off_pml = at;
    at += pad256(p->psplits * p->prows_up * 8);
    p->off_o = at;
    at += p->slots * p->slot_rows * kR * 4;
    p->off_po = at;
    at += p->psplits * p->prows_up * kR * 4;
    p->ws_bytes = at;
    return CK_OK;
}

template <int DT>
int launch(const DecodeArgs &a, hipStream_t s) {
    static std::atomic<uint64_t> lds_set{0};
    int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(&latent_decode_kernel<DT>), kLds, lds_set);
    if (rc != CK_OK) return rc;
    hipLaunchKernelGGL((latent_decode_kernel<DT>), dim3((unsigned)(a.teams * a.chunks)), dim3(kThreads), kLds, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return static_cast<int>(e);
    const int64_t blocks = (int64_t)a.batch * a.q_len * ceil_div(a.heads, 16);
    if (blocks >= kFoldBlocks)
        hipLaunchKernelGGL((latent_combine_kernel<DT, false>), dim3((unsigned)blocks), dim3(kFoldThreads), 0, s, a);
    else
        hipLaunchKernelGGL((latent_combine_kernel<DT, true>), dim3((unsigned)blocks, 32 / 4), dim3(kFoldThreads), 0, s, a);
    CK_RETURN_LAUNCH();
}

struct PrefixArgs {
    const void *cache;
    const int32_t *bt;
    const int64_t *len;
    int64_t cols, num_blocks;
};

int run(const void *q, const void *cache, const int32_t *block_table, int64_t bt_cols, const int64_t *kv_seqlens,
        int64_t batch, int64_t q_len, int64_t heads, int64_t num_blocks, int64_t block_size, int dtype, float scale,
        const PrefixArgs *prefix, void *out, float *lse, void *workspace, int64_t workspace_bytes, hipStream_t s) {
    auto tokens_of = [](int64_t cols) { return cols < 0 ? -1 : std::min(cols, (int64_t)1 << 30) * kPage; };  // no overflow
    LatentPlan p;
    int rc = make_plan(batch, q_len, heads, tokens_of(bt_cols), prefix != nullptr, prefix ? tokens_of(prefix->cols) : 0, &p);
    if (rc != CK_OK) return rc;
    if (block_size != kPage || (dtype != CK_DTYPE_BF16 && dtype != CK_DTYPE_F16)) return CK_E_UNSUPPORTED;
    if (num_blocks < 0 || num_blocks > ((int64_t)1 << 31)) return CK_E_INVALID_ARG;
    if (prefix && (prefix->num_blocks < 0 || prefix->num_blocks > ((int64_t)1 << 31))) return CK_E_INVALID_ARG;
    if (!(scale > 0.f) || !std::isfinite(scale * kLog2e)) return CK_E_INVALID_ARG;
    if (batch == 0) return CK_OK;
    if (!q || !kv_seqlens || !out || !lse || (bt_cols > 0 && (!block_table || (num_blocks > 0 && !cache))))
        return CK_E_NULL_PTR;
    if (prefix && (!prefix->len || (prefix->cols > 0 && (!prefix->bt || (prefix->num_blocks > 0 && !prefix->cache)))))
        return CK_E_NULL_PTR;
    if (!aligned_to(q, 16) || !aligned_to(cache, 16) || !aligned_to(out, 16) || !aligned_to(lse, 4) ||
        !aligned_to(workspace, 16) || !aligned_to(block_table, 4) || !aligned_to(kv_seqlens, 8))
        return CK_E_INVALID_ARG;
    if (prefix && (!aligned_to(prefix->cache, 16) || !aligned_to(prefix->bt, 4) || !aligned_to(prefix->len, 8)))
        return CK_E_INVALID_ARG;
    if (!workspace || workspace_bytes < p.ws_bytes) return CK_E_WORKSPACE;

    DecodeArgs a = {};
    char *ws = static_cast<char *>(workspace);
    a.q = static_cast<const uint16_t *>(q);
    a.cache = static_cast<const uint16_t *>(cache);
    a.bt = block_table;
    a.lens = kv_seqlens;
    a.bt_cols = bt_cols;
    a.num_blocks = num_blocks;
    a.batch = (int)batch;
    a.q_len = (int)q_len;
    a.heads = (int)heads;
    a.rows = (int)p.rows;
    a.teams = (int)p.teams;
    a.listed = (int)p.listed;
    a.chunks = (int)p.chunks;
    a.scale_log2 = scale * kLog2e;
    a.out = out;
    a.lse = lse;
    a.sums = reinterpret_cast<int32_t *>(ws);
    a.part_ml = reinterpret_cast<float2 *>(ws + p.off_ml);
    a.part_o = reinterpret_cast<float *>(ws + p.off_o);
    a.slot_rows = (int)p.slot_rows;
    a.head_groups = (int)p.head_groups;
    a.merge = prefix != nullptr;
    if (prefix) {
        a.pcache = static_cast<const uint16_t *>(prefix->cache);
        a.pbt = prefix->bt;
        a.plen = prefix->len;
        a.pcols = prefix->cols;
        a.pblocks = prefix->num_blocks;
        a.prows = (int)p.prows;
        a.prows_up = (int)p.prows_up;
        a.pmtiles = (int)p.pmtiles;
        a.most_splits = (int)p.psplits;
        a.ppart_ml = reinterpret_cast<float2 *>(ws + p.off_pml);
        a.ppart_o = reinterpret_cast<float *>(ws + p.off_po);
    }
    return dtype == CK_DTYPE_BF16 ? launch<CK_DTYPE_BF16>(a, s) : launch<CK_DTYPE_F16>(a, s);
}

}  // namespace
}  // namespace ck

using namespace ck;

extern "C" int ck_latent_decode_plan(int64_t batch, int64_t q_len, int64_t num_heads, int64_t kv_cap,
                                     int64_t *workspace_bytes) {
    if (!workspace_bytes) return CK_E_NULL_PTR;
    LatentPlan p;
    int rc = make_plan(batch, q_len, num_heads, kv_cap, false, 0, &p);
    if (rc == CK_OK) *workspace_bytes = p.ws_bytes;
    return rc;
}

extern "C" int ck_latent_decode(const void *q, const void *cache, const int32_t *block_table, int64_t bt_cols,
                                const int64_t *kv_seqlens, int64_t batch, int64_t q_len, int64_t num_heads,
                                int64_t num_blocks, int64_t block_size, int dtype, float scale, void *out, float *lse,
                                void *workspace, int64_t workspace_bytes, void *stream) {
    return run(q, cache, block_table, bt_cols, kv_seqlens, batch, q_len, num_heads, num_blocks, block_size, dtype,
               scale, nullptr, out, lse, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int ck_latent_cascade_decode_plan(int64_t batch, int64_t num_heads, int64_t prefix_cap, int64_t suffix_cap,
                                             int64_t *workspace_bytes) {
    if (!workspace_bytes) return CK_E_NULL_PTR;
    LatentPlan p;
    int rc = make_plan(batch, 1, num_heads, suffix_cap, true, prefix_cap, &p);
    if (rc == CK_OK) *workspace_bytes = p.ws_bytes;
    return rc;
}

extern "C" int ck_latent_cascade_decode(const void *q, const void *prefix_cache, const int32_t *prefix_block_table,
                                        int64_t prefix_bt_cols, const int64_t *prefix_kv_seqlen,
                                        int64_t prefix_num_blocks, const void *suffix_cache,
                                        const int32_t *suffix_block_table, int64_t suffix_bt_cols,
                                        const int64_t *suffix_kv_seqlens, int64_t suffix_num_blocks, int64_t batch,
                                        int64_t num_heads, int64_t block_size, int dtype, float scale, void *out,
                                        float *lse, void *workspace, int64_t workspace_bytes, void *stream) {
    const PrefixArgs prefix{prefix_cache, prefix_block_table, prefix_kv_seqlen, prefix_bt_cols, prefix_num_blocks};
    return run(q, suffix_cache, suffix_block_table, suffix_bt_cols, suffix_kv_seqlens, batch, 1, num_heads,
               suffix_num_blocks, block_size, dtype, scale, &prefix, out, lse, workspace, workspace_bytes,
               reinterpret_cast<hipStream_t>(stream));
}
