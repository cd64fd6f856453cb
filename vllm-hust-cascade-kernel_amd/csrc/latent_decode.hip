// latent_decode.hip - attention in the absorbed form over a paged latent cache (gfx950),
// alone or with a prefix that all sequences share.
//
// Row (token i, head h) of request b, cache rows x_j = [c_j (512) | r_j (64)]:
//   s_j = scale q . x_j (576 dims), j < len_b - q_len + 1 + i
//   o = sum_j softmax(s)_j c_j (512 dims),  lse = log sum_j exp(s_j)
// A row that sees no token gets o = 0, lse = -inf.
//
// One cache row serves every head as key and as value, so a tile of it in LDS feeds the
// query rows of up to 64 (token, head) pairs:
// * A workgroup (one per CU, 8 waves) streams 32-token tiles through a ring of 4 slots
//   (36 KB each, buffer -> LDS DMA), two of them in flight while one is computed, for up to
//   64 query rows. Wave w computes scores of rows 16 (w % 4) .. + 15 against tokens
//   16 (w / 4) .. + 15 (Q in registers, 72 of them), and owns value dims 64 w .. + 63 of all
//   64 rows (O in registers, 64 of them): P crosses the waves through LDS, O never does.
// * S^T = X Q^T and O^T = C^T P^T on 16x16x32 MFMAs: K fragments are 16-byte row reads, C^T
//   comes from the same tile through ds_read_b64_tr_b16, and a lane holds one query row of
//   the accumulator.
// * One barrier per tile. The softmax's reference point m of a row is not its running
//   maximum but a value that moves only when some score exceeds it by 2^kSlack (any point
//   gives the same result; p stays at or below 2^kSlack): a wave raises a flag beside its P,
//   and the raised tile alone exchanges maxima, rescales O and computes P again.
// * Tiles of all requests form one list, cut into equal chunks, one per workgroup (and per
//   64-row tile of a request), so ragged lengths balance. A request inside one chunk is
//   written as it is; parts of a cut one go to the workspace, normalised, with their lse, and
//   latent_combine_kernel folds them.
// * Shared prefix: the flattened rows of the batch (sequence, head) form 64-row units over
//   splits of the prefix, which read each prefix tile once per 64 rows; what a
//   workgroup has left after its unit it spends on suffix tiles, and the combine
//   folds prefix and suffix parts in fp32.
// P is rounded to the cache's 16-bit type before the second product (its sum l is not): the
// relative error of o stays near that of o's own rounding.
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
constexpr int kSlots = 4;
constexpr int kRows = 64;   // query rows per workgroup
constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kPPitch = 80;  // bytes per row of P (32 tokens; odd in 16-byte units, so rows spread over the banks)
constexpr int kPBytes = kRows * kPPitch;
constexpr int kPhase = 128;  // tiles described in LDS at a time
constexpr int kGroups = 256; // workgroups: one per CU
constexpr float kSlack = 8.f;

constexpr int kProducers = 4;  // waves that compute scores; the others own O

constexpr int kLdsP = kSlots * kTileBytes;
constexpr int kLdsDesc = kLdsP + 2 * kPBytes;
constexpr int kLdsMax = kLdsDesc + kPhase * 16;      // fp32 [2 token halves][64]: row maxima of a tile
constexpr int kLdsFac = kLdsMax + 2 * kRows * 4;     // fp32 [64]: what O is scaled by
constexpr int kLdsSum = kLdsFac + kRows * 4;         // fp32 [2][3][64]: a closing segment's sums and reference points
constexpr int kLdsFlag = kLdsSum + 2 * 3 * kRows * 4;
constexpr int kLdsScan = kLdsFlag + 16;
constexpr int kLds = kLdsScan + 64;
static_assert(kLds <= 160 * 1024, "LDS");

// XOR of a token's 16-byte chunks inside a 128-byte group. A row is 9 such groups, so row r
// starts in bank half r % 2; with bits 1, 3, 2 of r here, 16 consecutive rows' chunks lie in
// 16 distinct bank groups (score reads), and so do 4 consecutive rows x 2 chunks of rows
// r and r + 8 (transpose reads).
__device__ __forceinline__ int swz(int r) { return ((r & 2) << 1) | ((r >> 2) & 2) | ((r >> 2) & 1); }

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
    int teams;    // 64-row tiles of a request given to workgroups of their own
    int listed;   // 64-row tiles of a request listed one after another (teams == 1)
    int chunks;   // workgroups per team
    int min_tiles;  // least tiles per chunk
    float scale_log2;
    void *out;    // [batch * q_len, heads, 512]
    float *lse;   // [batch * q_len * heads]
    float *part_o;    // [slots][slot_rows][512]
    float *part_lse;  // [slots][slot_rows], log2
    int32_t *sums;    // [batch + 1]: tiles of the list before each request
    int slot_rows;
    int merge;        // 1: every part goes to the workspace (a prefix is folded in)
    // shared prefix (merge == 1)
    const uint16_t *pcache;
    const int32_t *pbt;
    const int64_t *plen;
    int64_t pcols;
    int64_t pblocks;
    int prows;    // batch * heads
    int pmtiles;
    int psplits;
    float *ppart_o;    // [psplits][prows][512]
    float *ppart_lse;  // [psplits][prows], log2
};

__device__ __forceinline__ int64_t prefix_tiles(const DecodeArgs &a) {
    int64_t n = a.plen[0];
    const int64_t cap = a.pcols * kPage;
    if (n > cap) n = cap;
    if (n < 0 || a.pblocks <= 0) n = 0;
    return (n + kTok - 1) / kTok;
}
__device__ __forceinline__ int64_t clamp_len(int64_t n, const DecodeArgs &a) {
    const int64_t cap = a.bt_cols * kPage;
    if (n > cap) n = cap;
    return n < 0 || a.num_blocks <= 0 ? 0 : n;
}

// What a workgroup works on, the same in all its threads but for the thread's requests.
struct Share {
    int team, wg;
    int units;           // prefix units, dealt round-robin
    int64_t ptiles, unit_tiles;
    int chunk;           // numbered chunk of the list: tiles [lo, hi)
    int64_t lo, hi;
    int b_lo, b_hi;      // this thread's requests
    int64_t my_start;    // and the list's tiles before them
};

// One role of a workgroup: the producers compute a tile's scores and P, the consumers move
// the tiles in and own O. Both walk the same tiles between the same barriers:
//   interval t: consumers issue tile t + 3; all look at tile t's flag; producers: scores and
//   P of tile t + 1; consumers: O += of tile t, wait for tile t + 2; barrier
template <int DT, int NB, bool PRODUCER>
__device__ __forceinline__ void role_loop(const DecodeArgs &a, const Share &w, CK_LDS char *smem) {
    using E = Elem<DT>;
    CK_LDS int *desc = (CK_LDS int *)(smem + kLdsDesc);  // {page, item, first token, length}
    CK_LDS float *xmax = (CK_LDS float *)(smem + kLdsMax);
    CK_LDS float *fac = (CK_LDS float *)(smem + kLdsFac);
    CK_LDS int *flag = (CK_LDS int *)(smem + kLdsFlag);
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int g = lane >> 4, n16 = lane & 15;

    // producer: rows 32 rh .. + 31 (two blocks of 16), tokens 16 tb .. + 15
    const int rh = wave & 1, tb = (wave >> 1) & 1;
    u32x4 qf[2][18];
    f32x4 s[2];
    float m_own[2], l_part[2];
    int limit[2];  // tokens that this lane's rows see
    const int krow = 16 * tb + n16;
    const int k_addr = krow * kRowBytes + ((g ^ swz(krow)) & 7) * 16;  // even steps; odd ones ^ 64

    // consumer: value dims 128 cw .. + 127 of all rows, and KB cw + 4 j of every tile
    const int cw = wave & 3;
    f32x4 oacc[8][NB];  // [16-dim block][16-row block]
    int dma_off[9], dma_row[9], v_addr[2];
    if constexpr (!PRODUCER) {
#pragma unroll
        for (int j = 0; j < 9; ++j) {
            const int l = (cw + 4 * j) * 64 + lane;  // 16-byte chunk of the tile in LDS
            const int r = l / (kRowBytes / 16), c = l - r * (kRowBytes / 16);
            dma_row[j] = r;
            dma_off[j] = r * kRowBytes + ((c & ~7) | ((c ^ swz(r)) & 7)) * 16;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = 8 * g + 4 * h + (n16 >> 2);
            v_addr[h] = r * kRowBytes + cw * 256 + ((((n16 >> 1) & 1) ^ swz(r)) << 4) + (n16 & 1) * 8;
        }
    }

    // the segment at hand: both roles, each at its own tile
    int item = -1;
    int64_t row0 = 0;
    int rows_n = 0, nblk = 0;  // rows, and this wave's 16-row blocks of them
    bool began_before = false, ends = false, goes_on = false;
    int parity = 0;  // of the segment, for its sums' place
    int stamp = 0;   // tiles before this phase's

    CK_LDS int *mark = (CK_LDS int *)(smem + kLdsP);  // in P's place: [kPhase] each
    CK_LDS int *seg_item = mark + kPhase, *seg_tile = seg_item + kPhase, *seg_len = seg_tile + kPhase;
    int unit = w.wg;
    int64_t at_prefix = 0, at_list = w.lo;  // within the unit; in the list
    for (;;) {
        // ---- describe the next tiles, at most kPhase: a prefix unit's, then the list's -------
        const bool in_prefix = unit < w.units;
        int n, sp = 0;
        bool last;
        const char *cache;
        if (in_prefix) {
            // row tiles inner: workgroups side by side read the same prefix tiles
            const int mt = unit % a.pmtiles;
            sp = unit / a.pmtiles;
            const int64_t p_lo = sp * w.unit_tiles + at_prefix, p_hi = min((sp + 1) * w.unit_tiles, w.ptiles);
            n = (int)max((int64_t)0, min((int64_t)kPhase, p_hi - p_lo));
            last = p_lo + n >= p_hi;
            cache = reinterpret_cast<const char *>(a.pcache);
            row0 = (int64_t)mt * kRows;
            rows_n = (int)min((int64_t)kRows, a.prows - row0);
            if (tid < n) {
                const int64_t tile = p_lo + tid;
                const int page = a.pbt[tile / kTilesPerPage];
                desc[4 * tid] = page >= 0 && page < a.pblocks ? page : -1;
                desc[4 * tid + 1] = unit;
                desc[4 * tid + 2] = (int)(tile * kTok);
                desc[4 * tid + 3] = (int)min(a.plen[0], a.pcols * kPage);
            }
            at_prefix += n;
            if (last) {
                unit += a.chunks;
                at_prefix = 0;
            }
            if (n == 0) continue;  // past a short prefix's end: the combine counts the splits the same way
        } else if (at_list < w.hi) {
            const int64_t ph = at_list;
            n = (int)min((int64_t)kPhase, w.hi - ph);
            last = ph + n >= w.hi;
            cache = reinterpret_cast<const char *>(a.cache);
            if (tid < kPhase) mark[tid] = 0;
            __syncthreads();
            int64_t at = w.my_start;
            for (int b = w.b_lo; b < w.b_hi && at < ph + n; ++b) {
                const int64_t len = clamp_len(a.lens[b], a);
                const int each = (int)((len + kTok - 1) / kTok);
                for (int m = 0; m < a.listed; ++m, at += each) {
                    if (each > 0 && at < ph + n && at + each > ph) {
                        const int i = (int)(max(at, ph) - ph);
                        mark[i] = 1;
                        seg_item[i] = b * a.listed + m;
                        seg_tile[i] = (int)(max(at, ph) - at);
                        seg_len[i] = (int)len;
                    }
                }
            }
            __syncthreads();
            // the last segment start at or before tile tid
            const uint64_t lo_mask = __builtin_amdgcn_ballot_w64(mark[lane] != 0);
            const uint64_t hi_mask = __builtin_amdgcn_ballot_w64(mark[64 + lane] != 0);
            if (tid < n) {
                const uint64_t upto = ~0ull >> (63 - lane);
                const int i = tid < 64 ? 63 - __clzll(lo_mask & upto)
                              : hi_mask & upto ? 127 - __clzll(hi_mask & upto) : 63 - __clzll(lo_mask);
                const int it = seg_item[i], tile = seg_tile[i] + tid - i;
                const int page = a.bt[(int64_t)(it / a.listed) * a.bt_cols + tile / kTilesPerPage];
                desc[4 * tid] = page >= 0 && page < a.num_blocks ? page : -1;
                desc[4 * tid + 1] = it;
                desc[4 * tid + 2] = tile * kTok;
                desc[4 * tid + 3] = seg_len[i];
            }
        } else {
            break;
        }
        if (!in_prefix) at_list += n;
        __syncthreads();

        // ---- a tile's item, length and first token; a new item's rows -------------------------
        int first = 0, len = 0;
        auto step_to = [&](int t) {  // true where tile t opens a segment
            const u32x4 d = *reinterpret_cast<const CK_LDS u32x4 *>(desc + 4 * t);
            const int it = __builtin_amdgcn_readfirstlane(d[1]);
            first = __builtin_amdgcn_readfirstlane(d[2]);
            len = __builtin_amdgcn_readfirstlane(d[3]);
            goes_on = first + kTok < len;
            ends = !goes_on || (last && t + 1 == n);
            if (it == item) return false;
            item = it;
            began_before = first > 0;
            if (!in_prefix) {
                const int b = it / a.listed, first_row = (a.teams > 1 ? w.team : it - b * a.listed) * kRows;
                row0 = (int64_t)b * a.rows + first_row;
                rows_n = min(kRows, a.rows - first_row);
            }
            return true;
        };

        if constexpr (PRODUCER) {
            auto write_p = [&](int t, int i) {
                const float sub = (m_own[i] == -INFINITY ? 0.f : m_own[i]) - E::kBias;
                float p[4], ls = 0.f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[r] = exp2_fast(s[i][r] - sub);
                    ls += p[r];
                }
                *reinterpret_cast<CK_LDS u32x2 *>(smem + kLdsP + (t & 1) * kPBytes + (32 * rh + 16 * i + n16) * kPPitch +
                                                  tb * 32 + g * 8) = u32x2{E::pack2(p[0], p[1]), E::pack2(p[2], p[3])};
                return ls;
            };
            float l_tile[2] = {0.f, 0.f};  // of tile t, not yet in l_part
            // scores and P of tile t
            auto scores = [&](int t) {
                if (step_to(t)) {
                    nblk = max(0, min(2, (rows_n + 15) / 16 - 2 * rh));
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int row = 32 * rh + 16 * i + n16;
                        m_own[i] = -INFINITY;
                        l_part[i] = 0.f;
                        const int from = (int)(row0 % a.rows);  // of the request
                        limit[i] = in_prefix ? len : max(0, min(len, len - a.q_len + 1 + (from + row) / a.heads));
#pragma unroll
                        for (int kk = 0; kk < 18; ++kk) {
                            qf[i][kk] = u32x4{0, 0, 0, 0};
                            if (row < rows_n)
                                qf[i][kk] = *reinterpret_cast<const u32x4 *>(a.q + (row0 + row) * kRow + 32 * kk + 8 * g);
                        }
                    }
                }
                if (nblk == 0) return;
                const CK_LDS char *tile = smem + (t & (kSlots - 1)) * kTileBytes;
                auto kfrag = [&](int kk) {
                    return *reinterpret_cast<const CK_LDS u32x4 *>(tile + (k_addr ^ ((kk & 1) << 6)) + (kk >> 1) * 128);
                };
                constexpr int kAhead = 6;
                u32x4 kf[kAhead];
                s[0] = s[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int kk = 0; kk < kAhead; ++kk) kf[kk] = kfrag(kk);
                __builtin_amdgcn_sched_barrier(0);
                if (nblk == 2) {
#pragma unroll
                    for (int kk = 0; kk < 18; ++kk) {
                        s[0] = E::mfma16(kf[kk % kAhead], qf[0][kk], s[0]);
                        s[1] = E::mfma16(kf[kk % kAhead], qf[1][kk], s[1]);
                        if (kk + kAhead < 18) kf[kk % kAhead] = kfrag(kk + kAhead);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else {
#pragma unroll
                    for (int kk = 0; kk < 18; ++kk) {  // two chains of products
                        s[kk & 1] = E::mfma16(kf[kk % kAhead], qf[0][kk], s[kk & 1]);
                        if (kk + kAhead < 18) kf[kk % kAhead] = kfrag(kk + kAhead);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    s[0] += s[1];
                }
                // lane (g, n): row n of block i, tokens 16 tb + 4 g + r
                const int tok0 = first + 16 * tb + 4 * g;
                bool moves = false;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (i >= nblk) break;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[i][r] = tok0 + r < limit[i] ? s[i][r] * a.scale_log2 : -INFINITY;
                        moves |= s[i][r] > m_own[i] + kSlack;
                    }
                    l_tile[i] = write_p(t, i);
                }
                if (__builtin_amdgcn_ballot_w64(moves) && lane == 0) flag[t & 1] = stamp + t + 1;
            };

            __syncthreads();  // tile 0 is in
            scores(0);
            __syncthreads();
            for (int t = 0; t < n; ++t) {
                if (__builtin_amdgcn_readfirstlane(flag[t & 1]) == stamp + t + 1) {  // rare: move the reference points
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float v = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
                        v = fmaxf(v, __shfl_xor(v, 16));
                        v = fmaxf(v, __shfl_xor(v, 32));
                        if (g == 0 && i < nblk) xmax[tb * kRows + 32 * rh + 16 * i + n16] = v;
                    }
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (i >= nblk) break;
                        const int row = 32 * rh + 16 * i + n16;
                        const float m_new = fmaxf(m_own[i], fmaxf(xmax[row], xmax[kRows + row]));
                        const float f = m_new == -INFINITY ? 1.f : exp2_fast(m_own[i] - m_new);
                        m_own[i] = m_new;
                        l_part[i] *= f;
                        l_tile[i] = write_p(t, i);
                        if (tb == 0 && g == 0) fac[row] = f;
                    }
                    __syncthreads();
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) l_part[i] += l_tile[i];
                if (ends) {
                    CK_LDS float *sums = (CK_LDS float *)(smem + kLdsSum) + parity * 3 * kRows;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float v = l_part[i] + __shfl_xor(l_part[i], 16);
                        v += __shfl_xor(v, 32);
                        const int row = 32 * rh + 16 * i + n16;
                        if (g == 0 && i < nblk) {
                            sums[tb * kRows + row] = v;
                            if (tb == 0) sums[2 * kRows + row] = m_own[i];
                        }
                    }
                    parity ^= 1;
                    item = -1;
                }
                if (t + 1 < n) scores(t + 1);
                __syncthreads();
            }
        } else {
            auto issue = [&](int t) {
                const int page = __builtin_amdgcn_readfirstlane(desc[4 * t]);
                const int from = __builtin_amdgcn_readfirstlane(desc[4 * t + 2]);
                const ck_rsrc_t r = buf_rsrc(
                    cache + (int64_t)max(page, 0) * kPageBytes + ((from / kTok) % kTilesPerPage) * kTileBytes, kTileBytes);
                CK_LDS char *dst = smem + (t & (kSlots - 1)) * kTileBytes + cw * 1024;
#pragma unroll
                for (int j = 0; j < 9; ++j) dma16_buf(r, dma_off[j], 0, dst + j * 4096);
            };
            // This wave's pieces of tile t are in (`younger` tiles behind it may not be); rows
            // past the length or of an invalid page become zeros: 0 * V must not be NaN,
            // and an invalid page reads as zeros.
            auto settle = [&](int t, int younger) {
                if (younger <= 0) wait_vmcnt<0>();
                else if (younger == 1) wait_vmcnt<9>();
                else if (younger == 2) wait_vmcnt<18>();
                else wait_vmcnt<27>();
                const int page = __builtin_amdgcn_readfirstlane(desc[4 * t]);
                const int z0 = page < 0 ? 0 : __builtin_amdgcn_readfirstlane(desc[4 * t + 3] - desc[4 * t + 2]);
                if (z0 < kTok) {
                    CK_LDS char *dst = smem + (t & (kSlots - 1)) * kTileBytes + cw * 1024 + lane * 16;
#pragma unroll
                    for (int j = 0; j < 9; ++j)
                        if (dma_row[j] >= z0) *reinterpret_cast<CK_LDS u32x4 *>(dst + j * 4096) = u32x4{0, 0, 0, 0};
                }
            };
            bool pending = false;  // the segment before tile t's is to be closed
            // O of the closed segment: to its place in the workspace, or to the result
            auto close = [&]() {
                const CK_LDS float *sums = (const CK_LDS float *)(smem + kLdsSum) + parity * 3 * kRows;
                const bool part = in_prefix || a.merge || began_before || goes_on;
                float *po = nullptr, *pl = nullptr;
                if (in_prefix) {
                    po = a.ppart_o + (sp * (int64_t)a.prows + row0) * kR;
                    pl = a.ppart_lse + sp * (int64_t)a.prows + row0;
                } else if (part) {
                    const int64_t slot = began_before || goes_on ? part_slot(began_before, w.chunk, a.teams, w.team)
                                                                 : (int64_t)2 * a.chunks * a.teams + item;
                    po = a.part_o + slot * a.slot_rows * kR;
                    pl = a.part_lse + slot * a.slot_rows;
                }
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    const int row = 16 * i + n16;
                    if (row >= rows_n) continue;
                    // l is 0 where no token was seen (or every score was -inf)
                    const float l = sums[row] + sums[kRows + row];
                    const float inv = l == 0.f ? 0.f : 1.0f / l;
                    const float lse2 = l == 0.f ? -INFINITY : sums[2 * kRows + row] - E::kBias + log2f(l);
                    if (part) {
#pragma unroll
                        for (int d = 0; d < 8; ++d)
                            *reinterpret_cast<f32x4 *>(po + (int64_t)row * kR + 128 * cw + 16 * d + 4 * g) = oacc[d][i] * inv;
                        if (cw == 0 && g == 0) pl[row] = lse2;
                    } else {
#pragma unroll
                        for (int d = 0; d < 8; ++d) {
                            const f32x4 o = oacc[d][i] * inv;
                            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + (row0 + row) * kR + 128 * cw +
                                                       16 * d + 4 * g) = make_uint2(E::pack2(o[0], o[1]), E::pack2(o[2], o[3]));
                        }
                        if (cw == 0 && g == 0) a.lse[row0 + row] = lse2 * kLn2;
                    }
                }
                parity ^= 1;
                item = -1;
            };
            // O^T += C^T P^T of tile t
            auto add = [&](int t) {
                const CK_LDS char *tile = smem + (t & (kSlots - 1)) * kTileBytes;
                const CK_LDS char *pbuf = smem + kLdsP + (t & 1) * kPBytes;
                u32x4 pf[NB];
#pragma unroll
                for (int i = 0; i < NB; ++i)
                    pf[i] = *reinterpret_cast<const CK_LDS u32x4 *>(pbuf + (16 * i + n16) * kPPitch + g * 16);
                auto vfrag = [&](int d) {
                    const uint2 v0 = lds_read_tr16(tile + (v_addr[0] ^ ((d & 3) << 5)) + (d >> 2) * 128);
                    const uint2 v1 = lds_read_tr16(tile + (v_addr[1] ^ ((d & 3) << 5)) + (d >> 2) * 128);
                    return u32x4{v0.x, v0.y, v1.x, v1.y};
                };
                constexpr int kAhead = 4;
                u32x4 vf[kAhead];
#pragma unroll
                for (int d = 0; d < kAhead; ++d) vf[d] = vfrag(d);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int d = 0; d < 8; ++d) {
#pragma unroll
                    for (int i = 0; i < NB; ++i) oacc[d][i] = E::mfma16(vf[d % kAhead], pf[i], oacc[d][i]);
                    if (d + kAhead < 8) vf[d % kAhead] = vfrag(d + kAhead);
                    __builtin_amdgcn_sched_barrier(0);
                }
            };

            for (int t = 0; t < kSlots && t < n; ++t) issue(t);
            settle(0, min(n - 1, 3));
            __syncthreads();  // tile 0 is in
            if (n > 1) settle(1, min(n - 2, 2));
            __syncthreads();
            for (int t = 0; t < n; ++t) {
                if (t > 0 && t + 3 < n) issue(t + 3);
                bool settled = t + 2 >= n;
                if (pending) {
                    // the tile's wait in front of the stores, which are counted with it
                    if (!settled) settle(t + 2, min(n - 3 - t, 1));
                    settled = true;
                    close();
                    pending = false;
                }
                if (step_to(t)) {
                    nblk = (rows_n + 15) / 16;
#pragma unroll
                    for (int d = 0; d < 8; ++d)
#pragma unroll
                        for (int i = 0; i < NB; ++i) oacc[d][i] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
                if (__builtin_amdgcn_readfirstlane(flag[t & 1]) == stamp + t + 1) {
                    __syncthreads();
                    __syncthreads();  // the factors are in
#pragma unroll
                    for (int i = 0; i < NB; ++i) {
                        const float f = i < nblk ? fac[16 * i + n16] : 1.f;
#pragma unroll
                        for (int d = 0; d < 8; ++d) oacc[d][i] *= f;
                    }
                }
                add(t);
                if (!settled) settle(t + 2, min(n - 3 - t, 1));
                pending = ends;
                __syncthreads();
            }
            if (pending) close();
        }
        stamp += n;
    }
}

// NB: 16-row blocks of the largest row tile
template <int DT, int NB>
__global__ __launch_bounds__(kThreads) void latent_decode_kernel(DecodeArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem_raw[];
    CK_LDS char *smem = (CK_LDS char *)smem_raw;
    CK_LDS int *scan = (CK_LDS int *)(smem + kLdsScan);
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    Share w;
    const uint32_t lw = xcd_remap(blockIdx.x, gridDim.x);
    w.team = lw % a.teams;
    w.wg = lw / a.teams;

    // ---- the list: this thread's requests, their first tile, the total --------------------
    const int per = (a.batch + kThreads - 1) / kThreads;
    w.b_lo = min(tid * per, a.batch);
    w.b_hi = min(w.b_lo + per, a.batch);
    auto tiles_of = [&](int b) { return (int)((clamp_len(a.lens[b], a) + kTok - 1) / kTok) * a.listed; };
    int mine = 0;
    for (int b = w.b_lo; b < w.b_hi; ++b) mine += tiles_of(b);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(incl, o);
        if (lane >= o) incl += up;
    }
    if (lane == 63) scan[wave] = incl;
    if (tid < 2) ((CK_LDS int *)(smem + kLdsFlag))[tid] = 0;
    __syncthreads();
    int start = incl - mine, total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        if (i < wave) start += scan[i];
        total += scan[i];
    }
    w.my_start = start;
    if (w.wg == 0 && w.team == 0) {
        for (int b = w.b_lo; b < w.b_hi; ++b) {
            a.sums[b] = start;
            start += tiles_of(b);
        }
        if (tid == 0) a.sums[a.batch] = total;
    }

    // ---- this workgroup's share ------------------------------------------------------------
    w.ptiles = w.unit_tiles = 0;
    w.units = 0;
    if (a.merge) {
        w.ptiles = prefix_tiles(a);
        w.unit_tiles = (w.ptiles + a.psplits - 1) / a.psplits;
        w.units = w.ptiles > 0 ? a.pmtiles * a.psplits : 0;
    }
    const ListMap map = list_map(total, a.chunks, a.min_tiles, w.units, w.unit_tiles);
    w.chunk = w.wg < map.ra ? w.wg : w.wg - map.ra + map.na;
    const bool has_list = w.wg < map.ra ? w.wg < map.na : w.wg - map.ra < map.nb;
    w.lo = has_list ? list_lo(map, w.chunk) : 0;
    w.hi = has_list ? list_lo(map, w.chunk + 1) : 0;

    if (wave < kProducers) role_loop<DT, NB, true>(a, w, smem);
    else role_loop<DT, NB, false>(a, w, smem);
}

// Folds the parts of every row that has some, in list order and after the prefix's, and
// writes rows that see nothing. 128 threads a row, 4 dims each; parts are loaded kBatch at a
// time, independent of each other.
template <int DT>
__global__ __launch_bounds__(256) void latent_combine_kernel(DecodeArgs a) {
    using E = Elem<DT>;
    constexpr int kBatch = 8;
    const int64_t r = (int64_t)blockIdx.x * 2 + (threadIdx.x >> 7);
    const int d4 = 4 * (threadIdx.x & 127);
    if (r >= (int64_t)a.batch * a.rows) return;
    const int b = (int)(r / a.rows), rr = (int)(r - (int64_t)b * a.rows);
    const int mt = rr / kRows, row = rr - mt * kRows;
    const int team = a.teams > 1 ? mt : 0, m = a.teams > 1 ? 0 : mt;
    const int64_t all = a.sums[b + 1] - a.sums[b], each = all / a.listed, s0 = a.sums[b] + m * each;

    int psplits = 0, units = 0;
    int64_t unit_tiles = 0;
    if (a.merge) {
        const int64_t ptiles = prefix_tiles(a);
        unit_tiles = (ptiles + a.psplits - 1) / a.psplits;
        if (ptiles > 0) {
            units = a.pmtiles * a.psplits;
            psplits = (int)((ptiles + unit_tiles - 1) / unit_tiles);
        }
    }
    int c0 = 0, parts = 0;
    bool whole = false;
    if (each > 0) {
        const ListMap map = list_map(a.sums[a.batch], a.chunks, a.min_tiles, units, unit_tiles);
        c0 = list_chunk(map, s0);
        parts = list_chunk(map, s0 + each - 1) - c0 + 1;
        whole = parts == 1;
        if (whole && !a.merge) return;  // written by its workgroup
    }
    const int total = psplits + parts;
    float mx = -INFINITY, sum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < total; p0 += kBatch) {
        float ls[kBatch];
        f32x4 o[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int p = min(p0 + j, total - 1);  // past the last part: it again, at weight 0
            const float *po, *pl;
            if (p < psplits) {
                pl = a.ppart_lse + (int64_t)p * a.prows + r;
                po = a.ppart_o + ((int64_t)p * a.prows + r) * kR;
            } else {
                const int c = c0 + p - psplits;
                const int64_t slot = whole ? (int64_t)2 * a.chunks * a.teams + b * a.listed + m
                                           : part_slot(c > c0, c, a.teams, team);
                pl = a.part_lse + slot * a.slot_rows + row;
                po = a.part_o + (slot * a.slot_rows + row) * kR;
            }
            ls[j] = p0 + j < total ? *pl : -INFINITY;
            o[j] = *reinterpret_cast<const f32x4 *>(po + d4);
        }
        float mb = mx;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) mb = fmaxf(mb, ls[j]);
        const float mu = mb == -INFINITY ? 0.f : mb;
        const float f = exp2_fast(mx - mu);
        acc *= f;
        sum *= f;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            // a part that saw nothing holds zeros
            const float w = exp2_fast(ls[j] - mu);
            if (p0 + j < total) acc += o[j] * w;
            sum += w;
        }
        mx = mb;
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    acc *= inv;
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + r * kR + d4) =
        make_uint2(E::pack2(acc[0], acc[1]), E::pack2(acc[2], acc[3]));
    if (d4 == 0) a.lse[r] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
}

int64_t ceil_div(int64_t x, int64_t y) { return (x + y - 1) / y; }
int64_t pad256(int64_t n) { return (n + 255) & ~(int64_t)255; }

// Sizes of a call: the list's and the prefix's partition, and the workspace.
struct LatentPlan {
    int64_t rows, mtiles, teams, listed, chunks, slot_rows, slots;
    int64_t prows, pmtiles, psplits;
    int64_t off_lse, off_o, off_plse, off_po, ws_bytes;
};

int make_plan(int64_t batch, int64_t q_len, int64_t heads, int64_t kv_cap, bool merge, int64_t prefix_cap,
              LatentPlan *p) {
    if (batch < 0 || q_len < 1 || heads < 1 || kv_cap < 0 || prefix_cap < 0) return CK_E_INVALID_ARG;
    if (batch > (1 << 24) || q_len > (1 << 24) || heads > (1 << 16) || kv_cap > ((int64_t)1 << 30) ||
        prefix_cap > ((int64_t)1 << 30) || batch * q_len > ((int64_t)1 << 31) / heads)
        return CK_E_INVALID_ARG;
    p->rows = q_len * heads;
    p->mtiles = ceil_div(p->rows, kRows);
    p->teams = merge ? 1 : p->mtiles;
    p->listed = merge ? p->mtiles : 1;
    p->chunks = p->teams >= kGroups ? 1 : kGroups / p->teams;
    // the list's places and the sums are 32-bit
    if (batch * p->listed * ceil_div(kv_cap, kTok) >= (int64_t)1 << 31) return CK_E_INVALID_ARG;
    p->slot_rows = p->rows < kRows ? p->rows : kRows;
    p->slots = 2 * p->chunks * p->teams + (merge ? batch * p->listed : 0);
    p->prows = merge ? batch * heads : 0;
    p->pmtiles = ceil_div(p->prows, kRows);
    p->psplits = 0;
    if (merge && p->pmtiles > 0) {
        p->psplits = p->pmtiles >= kGroups ? 1 : kGroups / p->pmtiles;
        const int64_t most = ceil_div(prefix_cap, 4 * kTok);
        if (p->psplits > most) p->psplits = most < 1 ? 1 : most;
    }
    int64_t at = pad256((batch + 1) * 4);
    p->off_lse = at;
    at += pad256(p->slots * p->slot_rows * 4);
    p->off_plse = at;
    at += pad256(p->psplits * p->prows * 4);
    p->off_o = at;
    at += p->slots * p->slot_rows * kR * 4;
    p->off_po = at;
    at += p->psplits * p->prows * kR * 4;
    p->ws_bytes = at;
    return CK_OK;
}

template <int DT, int NB>
int launch_decode(const DecodeArgs &a, hipStream_t s) {
    static std::atomic<uint64_t> lds_set{0};
    int rc = ensure_dynamic_lds(reinterpret_cast<const void *>(&latent_decode_kernel<DT, NB>), kLds, lds_set);
    if (rc != CK_OK) return rc;
    hipLaunchKernelGGL((latent_decode_kernel<DT, NB>), dim3((unsigned)(a.teams * a.chunks)), dim3(kThreads), kLds, s, a);
    CK_RETURN_LAUNCH();
}

template <int DT>
int launch(const DecodeArgs &a, hipStream_t s) {
    const int rows = a.merge ? kRows : a.rows;  // of the largest row tile
    int rc = rows <= 16 ? launch_decode<DT, 1>(a, s) : rows <= 32 ? launch_decode<DT, 2>(a, s) : launch_decode<DT, 4>(a, s);
    if (rc != CK_OK) return rc;
    hipLaunchKernelGGL((latent_combine_kernel<DT>), dim3((unsigned)ceil_div((int64_t)a.batch * a.rows, 2)), dim3(256), 0,
                       s, a);
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
        int64_t kv_cap, const PrefixArgs *prefix, int64_t prefix_cap, void *out, float *lse, void *workspace,
        int64_t workspace_bytes, hipStream_t s) {
    LatentPlan p;
    int rc = make_plan(batch, q_len, heads, kv_cap, prefix != nullptr, prefix_cap, &p);
    if (rc != CK_OK) return rc;
    if (block_size != kPage || (dtype != CK_DTYPE_BF16 && dtype != CK_DTYPE_F16)) return CK_E_UNSUPPORTED;
    if (bt_cols < 0 || num_blocks < 0 || num_blocks > ((int64_t)1 << 31) || kv_cap != bt_cols * kPage)
        return CK_E_INVALID_ARG;
    if (prefix && (prefix->cols < 0 || prefix->num_blocks < 0 || prefix->num_blocks > ((int64_t)1 << 31) ||
                   prefix_cap != prefix->cols * kPage))
        return CK_E_INVALID_ARG;
    if (!(scale > 0.f) || !std::isfinite(scale)) return CK_E_INVALID_ARG;
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
    a.min_tiles = 4;
    a.scale_log2 = scale * kLog2e;
    a.out = out;
    a.lse = lse;
    a.sums = reinterpret_cast<int32_t *>(ws);
    a.part_lse = reinterpret_cast<float *>(ws + p.off_lse);
    a.part_o = reinterpret_cast<float *>(ws + p.off_o);
    a.slot_rows = (int)p.slot_rows;
    a.merge = prefix != nullptr;
    if (prefix) {
        a.pcache = static_cast<const uint16_t *>(prefix->cache);
        a.pbt = prefix->bt;
        a.plen = prefix->len;
        a.pcols = prefix->cols;
        a.pblocks = prefix->num_blocks;
        a.prows = (int)p.prows;
        a.pmtiles = (int)p.pmtiles;
        a.psplits = (int)p.psplits;
        a.ppart_lse = reinterpret_cast<float *>(ws + p.off_plse);
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
               scale, bt_cols * kPage, nullptr, 0, out, lse, workspace, workspace_bytes,
               reinterpret_cast<hipStream_t>(stream));
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
               suffix_num_blocks, block_size, dtype, scale, suffix_bt_cols * kPage, &prefix, prefix_bt_cols * kPage, out,
               lse, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}
