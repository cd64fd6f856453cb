// kv4_map.h - how the 4-bit decode kernels cut their list of units over waves. Plain C++, so that
// a host program can check the same code.
#pragma once

#include "latent_map.h"

namespace ck {
namespace kv4 {

using lat::Cut;
using lat::cut_chunk;
using lat::cut_evenly;
using lat::cut_lo;

// The list holds, request after request and within it kv head after kv head, the units (64 tokens)
// of each: n units of request b's head h from n * h + kv_heads * (units of the requests before) on.
// Its w places are cut evenly into at most `waves` shares, and at most ceil(w / least): of about `least` places and more (of 5
// places and a least of 4: 3 and 2).
// pieces > 0: the list is items of `each` places, which may be cut into so many shares each. A share that goes from one
// item into the next costs about kSpan places (a second start and joint of its parts); where shares that end with the
// items are not longer than that, they are taken. us without / with: 48 x 48 heads (6 kv heads) on 8000 tokens 42.4 / 36.3,
// 16 x 32 (8) on 6000 31.6 / 25.9, 117 x 64 on 1000 39.0 / 32.6, on 16001 105.3 / 103.1.
constexpr int kSpan = 8;
struct Shares {
    Cut cut;    // of the list, or of an item
    int each;   // an item's places, or 0
    int count;  // of all
};
// About how many places a share of a call with more than 32 rows a kv head holds at least. Of one request fewer shares leave fewer parts:
// us with 1 / 2 / 4 / 8, 16 x 32 heads on 2048 tokens 26.1 / 24.2 / 23.3 / 25.9, on 512 22.3 / 21.8 / 21.5 / 23.0, 20 x 16 (4 kv
// heads) on 4000 24.1 / 24.2 / 23.1 / 24.7, 64 x 32 on 1000 26.9 / 27.0 / 27.1 / 27.7. Of several, a share of more places is several items one after another,
// each with its start and joint: us with 1 / 2 / 4, 5 tokens of 64 heads (8 kv heads), 16 requests of 64 tokens 17.0 / 25.8 / 42.9,
// 64 of 64 26.7 / 26.8 / 44.3, 4 of 125 to 500 17.2 / 23.8 / 24.4, 64 of 4000 99.0 / 99.0 / 98.7; 4 of 500 17.6 / 17.4 / 17.0.
CK_HD int list_least(int batch) { return batch == 1 ? 4 : 1; }

CK_HD int longest(const Cut &c) { return c.q + (c.rem > 0 ? 1 : 0); }
CK_HD Shares list_shares(int w, int waves, int least, int each, int pieces) {
    const int most = w > 0 ? (w - 1) / least + 1 : 0;
    Shares s;
    s.each = 0;
    s.count = most < waves ? most : waves;
    s.cut = cut_evenly(w, s.count);
    if (pieces > 0 && each > 0) {
        const int n = (each - 1) / least + 1;
        const Cut c = cut_evenly(each, n < pieces ? n : pieces);
        if (longest(c) <= longest(s.cut) + kSpan) {
            s.each = each;
            s.count = w / each * c.chunks;
            s.cut = c;
        }
    }
    return s;
}
CK_HD int share_lo(const Shares &s, int k) {
    if (s.each == 0) return cut_lo(s.cut, k);
    const int item = k / s.cut.chunks;
    return item * s.each + cut_lo(s.cut, k - item * s.cut.chunks);
}
// The first share that holds some of places u .. u + n - 1, item h's, and how many do.
struct ShareRange {
    int first, count;
};
CK_HD ShareRange shares_of(const Shares &s, int h, int u, int n) {
    if (s.each > 0) return {h * s.cut.chunks, s.cut.chunks};
    const int first = cut_chunk(s.cut, u);
    return {first, cut_chunk(s.cut, u + n - 1) - first + 1};
}

// Where a wave leaves its part of an item (a request's kv head): the wave's first slot when the item began in
// an earlier wave's share, its second when it began here and goes on. A whole item needs none, or where parts
// are folded in any case (a prefix), one of its own behind those.
CK_HD int64_t part_slot(bool before, bool after, int wave, int waves, int item) {
    return before ? 2 * (int64_t)wave : after ? 2 * (int64_t)wave + 1 : 2 * (int64_t)waves + item;
}

}  // namespace kv4
}  // namespace ck
