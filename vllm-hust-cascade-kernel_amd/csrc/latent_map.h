// latent_map.h - how the latent decode kernels cut their list of tiles over workgroups.
// Plain C++, so that a host program can check the same code.
#pragma once

#include "chunk_map.h"

namespace ck {
namespace lat {

// An item (a request's row tile) takes its tiles' places on the list and kItemPlaces before
// them, empty: about what opening and closing it costs, so that chunks of many short items
// hold fewer tiles. Measured with 128 rows, in cycles: a tile 3450, an item 7000 to 15000. 3 places
// against none, with what else changed beside them: 19 x 2 x 64 heads over 92 tokens 31 / 58 us.
constexpr int kItemPlaces = 3;

// n places cut evenly into `chunks` <= n: the first `rem` have q + 1.
struct Cut {
    int chunks, q, rem;
};
CK_HD Cut cut_evenly(int n, int chunks) {
    Cut c;
    c.chunks = chunks;
    c.q = chunks > 0 ? n / chunks : 0;
    c.rem = n - c.q * chunks;
    return c;
}
CK_HD int cut_lo(const Cut &c, int k) { return k * c.q + (k < c.rem ? k : c.rem); }
CK_HD int cut_chunk(const Cut &c, int x) {  // the chunk that holds place x
    const int big = c.rem * (c.q + 1);
    return x < big ? x / (c.q + 1) : c.rem + (x - big) / c.q;
}

// The list's w places cut over workgroups: part A's workgroups c < ra share the first ta
// places evenly, part B's the rest; a part with few places uses fewer workgroups, so that none
// in use is empty. Workgroups are numbered 0 .. a.chunks + b.chunks - 1 along the list.
struct ListMap {
    int w, ta, ra;
    Cut a, b;
};
CK_HD int used_chunks(int places, int groups, int min_places) {
    if (places <= 0 || groups <= 0) return 0;
    const int n = (places - 1) / min_places + 1;
    return n < groups ? n : groups;
}
// The prefix's units (`units` of up to `unit_places`, dealt round-robin over `groups`
// workgroups) come first: the first units % groups workgroups have one more. The list
// fills the others up to their level, and what remains goes evenly to all.
CK_HD ListMap list_map(int w, int groups, int min_places, int units, int unit_places) {
    ListMap m;
    m.w = w;
    m.ra = units % groups;
    const int64_t level = (int64_t)(groups - m.ra) * unit_places;
    m.ta = 0;
    if (m.ra > 0 && w > level) {
        const int over = (int)(w - level), q = over / groups;
        m.ta = q * m.ra + (over - q * groups) * m.ra / groups;
    }
    m.a = cut_evenly(m.ta, used_chunks(m.ta, m.ra, min_places));
    m.b = cut_evenly(w - m.ta, used_chunks(w - m.ta, groups - m.ra, min_places));
    return m;
}
CK_HD int list_used(const ListMap &m) { return m.a.chunks + m.b.chunks; }
// First place of numbered chunk n (n = list_used: w).
CK_HD int list_lo(const ListMap &m, int n) {
    if (n < m.a.chunks) return cut_lo(m.a, n);
    return m.ta + cut_lo(m.b, n - m.a.chunks);
}
// The numbered chunk that holds place x, 0 <= x < w.
CK_HD int list_chunk(const ListMap &m, int x) {
    return x < m.ta ? cut_chunk(m.a, x) : m.a.chunks + cut_chunk(m.b, x - m.ta);
}
// A part's place in the workspace: the chunk's first when the item began in an earlier
// chunk, its second when it began here and goes on; a whole item has one of its own.
CK_HD int64_t part_slot(bool began_before, int n, int teams, int team) {
    return ((int64_t)2 * n + (began_before ? 0 : 1)) * teams + team;
}

// How often the prefix's tiles are split, for `row_tiles` row tiles beside a list of w places.
// A split more shortens the units, but adds a part to fold for each row. Tried are one, what
// fills the prefix's share of one round of the workgroups (the list takes the others), one round
// and two, and taken is the one after which the last workgroup ends first, the first of equals.
constexpr int kSplitChoices = 4;
struct Split {
    int splits;
    float end;
};
CK_HD Split split_choice(int i, int row_tiles, int tiles, int w, int groups, int most) {
    const float work = (float)row_tiles * (float)tiles;
    const float room = i == 0 ? 0.f : i == 1 ? (float)groups * work / (work + (float)w) : (float)((i - 1) * groups);
    int s = (int)(room / (float)row_tiles);
    s = s < 1 ? 1 : s > most ? most : s;
    const int units = row_tiles * s, each = (tiles + s - 1) / s + kItemPlaces;
    const float rounds = (float)((units + groups - 1) / groups) * (float)each;
    const float left = rounds * (float)groups - (float)units * (float)each;
    // a list that the others do not hold is cut over all of them once more
    return Split{s, (float)w <= left ? rounds : rounds + ((float)w - left) / (float)groups + (float)kItemPlaces};
}
CK_HD bool better(const Split &x, const Split &than) { return x.end < than.end; }

}  // namespace lat
}  // namespace ck
