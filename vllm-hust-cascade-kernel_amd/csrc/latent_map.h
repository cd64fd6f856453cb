// latent_map.h - how the latent decode kernels cut their list of tiles over workgroups.
// Plain C++, so that a host program can check the same code.
#pragma once

#include "chunk_map.h"

namespace ck {
namespace lat {

// The list of W tiles cut over workgroups: part A's workgroups c < ra share the first ta
// tiles evenly, part B's the rest; a part with few tiles uses fewer workgroups, so that none
// in use is empty. Workgroups are numbered 0 .. na + nb - 1 along the list.
struct ListMap {
    int64_t w, ta;
    int ra, na, nb;
};
CK_HD int used_chunks(int64_t tiles, int groups, int min_tiles) {
    if (tiles <= 0 || groups <= 0) return 0;
    const int64_t n = (tiles + min_tiles - 1) / min_tiles;
    return n < groups ? (int)n : groups;
}
// The prefix's units (`units` of up to `unit_tiles` tiles, dealt round-robin over `groups`
// workgroups) come first: the first units % groups workgroups have one more. The list
// fills the others up to their level, and what remains goes evenly to all.
CK_HD ListMap list_map(int64_t w, int groups, int min_tiles, int units, int64_t unit_tiles) {
    ListMap m;
    m.w = w;
    m.ra = units % groups;
    const int64_t over = m.ra > 0 ? w - (int64_t)(groups - m.ra) * unit_tiles : 0;
    m.ta = over > 0 ? div_nonneg(over * m.ra, groups) : 0;
    m.na = used_chunks(m.ta, m.ra, min_tiles);
    m.nb = used_chunks(w - m.ta, groups - m.ra, min_tiles);
    return m;
}
// First tile of numbered chunk n (n = na + nb: w).
CK_HD int64_t list_lo(const ListMap &m, int n) {
    if (n < m.na) return div_nonneg((int64_t)n * m.ta, m.na);
    if (n >= m.na + m.nb) return m.w;
    return m.ta + div_nonneg((int64_t)(n - m.na) * (m.w - m.ta), m.nb);
}
// The numbered chunk that holds tile x, 0 <= x < w: the largest n with list_lo(n) <= x.
CK_HD int list_chunk(const ListMap &m, int64_t x) {
    if (x < m.ta) return (int)div_nonneg((x + 1) * m.na - 1, m.ta);
    return m.na + (int)div_nonneg((x - m.ta + 1) * m.nb - 1, m.w - m.ta);
}
// A part's place in the workspace: the chunk's first when the item began in an earlier
// chunk, its second when it began here and goes on; a whole item has one of its own.
CK_HD int64_t part_slot(bool began_before, int n, int teams, int team) {
    return ((int64_t)2 * n + (began_before ? 0 : 1)) * teams + team;
}

}  // namespace lat
}  // namespace ck
