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
// Its w places are cut evenly over at most `waves` waves.
CK_HD Cut list_cut(int w, int waves) { return cut_evenly(w, w < waves ? w : waves); }

// Where a wave leaves its part of an item (a request's kv head): the wave's first slot when the item began in
// an earlier wave's share, its second when it began here and goes on. A whole item needs none, or where parts
// are folded in any case (a prefix), one of its own behind those.
CK_HD int64_t part_slot(bool before, bool after, int wave, int waves, int item) {
    return before ? 2 * (int64_t)wave : after ? 2 * (int64_t)wave + 1 : 2 * (int64_t)waves + item;
}

}  // namespace kv4
}  // namespace ck
