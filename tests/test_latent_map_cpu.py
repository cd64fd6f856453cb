"""How the latent decode kernels cut their list over workgroups (csrc/latent_map.h),
compiled for the host: every tile has one owner, no workgroup in use is empty, and what the
fold computes from an item's places (its first chunk and their number) is what the
workgroups hold."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-hust-cascade-kernel_amd", "csrc")
LEAST = 2


@pytest.fixture(scope="module")
def header(tmp_path_factory):
    d = tmp_path_factory.mktemp("latent_map")
    src = d / "latent_map.cpp"
    src.write_text("""#include "latent_map.h"
using namespace ck::lat;
extern "C" int places() { return kItemPlaces; }
extern "C" int bounds(int w, int groups, int least, int units, int unit, int *lo, int *wg) {
    const ListMap m = list_map(w, groups, least, units, unit);
    const int n = list_used(m);
    for (int i = 0; i <= n; ++i) lo[i] = list_lo(m, i);
    for (int g = 0; g < groups; ++g)
        wg[g] = g < m.ra ? (g < m.a.chunks ? g : -1) : (g - m.ra < m.b.chunks ? g - m.ra + m.a.chunks : -1);
    return n;
}
extern "C" void owner(int w, int groups, int least, int units, int unit, const int *x, int n, int *out) {
    const ListMap m = list_map(w, groups, least, units, unit);
    for (int i = 0; i < n; ++i) out[i] = list_chunk(m, x[i]);
}
extern "C" int splits(int row_tiles, int tiles, int w, int groups, int most) {
    Split best = split_choice(0, row_tiles, tiles, w, groups, most);
    for (int i = 1; i < kSplitChoices; ++i) {
        const Split x = split_choice(i, row_tiles, tiles, w, groups, most);
        if (better(x, best)) best = x;
    }
    return best.splits;
}
""")
    lib = d / "latent_map.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I", CSRC, str(src), "-o", str(lib)], check=True)
    return ctypes.CDLL(str(lib))


def _int_array(n):
    return (ctypes.c_int * n)()


@pytest.mark.parametrize("groups", [1, 2, 85, 256])
@pytest.mark.parametrize("units,unit", [(0, 3), (1, 40), (17, 5), (256, 33), (300, 90)])
def test_every_place_has_one_owner(header, groups, units, unit):
    for w in sorted({0, 1, 3, 4, 5, LEAST * groups - 1, LEAST * groups, 1237, 50000, 2 ** 31 - 1}):
        lo, wg = _int_array(groups + 1), _int_array(groups)
        n = header.bounds(w, groups, LEAST, units, unit, lo, wg)
        assert 0 <= n <= groups
        if w == 0:
            assert n == 0
            continue
        lo = np.array(lo[:n + 1])
        assert lo[0] == 0 and lo[-1] == w and (np.diff(lo) > 0).all()
        assert sorted(g for g in wg if g >= 0) == list(range(n))  # each chunk is one workgroup's
        x = np.unique(np.r_[lo[:-1], lo[1:] - 1, np.random.default_rng(0).integers(0, w, 500)]).astype(np.int32)
        out = np.empty_like(x)
        p = ctypes.POINTER(ctypes.c_int)
        header.owner(w, groups, LEAST, units, unit, x.ctypes.data_as(p), x.size, out.ctypes.data_as(p))
        assert (lo[out] <= x).all() and (x < lo[out + 1]).all()


def test_the_list_levels_what_the_prefix_leaves(header):
    # 16 units of 20 places on 64 workgroups, 48 free: a list within their level stays there
    wg = _int_array(64)
    n = header.bounds(48 * 20, 64, LEAST, 16, 20, _int_array(65), wg)
    assert n == 48 and all(g == -1 for g in wg[:16])
    n = header.bounds(48 * 20 + 640, 64, LEAST, 16, 20, _int_array(65), wg)
    assert n == 64


@pytest.mark.parametrize("row_tiles", [1, 3, 16, 117, 150, 300])
@pytest.mark.parametrize("tiles", [1, 2, 64, 501])
@pytest.mark.parametrize("w", [0, 40, 2200])
def test_prefix_splits_bounds(header, row_tiles, tiles, w):
    most = max(1, min(512 // row_tiles, tiles))
    s = header.splits(row_tiles, tiles, w, 256, most)
    assert 1 <= s <= most

    def end(n):  # the longest workgroup, as the header counts it
        units, each = row_tiles * n, -(-tiles // n) + header.places()
        level = -(-units // 256) * each
        left = level * 256 - units * each
        return level if w <= left else level + (w - left) / 256 + header.places()
    assert end(s) <= end(1) + 1e-3
