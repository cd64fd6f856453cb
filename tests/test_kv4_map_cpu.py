"""How the list of a 4-bit decode of more than 32 rows a kv head is cut (csrc/kv4_map.h), by the rule that the kernel takes."""
import ctypes
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-hust-cascade-kernel_amd", "csrc")


@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv4_rule")
    src = d / "rule.cpp"
    src.write_text("""#include "kv4_map.h"
using namespace ck::kv4;
extern "C" int shares(int batch, int units, int kv_heads, int groups, int *lo) {
    const int pieces = batch == 1 ? groups / kv_heads : 0;
    const Shares s = list_shares(units * kv_heads, groups, list_least(batch), units, pieces);
    for (int k = 0; k <= s.count; ++k) lo[k] = share_lo(s, k);
    return s.count;
}
""")
    lib = d / "rule.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I", CSRC, str(src), "-o", str(lib)], check=True)
    lib = ctypes.CDLL(str(lib))

    def shares(batch, units, kv_heads, groups):
        lo = (ctypes.c_int * (groups + 1))()
        n = lib.shares(batch, units, kv_heads, groups, lo)
        return list(lo)[:n + 1]
    return shares


@pytest.mark.parametrize("groups", [1, 85, 256])
@pytest.mark.parametrize("kv_heads", [1, 8])
@pytest.mark.parametrize("batch,units", [(2, 2), (4, 20), (16, 16), (16, 40), (64, 64), (64, 512)])
def test_several_requests_leave_no_workgroup_idle(cut, batch, units, kv_heads, groups):
    """Short requests are not put one behind another into a share while there are workgroups for them."""
    lo = cut(batch, units, kv_heads, groups)
    assert len(lo) - 1 == min(units * kv_heads, groups)
    assert lo[0] == 0 and lo[-1] == units * kv_heads and max(b - a for a, b in zip(lo, lo[1:])) == -(-units * kv_heads // (len(lo) - 1))


@pytest.mark.parametrize("units", [1, 5, 32, 251, 5000])
def test_one_request_is_cut_to_about_four_units(cut, units):
    """ceil(units / 4) shares a kv head at most, as even as can be."""
    lo = cut(1, units, 8, 256)
    sizes = [b - a for a, b in zip(lo, lo[1:])]
    assert sum(sizes) == 8 * units and max(sizes) - min(sizes) <= 1
    assert len(sizes) <= 8 * -(-units // 4) and (units < 4 or min(sizes) >= 2)
