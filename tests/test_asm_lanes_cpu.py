"""Vector instructions before switched-off lanes are back (asm_lanes.py): planted listings, and the kernels as they are
built."""
import pytest

import asm_lanes
import build
from tests.test_asm_waits_cpu import listings  # noqa: F401

OFF = "s_and_saveexec_b64 s[18:19], vcc\ns_cbranch_execz .LBB0_2\nv_mov_b32_e32 v95, v75\ns_and_b64 exec, exec, s[2:3]\n" \
      "s_cbranch_execz .LBB0_1\nglobal_store_dword v[34:35], v36, off\n.LBB0_1:\n"
ON = ".LBB0_2:\ns_or_b64 exec, exec, s[18:19]\nv_mov_b32_e32 v34, v170\ns_endpgm\n"


def _found(text):
    return [(o.op, c.text) for _, o, c in asm_lanes.lost_lanes(("kernel:\n" + text).splitlines())]


def test_copies_before_the_lanes_are_back():
    # what a kernel once had: registers given back to the lanes of the inner condition only
    assert _found(OFF + "v_mov_b32_e32 v85, v94\nscratch_load_dword v75, off, off\n" + ON) == [
        ("s_and_b64", "v_mov_b32_e32 v85, v94"), ("s_and_b64", "scratch_load_dword v75, off, off")]
    assert _found(OFF + ON) == []
    assert _found(OFF + "s_mov_b32 s4, 0\n" + ON) == []


def test_conditions_with_an_end_of_their_own():
    own = OFF.replace("s_and_b64 exec, exec, s[2:3]", "s_and_saveexec_b64 s[4:5], s[2:3]") + "s_or_b64 exec, exec, s[4:5]\n"
    assert _found(own + "v_mov_b32_e32 v85, v94\n" + ON) == []
    assert _found("s_and_b64 exec, exec, s[2:3]\ns_cbranch_execz .LBB0_9\nv_mov_b32_e32 v1, v2\n.LBB0_9:\ns_endpgm\n") == []


@pytest.mark.parametrize("src", build.CHECKED_WAITS)
def test_kernels_lose_no_lanes(src, listings):  # noqa: F811
    with open(listings(src)) as f:
        found = asm_lanes.lost_lanes(f)
    assert not found, found[:3]
