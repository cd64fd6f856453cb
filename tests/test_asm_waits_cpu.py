"""Waits around hand-written instructions (asm_waits.py): what it finds in planted listings, and on
the assembly of the kernels as they are built."""
import os

import pytest

import asm_waits
import build


def _pairs(text):
    return [(f.op, t.op, kept, need) for _, f, t, _, kept, need in
            asm_waits.missing_waits(("kernel:\n" + text.replace("[[", ";#ASMSTART\n").replace("]]", "\n;#ASMEND")).splitlines())]


PRODUCT = "v_mfma_f32_32x32x16_bf16 v[2:17], v[38:41], v[158:161], v[2:17]\n"
OTHER = "v_mfma_f32_32x32x16_bf16 v[18:33], v[42:45], v[158:161], v[18:33]\n"
READ = "[[v_max3_f32 v37, v2, v3, v50]]\n"


def test_a_read_right_behind_a_product():
    # what two kernels once held: an inline v_max3_f32, one product and nothing else between
    got = _pairs(PRODUCT + OTHER + READ)
    assert got == [("v_mfma_f32_32x32x16_bf16", "v_max3_f32", 1, 12)] * 2  # v2 and v3
    assert _pairs(PRODUCT + "s_nop 10\n" + READ) == [("v_mfma_f32_32x32x16_bf16", "v_max3_f32", 11, 12)] * 2
    assert _pairs(PRODUCT + "s_nop 11\n" + READ) == []
    assert _pairs(PRODUCT + OTHER + "v_max3_f32 v37, v2, v3, v50\n") == []  # the compiler's own
    assert _pairs(PRODUCT + "v_mov_b32_e32 v2, 0\nv_mov_b32_e32 v3, 0\n" + READ) == []  # another value by then


def test_smaller_products_accumulation_registers_and_overwriting():
    small = "[[v_mfma_f32_16x16x32_f16 a[8:11], v[38:41], v[158:161], a[8:11]]]\n"
    assert _pairs(small + "s_nop 6\n[[v_accvgpr_read_b32 v1, a9]]\n") == [("v_mfma_f32_16x16x32_f16", "v_accvgpr_read_b32", 7, 8)]
    assert _pairs(small + "s_nop 7\n[[global_store_dwordx4 v0, a[8:11], s[2:3] offset:16]]\n") == []
    assert len(_pairs(small + "[[global_store_dwordx4 v0, a[8:11], s[2:3] offset:16]]\n")) == 4
    assert len(_pairs(small + "[[v_accvgpr_write_b32 a10, v1]]\n")) == 1
    assert _pairs(small + small) == []  # a sum that goes on
    with pytest.raises(ValueError, match="no known distance"):
        _pairs("v_mfma_f64_4x4x4_4b_f64 v[0:1], v[2:3], v[4:5], v[0:1]\n")


def test_operands_of_hand_written_products_and_loads():
    product = "[[v_mfma_f32_16x16x32_f16 a[8:11], v[38:41], v[158:161], a[8:11]]]\n"
    assert _pairs("v_cvt_pk_bf16_f32 v40, v1, v2\ns_nop 0\n" + product) == [("v_cvt_pk_bf16_f32", "v_mfma_f32_16x16x32_f16", 1, 2)]
    assert _pairs("v_cvt_pk_bf16_f32 v40, v1, v2\ns_nop 1\n" + product) == []
    load = "[[s_add_i32 m0, s4, 16\n\tbuffer_load_dwordx4 v1, s[8:11], s5 offen lds]]\n"
    assert ("v_readfirstlane_b32", "buffer_load_dwordx4", 1, 5) in _pairs("v_readfirstlane_b32 s10, v2\n" + load)
    assert _pairs("v_readfirstlane_b32 s10, v2\ns_nop 3\n" + load.replace("\tbuffer", "\ts_nop 0\n\tbuffer")) == []


@pytest.mark.parametrize("load", ["buffer_load_dwordx4 v1, s[8:11], s5 offen lds", "global_load_lds_dwordx4 v[2:3], off",
                                  "global_load_lds_dword v[2:3], off"])
@pytest.mark.parametrize("m0", ["s_mov_b32 m0, s4", "s_add_i32 m0, s4, 16"])
def test_loads_to_lds_behind_m0(load, m0):
    op, m0_op = load.split()[0], m0.split()[0]
    assert _pairs("[[%s\n\t%s]]\n" % (m0, load)) == [(m0_op, op, 0, 1)]
    assert _pairs("%s\n[[%s]]\n" % (m0, load)) == [(m0_op, op, 0, 1)]
    assert _pairs("[[%s\n\ts_nop 0\n\t%s]]\n" % (m0, load)) == []
    assert _pairs("[[%s\n\ts_nop 0\n\t%s]]\n" % (m0, load) * 2) == []
    assert _pairs("[[%s\n\t%s]]\n" % (m0, load.replace(" lds", "").replace("_lds", ""))) == []  # not to LDS


def test_paths_through_branches():
    # the short way round leaves too little, the long one enough; and a loop's last product before its first read
    text = PRODUCT + "s_cbranch_scc1 .LBB0_2\ns_nop 11\n.LBB0_2:\n" + READ
    assert len(_pairs(text)) == 2
    assert _pairs(PRODUCT + "s_nop 7\ns_cbranch_scc1 .LBB0_2\ns_nop 11\n.LBB0_2:\ns_nop 2\n" + READ) == []
    loop = ".LBB0_1:\n" + READ + "s_nop 11\n" + PRODUCT + "s_cbranch_scc1 .LBB0_1\ns_endpgm\n"
    assert _pairs(loop) == [("v_mfma_f32_32x32x16_bf16", "v_max3_f32", 1, 12)] * 2


@pytest.fixture(scope="module")
def listings():
    made = {}

    def of(src):
        """The build's listing of a source; made here where none is there or a source is newer."""
        path = os.path.join(build.OBJDIR, os.path.splitext(src)[0] + ".s")
        newest = max(os.path.getmtime(os.path.join(d, f)) for d in (build.CSRC, build.INCLUDE) for f in os.listdir(d))
        if src not in made and not (os.path.exists(path) and os.path.getmtime(path) > newest):
            path = build.assembly(src)
        return made.setdefault(src, path)
    return of


@pytest.mark.parametrize("src", build.CHECKED_WAITS)
def test_kernels_keep_their_waits(src, listings):
    with open(listings(src)) as f:
        text = f.read().splitlines()
    assert any(i.inline and i.op != "s_nop" for code, _ in asm_waits.parse(text).values() for i in code)
    found = ["%s | %s | %s: %d of %d" % (f.text, t.text, r, k, n) for _, f, t, r, k, n in asm_waits.missing_waits(text)]
    assert not found, found[:5]
