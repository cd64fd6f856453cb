"""Host-side checks of the 4-bit cache's operators (no GPU): shapes on meta tensors, refusals of the torch ops
and of the C entry points, how a list is cut (csrc/kv4_map.h), and the oracle against what it states."""
import ctypes
import math
import os
import subprocess

import numpy as np
import pytest
import torch

import cascade_amd  # noqa: F401
from cascade_amd import abi
from oracle import kv4 as o4
from oracle.latent import close

M = "meta"
OPS = torch.ops.npu
BF, HF = torch.bfloat16, torch.float16
CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-hust-cascade-kernel_amd", "csrc")


def _e(*shape, dtype=BF):
    return torch.empty(*shape, dtype=dtype, device=M)


def _i64(*shape):
    return _e(*shape, dtype=torch.int64)


def _pool(*shape):
    return _e(*shape, dtype=torch.uint8)


def _write(**kw):
    a = dict(key=_e(5, 4, 128), value=_e(5, 4, 128), slots=_i64(5), cache=_pool(9, 4, 17408))
    a.update(kw)
    return OPS.kv4_cache_write(*a.values())


def _read(**kw):
    a = dict(cache=_pool(9, 4, 17408), slots=_i64(5), dtype=None)
    a.update(kw)
    return OPS.kv4_cache_read(*a.values())


def _decode(**kw):
    a = dict(query=_e(6, 16, 128), cache=_pool(9, 4, 17408), block_table=_e(3, 4, dtype=torch.int32), lens=_i64(3),
             scale=0.1, q_len=2)
    a.update(kw)
    return OPS.kv4_decode(*a.values())


def _cascade(**kw):
    a = dict(query=_e(3, 16, 128), pc=_pool(9, 4, 17408), pbt=_e(1, 4, dtype=torch.int32), plen=_i64(1),
             sc=_pool(2, 4, 17408), sbt=_e(3, 4, dtype=torch.int32), slens=_i64(3), scale=0.1)
    a.update(kw)
    return OPS.kv4_cascade_decode(*a.values())


def test_shapes():
    assert _write() is None
    qkv = _e(5, 24, 128)
    assert _write(key=qkv[:, 16:20], value=qkv[:, 20:]) is None
    assert _write(key=_e(0, 4, 128), value=_e(0, 4, 128), slots=_i64(0)) is None
    for dt in (BF, HF):
        k, v = _read(dtype=dt)
        assert k.shape == v.shape == (5, 4, 128) and k.dtype == v.dtype == dt
        out, lse = _decode(query=_e(6, 16, 128, dtype=dt))
        assert out.shape == (6, 16, 128) and out.dtype == dt and lse.shape == (96,) and lse.dtype == torch.float32
    assert _read()[0].dtype == BF
    out, lse = _cascade()
    assert out.shape == (3, 16, 128) and lse.shape == (48,)
    out, lse = _decode(query=_e(0, 16, 128), block_table=_e(0, 4, dtype=torch.int32), lens=_i64(0))
    assert out.shape == (0, 16, 128) and lse.shape == (0,)


@pytest.mark.parametrize("bad,msg", [
    (dict(key=_e(5, 4, 128, dtype=torch.float32)), "key must be bf16 or fp16"),
    (dict(value=_e(5, 4, 128, dtype=HF)), "value must have key's dtype"),
    (dict(key=_e(5, 4, 64)), r"must be \(T, KVH, 128\)"),
    (dict(key=_e(5, 512)), r"must be \(T, KVH, 128\)"),
    (dict(value=_e(5, 3, 128)), "cache's kv heads"),
    (dict(value=_e(4, 4, 128)), "slots' tokens"),
    (dict(key=_e(5, 4, 256)[..., ::2]), "unit stride"),
    (dict(key=_e(5, 4, 132)[..., :128]), "multiples of 8"),
    (dict(value=torch.empty_strided((5, 4, 128), (2 ** 28 + 8, 128, 1), dtype=BF, device=M)), "at most 2"),
    (dict(slots=_e(5, dtype=torch.int32)), "slots must be"),
    (dict(slots=_i64(10)[::2]), "slots must be"),
    (dict(slots=_i64(5, 1)), "slots must be"),
    (dict(cache=_pool(9, 4, 17400)), "contiguous uint8"),
    (dict(cache=_e(9, 4, 17408, dtype=torch.int8)), "contiguous uint8"),
    (dict(cache=_pool(9, 8, 17408)[:, ::2]), "contiguous uint8"),
    (dict(cache=_pool(9, 0, 17408)), "must have kv heads"),
    (dict(slots=torch.empty(5, dtype=torch.int64)), "same HIP device"),
])
def test_write_refusals(bad, msg):
    with pytest.raises(RuntimeError, match="kv4_cache_write: .*" + msg):
        _write(**bad)


@pytest.mark.parametrize("bad,msg", [
    (dict(dtype=torch.float32), "dtype must be bf16 or fp16"),
    (dict(cache=_pool(9, 17408)), "contiguous uint8"),
    (dict(slots=_e(5, dtype=torch.int32)), "slots must be"),
    (dict(slots=torch.empty(5, dtype=torch.int64)), "same HIP device"),
])
def test_read_refusals(bad, msg):
    with pytest.raises(RuntimeError, match="kv4_cache_read: .*" + msg):
        _read(**bad)


@pytest.mark.parametrize("bad,msg", [
    (dict(query=_e(6, 16, 64)), r"query must be a contiguous \(T, H, 128\)"),
    (dict(query=_e(16, 6, 128).transpose(0, 1)), "query must be a contiguous"),
    (dict(query=_e(6, 0, 128)), "query must have heads"),
    (dict(query=_e(6, 18, 128)), "multiple of the cache's kv heads"),
    (dict(query=_e(6, 2, 128)), "multiple of the cache's kv heads"),
    (dict(query=_e(6, 16, 128, dtype=torch.float32)), "query must be bf16 or fp16"),
    (dict(q_len=0), "q_seqlen_value must be >= 1"),
    (dict(q_len=4), "multiple of q_seqlen_value"),
    (dict(q_len=3), "batch entries"),
    (dict(cache=_pool(9, 4, 8704)), "cache must be a contiguous uint8"),
    (dict(block_table=_i64(3, 4)), "int32"),
    (dict(block_table=_e(2, 4, dtype=torch.int32)), "batch entries"),
    (dict(block_table=_e(3, 8, dtype=torch.int32)[:, ::2]), "contiguous int32"),
    (dict(lens=_e(3, dtype=torch.int32)), "int64"),
    (dict(scale=0.0), "scale must be"),
    (dict(scale=math.nan), "scale must be"),
    (dict(scale=3e38), "scale must be"),
    (dict(lens=torch.empty(3, dtype=torch.int64)), "same HIP device"),
])
def test_decode_refusals(bad, msg):
    with pytest.raises(RuntimeError, match="kv4_decode: .*" + msg):
        _decode(**bad)


@pytest.mark.parametrize("bad,msg", [
    (dict(query=_e(3, 16, 127)), "query must be"),
    (dict(query=_e(3, 17, 128)), "multiple of the cache's kv heads"),
    (dict(pc=_pool(9, 4, 512)), "prefix_cache must be"),
    (dict(sc=_pool(9, 4, 512)), "suffix_cache must be"),
    (dict(sc=_pool(9, 2, 17408)), "same kv heads"),
    (dict(pbt=_e(2, 4, dtype=torch.int32)), "prefix block_table rows"),
    (dict(plen=_i64(3)), "prefix block_table rows"),
    (dict(sbt=_e(2, 4, dtype=torch.int32)), "suffix block_table rows"),
    (dict(slens=_e(3, dtype=torch.int32)), "suffix kv seqlens"),
    (dict(scale=-1.0), "scale must be"),
    (dict(sc=torch.empty(2, 4, 17408, dtype=torch.uint8)), "same HIP device"),
])
def test_cascade_refusals(bad, msg):
    with pytest.raises(RuntimeError, match="kv4_cascade_decode: .*" + msg):
        _cascade(**bad)


def test_ops_refuse_host_tensors():
    with pytest.raises((RuntimeError, NotImplementedError)):
        OPS.kv4_cache_read(torch.zeros(1, 1, 17408, dtype=torch.uint8), torch.zeros(1, dtype=torch.int64))


# ---- the C entry points refuse before anything is launched ---------------------------------------
# addresses that are never followed: aligned, or not
A, ODD = 4096, 4100
TEXT = open(abi._HEADER).read()
INVALID, UNSUPPORTED, NULL, WORKSPACE = (int(TEXT.split("#define " + n)[1].split()[0].strip("()")) for n in (
    "CK_E_INVALID_ARG", "CK_E_UNSUPPORTED", "CK_E_NULL_PTR", "CK_E_WORKSPACE"))


def _c_write(**kw):
    a = dict(k=A, kts=512, khs=128, v=A, vts=512, vhs=128, slots=A, cache=A, blocks=4, tokens=5, kv_heads=4, dtype=0, stream=None)
    a.update(kw)
    return abi.lib().ck_kv4_cache_write(*a.values())


def _c_read(**kw):
    a = dict(cache=A, slots=A, blocks=4, tokens=5, kv_heads=4, dtype=0, k=A, v=A, stream=None)
    a.update(kw)
    return abi.lib().ck_kv4_cache_read(*a.values())


def _c_decode(**kw):
    a = dict(q=A, cache=A, bt=A, cols=4, lens=A, batch=3, q_len=1, heads=16, kv_heads=4, blocks=9, page=128, dtype=0,
             scale=0.1, out=A, lse=A, ws=A, ws_bytes=0, stream=None)
    a.update(kw)
    return abi.lib().ck_kv4_decode(*a.values())


def _c_cascade(**kw):
    a = dict(q=A, pc=A, pbt=A, pcols=4, plen=A, pblocks=9, sc=A, sbt=A, scols=4, slens=A, sblocks=9, batch=3, heads=16,
             kv_heads=4, page=128, dtype=0, scale=0.1, out=A, lse=A, ws=A, ws_bytes=0, stream=None)
    a.update(kw)
    return abi.lib().ck_kv4_cascade_decode(*a.values())


def test_c_write_refuses():
    for bad in (dict(kts=4), dict(khs=-8), dict(vts=2 ** 28 + 8), dict(vhs=129), dict(tokens=-1), dict(blocks=-1), dict(kv_heads=0),
                dict(kv_heads=1025), dict(blocks=2 ** 31 + 1), dict(k=ODD), dict(v=ODD), dict(slots=ODD), dict(cache=ODD),
                dict(tokens=2 ** 28), dict(tokens=2 ** 63 - 1)):
        assert _c_write(**bad) == INVALID, bad
    for name in ("k", "v", "slots", "cache"):
        assert _c_write(**{name: None}) == NULL, name
    assert _c_write(dtype=1) == UNSUPPORTED
    assert _c_write(tokens=0, k=None) == 0 and _c_write(blocks=0, cache=None) == 0


def test_c_read_refuses():
    for bad in (dict(tokens=-1), dict(blocks=-1), dict(kv_heads=0), dict(kv_heads=1025), dict(cache=ODD), dict(slots=ODD),
                dict(k=ODD), dict(v=ODD), dict(tokens=2 ** 28)):
        assert _c_read(**bad) == INVALID, bad
    for name in ("k", "v", "slots", "cache"):
        assert _c_read(**{name: None}) == NULL, name
    assert _c_read(dtype=3) == UNSUPPORTED
    assert _c_read(tokens=0, k=None) == 0


@pytest.mark.parametrize("bad,code", [
    (dict(dtype=1), UNSUPPORTED),
    (dict(page=64), UNSUPPORTED),
    (dict(q_len=0), INVALID),
    (dict(heads=0), INVALID),
    (dict(kv_heads=0), INVALID),
    (dict(kv_heads=5), INVALID),
    (dict(kv_heads=32), INVALID),
    (dict(heads=2 ** 16, kv_heads=2 ** 11), INVALID),
    (dict(heads=2 ** 17), INVALID),
    (dict(batch=-1), INVALID),
    (dict(cols=-1), INVALID),
    (dict(cols=2 ** 23 + 1), INVALID),
    (dict(cols=2 ** 57), INVALID),                        # times 128 it is 0 in 64 bits
    (dict(batch=2 ** 18, cols=2 ** 10), INVALID),         # the list passes 2^31 places
    (dict(batch=2 ** 20), INVALID),                       # 2^24 rows
    (dict(batch=2 ** 62, q_len=2 ** 62), INVALID),
    (dict(blocks=2 ** 31 + 1), INVALID),
    (dict(blocks=-1), INVALID),
    (dict(scale=0.0), INVALID),
    (dict(scale=math.nan), INVALID),
    (dict(scale=3e38), INVALID),
    (dict(q=None), NULL),
    (dict(cache=None), NULL),
    (dict(bt=None), NULL),
    (dict(lens=None), NULL),
    (dict(lse=None), NULL),
    (dict(q=ODD), INVALID),
    (dict(out=ODD), INVALID),
    (dict(cache=ODD), INVALID),
    (dict(lens=ODD), INVALID),
    (dict(bt=A + 2), INVALID),
    (dict(ws=ODD, ws_bytes=1 << 40), INVALID),
    (dict(ws_bytes=1 << 40, ws=None), WORKSPACE),
    (dict(), WORKSPACE),
    (dict(batch=2 ** 20 - 1), WORKSPACE),                 # the last size before a limit is planned
    (dict(q_len=2 ** 18, batch=1, kv_heads=1), WORKSPACE),
])
def test_c_decode_refuses(bad, code):
    assert _c_decode(**bad) == code


def test_c_workspaces_are_the_plans():
    n = ctypes.c_int64(0)
    p = ctypes.byref(n)
    lib = abi.lib()
    assert lib.ck_kv4_decode_plan(3, 1, 16, 4, 512, p) == 0 and n.value > 0
    assert _c_decode(ws_bytes=n.value - 1) == WORKSPACE
    assert lib.ck_kv4_cascade_decode_plan(3, 16, 4, 512, 512, p) == 0 and n.value > 0
    assert _c_cascade(ws_bytes=n.value - 1) == WORKSPACE
    assert lib.ck_kv4_decode_plan(3, 1, 16, 4, 512, None) == NULL
    assert lib.ck_kv4_decode_plan(3, 0, 16, 4, 512, p) == INVALID
    assert lib.ck_kv4_decode_plan(3, 1, 16, 3, 512, p) == INVALID
    assert lib.ck_kv4_cascade_decode_plan(3, 16, 4, -1, 512, p) == INVALID
    assert lib.ck_kv4_cascade_decode_plan(3, 16, 4, 512, 512, None) == NULL
    assert _c_decode(batch=0, ws=None) == 0 and _c_cascade(batch=0, ws=None) == 0  # nothing to do


def test_c_cascade_refuses():
    assert _c_cascade() == WORKSPACE
    for name in ("q", "plen", "pbt", "pc", "slens", "sbt", "sc", "out", "lse"):
        assert _c_cascade(**{name: None}) == NULL, name
    for bad in (dict(pc=ODD), dict(plen=ODD), dict(pcols=-1), dict(pblocks=-1), dict(scale=-1.0), dict(pcols=2 ** 23 + 1),
                dict(scols=2 ** 57), dict(heads=18), dict(batch=2 ** 20)):
        assert _c_cascade(**bad) == INVALID, bad
    assert _c_cascade(dtype=7) == UNSUPPORTED and _c_cascade(page=256) == UNSUPPORTED


# ---- the list ------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def header(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv4_map")
    src = d / "kv4_map.cpp"
    src.write_text("""#include "kv4_map.h"
using namespace ck::kv4;
extern "C" int shares(int w, int waves, int least, int each, int pieces, int *lo) {
    const Shares s = list_shares(w, waves, least, each, pieces);
    for (int k = 0; k <= s.count; ++k) lo[k] = share_lo(s, k);
    return s.count;
}
extern "C" void range(int w, int waves, int least, int each, int pieces, int h, int u, int n, int *out) {
    const ShareRange r = shares_of(list_shares(w, waves, least, each, pieces), h, u, n);
    out[0] = r.first, out[1] = r.count;
}
extern "C" long long slot(int before, int after, int wave, int waves, int item) { return part_slot(before, after, wave, waves, item); }
""")
    lib = d / "kv4_map.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-I", CSRC, str(src), "-o", str(lib)], check=True)
    lib = ctypes.CDLL(str(lib))
    lib.slot.restype = ctypes.c_longlong
    return lib


@pytest.mark.parametrize("merge", [False, True])
@pytest.mark.parametrize("least", [1, 4])
@pytest.mark.parametrize("waves", [1, 3, 17, 85, 256, 2048])
@pytest.mark.parametrize("units", [[1], [3], [251], [0, 0, 7], [5, 0, 1, 300, 2], [1] * 400, [9000], [64, 64, 64], [0]])
def test_parts_of_the_list(header, units, waves, least, merge):
    """The shares, walked as the kernels walk them: every place once, a slot for one part only and within the
    workspace, and the parts that the fold looks for are those that were left. Of one request's list an item's
    shares may be its own."""
    kv_heads = 3
    w = sum(units) * kv_heads
    pieces = waves // kv_heads if least > 1 and len(units) == 1 else 0
    args = (w, waves, least, units[0], pieces)
    lo = (ctypes.c_int * (waves + 1))()
    n = header.shares(*args, lo)
    lo = list(lo)[:n + 1]
    assert 0 <= n <= waves and (n == 0) == (w == 0)
    assert w == 0 or (lo[0] == 0 and lo[-1] == w and min(np.diff(lo)) > 0)
    if pieces and w:  # cut at the items, unless that makes shares much longer
        assert all(x in lo for x in range(0, w, units[0])) or max(np.diff(lo)) + 8 < -(-units[0] // pieces)
    left, at, item = {}, 0, 0
    for each in units:
        for h in range(kv_heads):
            if each:
                out = (ctypes.c_int * 2)()
                header.range(*args, h if len(units) == 1 else 0, at, each, out)
                c0, c1 = out[0], out[0] + out[1] - 1
                assert lo[c0] <= at < lo[c0 + 1] and lo[c1] <= at + each - 1 < lo[c1 + 1]
                for k in range(c0, c1 + 1):  # what wave k has of the item
                    before, after = int(lo[k] > at), int(lo[k + 1] < at + each)
                    assert (before, after) == (int(k > c0), int(k < c1))
                    if before or after or merge:
                        slot = header.slot(before, after, k, waves, item)
                        assert 0 <= slot < 2 * waves + (len(units) * kv_heads if merge else 0)
                        assert slot not in left
                        left[slot] = item
            at += each
            item += 1


# ---- the oracle ------------------------------------------------------------------------------------
def test_oracle_places_are_one_byte_each():
    codes_k, codes_v, ks, vs = o4.places(torch.arange(128))
    every = torch.cat([x.flatten() for x in (codes_k, codes_v, ks, vs)])
    assert torch.equal(every.sort().values, torch.arange(17408))


def test_oracle_quantises_to_the_nearest():
    """Against a search over all 16 codes of each scale; the scale rule by hand."""
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(64, 128, generator=g) * torch.exp(torch.randn(64, 1, generator=g) * 5)).to(BF)
    codes, e = o4.quantise(x)
    grp = x.double().view(64, 4, 32)
    most = grp.abs().amax(-1)
    for i in range(64):
        for k in range(4):
            f = math.frexp(most[i, k].item())[1] - 1
            want = f - 2 + (most[i, k].item() > 1.75 * 2.0 ** f) + 127
            assert e[i, k] == min(max(want, 8), 252)
    got = o4.values(codes, e).view(64, 4, 32)
    step = torch.exp2(e.double() - 127)[..., None]
    grid = torch.tensor(o4.E2M1 + tuple(-v for v in o4.E2M1), dtype=torch.float64)
    best = (grp[..., None] - grid * step[..., None]).abs().amin(-1)
    assert torch.equal((grp - got).abs(), best)
    # the largest is in (3.5, 7] steps, the numbers up to 4, 6 and 8 are 1 or 2 apart
    assert ((grp - got).abs() <= step).all()


def test_oracle_reads_what_it_writes():
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(200, 2, 128, generator=g).to(HF) for _ in range(2))
    slots = torch.randperm(3 * 128, generator=g)[:200]
    slots[7] = -1
    pool = o4.write(torch.zeros(3, 2, 17408, dtype=torch.uint8), k, v, slots)
    for got, x in zip(o4.read(pool, slots), (k, v)):
        want = o4.values(*o4.quantise(x))
        want[7] = 0
        assert torch.equal(got, want)
    # 1 is 4 * 2^-2: e = 125
    codes, e = o4.quantise(torch.tensor([[math.inf] + [1.0] * 127, [0.0] * 128], dtype=BF))
    assert e[0].tolist() == [255, 125, 125, 125] and e[1].tolist() == [8] * 4 and (codes[1] == 0).all()
    assert o4.values(codes, e)[0, :32].isnan().all() and (o4.values(codes, e)[0, 32:] == 1).all()


def test_oracle_is_the_formula():
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(n, 128, generator=g, dtype=torch.float64) for n in (3, 5, 5))
    o, lse, _, _ = o4.attend(q, k, v, [4, 2, 0], 0.1, BF, 3)
    for i, n in enumerate((4, 2, 0)):
        if n == 0:
            assert (o[i] == 0).all() and lse[i] == -math.inf
            continue
        w = [math.exp(0.1 * float(q[i] @ k[j])) for j in range(n)]
        assert abs(lse[i].item() - math.log(sum(w))) < 1e-12
        assert (o[i] - sum(w[j] * v[j] for j in range(n)) / sum(w)).abs().max() < 1e-12


@pytest.mark.parametrize("rows", [16, 17])
def test_oracle_bounds_have_teeth(rows):
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(n, 128, generator=g) for n in (4, 70, 70))
    ref = o4.attend(q, k, v, 70, 0.05, BF, rows)
    close(ref[0].bfloat16(), ref[1], ref)
    with pytest.raises(AssertionError):  # a token left out
        short = o4.attend(q, k[:69], v[:69], 69, 0.05, BF, rows)
        close(short[0].bfloat16(), short[1], ref)
