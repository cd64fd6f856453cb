"""Host-side checks of the latent operators (no GPU): shapes on meta tensors, refusals of the
torch ops and of the C entry points, and the oracle against a direct sum."""
import ctypes
import math

import pytest
import torch

import cascade_amd  # noqa: F401
from cascade_amd import abi
from oracle import latent as ol

M = "meta"
OPS = torch.ops.npu


def _e(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device=M)


def _i64(*shape):
    return _e(*shape, dtype=torch.int64)


def _write(**kw):
    a = dict(kv=_e(5, 576), gamma=_e(512), cos_sin=_e(64, 64, dtype=torch.float32), positions=_i64(5), slots=_i64(5),
             cache=_e(4, 128, 576), eps=1e-6, interleaved=True)
    a.update(kw)
    return OPS.latent_cache_write(*a.values())


def _decode(**kw):
    a = dict(query=_e(6, 16, 576), cache=_e(9, 128, 576), block_table=_e(3, 4, dtype=torch.int32), lens=_i64(3),
             scale=0.1, q_len=2)
    a.update(kw)
    return OPS.latent_decode(*a.values())


def _cascade(**kw):
    a = dict(query=_e(3, 16, 576), pc=_e(9, 128, 576), pbt=_e(1, 4, dtype=torch.int32), plen=_i64(1),
             sc=_e(9, 128, 576), sbt=_e(3, 4, dtype=torch.int32), slens=_i64(3), scale=0.1)
    a.update(kw)
    return OPS.latent_cascade_decode(*a.values())


def _prefill(**kw):
    a = dict(query=_e(10, 4, 192), key=_e(12, 4, 128), key_rope=_e(12, 64), value=_e(12, 4, 128), ql=_i64(2), kl=_i64(2),
             scale=0.1, causal=True)
    a.update(kw)
    return OPS.latent_prefill(*a.values())


def test_shapes():
    assert _write() is None
    for dt in (torch.bfloat16, torch.float16):
        out, lse = _decode(query=_e(6, 16, 576, dtype=dt), cache=_e(9, 128, 576, dtype=dt))
        assert out.shape == (6, 16, 512) and out.dtype == dt and lse.shape == (96,) and lse.dtype == torch.float32
    out, lse = _cascade()
    assert out.shape == (3, 16, 512) and lse.shape == (48,)
    out, lse = _prefill()
    assert out.shape == (10, 4, 128) and lse.shape == (40,)
    out, lse = _decode(query=_e(0, 16, 576), block_table=_e(0, 4, dtype=torch.int32), lens=_i64(0))
    assert out.shape == (0, 16, 512) and lse.shape == (0,)
    out, lse = _prefill(query=_e(0, 4, 192))
    assert out.shape == (0, 4, 128) and lse.shape == (0,)


@pytest.mark.parametrize("bad,msg", [
    (dict(kv=_e(5, 575)), r"kv must be \(T, 576\)"),
    (dict(kv=_e(5, 576, dtype=torch.float32)), "kv must be bf16 or fp16"),
    (dict(kv=_e(5, 580)[:, :576]), "row stride"),
    (dict(kv=_e(576, 5).t()), "unit column stride"),
    (dict(gamma=_e(512, dtype=torch.float16)), "gamma must be"),
    (dict(gamma=_e(511)), "gamma must be"),
    (dict(cos_sin=_e(64, 64)), "cos_sin must be"),
    (dict(cos_sin=_e(64, 32, dtype=torch.float32)), "cos_sin must be"),
    (dict(positions=_i64(4)), "positions and slots"),
    (dict(slots=_e(5, dtype=torch.int32)), "positions and slots"),
    (dict(slots=_i64(10)[::2]), "positions and slots"),
    (dict(cache=_e(4, 64, 576)), "pool"),
    (dict(cache=_e(4, 128, 576, dtype=torch.float16)), "dtype"),
    (dict(cache=_e(4, 128, 640)[:, :, :576]), "contiguous"),
    (dict(eps=0.0), "eps must be"),
    (dict(eps=math.inf), "eps must be"),
    (dict(slots=torch.empty(5, dtype=torch.int64)), "same HIP device"),
])
def test_write_refusals(bad, msg):
    with pytest.raises(RuntimeError, match="latent_cache_write: .*" + msg):
        _write(**bad)


@pytest.mark.parametrize("bad,msg", [
    (dict(query=_e(6, 16, 512)), r"query must be a contiguous \(T, H, 576\)"),
    (dict(query=_e(16, 6, 576).transpose(0, 1)), "query must be a contiguous"),
    (dict(query=_e(6, 0, 576)), "query must have heads"),
    (dict(query=_e(6, 16, 576, dtype=torch.float32)), "query must be bf16 or fp16"),
    (dict(q_len=0), "q_seqlen_value must be >= 1"),
    (dict(q_len=4), "multiple of q_seqlen_value"),
    (dict(q_len=3), "batch entries"),
    (dict(cache=_e(9, 64, 576)), "pool"),
    (dict(cache=_e(9, 128, 576, dtype=torch.float16)), "dtype"),
    (dict(block_table=_e(3, 4, dtype=torch.int64)), "int32"),
    (dict(block_table=_e(2, 4, dtype=torch.int32)), "batch entries"),
    (dict(block_table=_e(3, 8, dtype=torch.int32)[:, ::2]), "contiguous int32"),
    (dict(lens=_e(3, dtype=torch.int32)), "int64"),
    (dict(scale=0.0), "scale must be"),
    (dict(scale=math.nan), "scale must be"),
    (dict(scale=1e300), "scale must be"),
    (dict(scale=3e38), "scale must be"),
    (dict(lens=torch.empty(3, dtype=torch.int64)), "same HIP device"),
])
def test_decode_refusals(bad, msg):
    with pytest.raises(RuntimeError, match="latent_decode: .*" + msg):
        _decode(**bad)


@pytest.mark.parametrize("bad,msg", [
    (dict(query=_e(3, 16, 575)), "query must be"),
    (dict(pc=_e(9, 128, 512)), "prefix_cache must be"),
    (dict(sc=_e(9, 128, 576, dtype=torch.float16)), "suffix_cache must have the dtype"),
    (dict(pbt=_e(2, 4, dtype=torch.int32)), "prefix block_table rows"),
    (dict(plen=_i64(3)), "prefix block_table rows"),
    (dict(sbt=_e(2, 4, dtype=torch.int32)), "suffix block_table rows"),
    (dict(slens=_e(3, dtype=torch.int32)), "suffix kv seqlens"),
    (dict(scale=-1.0), "scale must be"),
])
def test_cascade_refusals(bad, msg):
    with pytest.raises(RuntimeError, match="latent_cascade_decode: .*" + msg):
        _cascade(**bad)


@pytest.mark.parametrize("bad,msg", [
    (dict(query=_e(10, 4, 128)), r"query must be a contiguous \(T, H, 192\)"),
    (dict(key=_e(12, 5, 128)), "key and value must be"),
    (dict(value=_e(12, 4, 64)), "key and value must be"),
    (dict(value=_e(11, 4, 128)), "key and value must be"),
    (dict(key_rope=_e(12, 32)), "key_rope must be"),
    (dict(key_rope=_e(11, 64)), "key_rope must be"),
    (dict(key=_e(12, 4, 128, dtype=torch.float16)), "query's dtype"),
    (dict(key=_e(12, 4, 256)[..., ::2]), "unit stride"),
    (dict(value=_e(12, 4, 132)[..., :128]), "multiples of 8"),
    (dict(key=torch.empty_strided((12, 4, 128), (2 ** 25, 128, 1), dtype=torch.bfloat16, device=M)), "at most 2"),
    (dict(ql=_e(2, dtype=torch.int32)), "seqlens must be"),
    (dict(kl=_i64(3)), "batch entries"),
    (dict(scale=math.inf), "scale must be"),
    (dict(kl=torch.empty(2, dtype=torch.int64)), "same HIP device"),
])
def test_prefill_refusals(bad, msg):
    with pytest.raises(RuntimeError, match="latent_prefill: .*" + msg):
        _prefill(**bad)


def test_ops_refuse_host_tensors():
    with pytest.raises((RuntimeError, NotImplementedError)):
        OPS.latent_decode(torch.zeros(1, 1, 576, dtype=torch.bfloat16), torch.zeros(1, 128, 576, dtype=torch.bfloat16),
                          torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int64), 1.0)


# ---- the C entry points refuse before anything is launched ---------------------------------------
# addresses that are never followed: aligned, or not
A, ODD = 4096, 4100


def _codes():
    text = open(abi._HEADER).read()
    return {n: int(text.split("#define " + n)[1].split()[0].strip("()")) for n in
            ("CK_E_INVALID_ARG", "CK_E_UNSUPPORTED", "CK_E_NULL_PTR", "CK_E_WORKSPACE")}


def _c_decode(**kw):
    a = dict(q=A, cache=A, bt=A, cols=4, lens=A, batch=3, q_len=1, heads=16, blocks=9, page=128, dtype=0, scale=0.1,
             out=A, lse=A, ws=A, ws_bytes=0, stream=None)
    a.update(kw)
    return abi.lib().ck_latent_decode(*a.values())


@pytest.mark.parametrize("bad,code", [
    (dict(dtype=1), "CK_E_UNSUPPORTED"),
    (dict(page=64), "CK_E_UNSUPPORTED"),
    (dict(q_len=0), "CK_E_INVALID_ARG"),
    (dict(heads=0), "CK_E_INVALID_ARG"),
    (dict(batch=-1), "CK_E_INVALID_ARG"),
    (dict(cols=-1), "CK_E_INVALID_ARG"),
    (dict(cols=2 ** 23 + 1), "CK_E_INVALID_ARG"),
    (dict(batch=2 ** 20, cols=2 ** 12), "CK_E_INVALID_ARG"),      # the list passes 2^31 places
    (dict(batch=2 ** 20, heads=2 ** 11), "CK_E_INVALID_ARG"),     # 2^31 rows
    (dict(blocks=2 ** 31 + 1), "CK_E_INVALID_ARG"),
    (dict(scale=0.0), "CK_E_INVALID_ARG"),
    (dict(scale=math.nan), "CK_E_INVALID_ARG"),
    (dict(scale=3e38), "CK_E_INVALID_ARG"),
    (dict(q=None), "CK_E_NULL_PTR"),
    (dict(cache=None), "CK_E_NULL_PTR"),
    (dict(bt=None), "CK_E_NULL_PTR"),
    (dict(lse=None), "CK_E_NULL_PTR"),
    (dict(q=ODD), "CK_E_INVALID_ARG"),
    (dict(cache=ODD), "CK_E_INVALID_ARG"),
    (dict(lens=ODD), "CK_E_INVALID_ARG"),
    (dict(ws_bytes=1 << 40, ws=None), "CK_E_WORKSPACE"),
    (dict(), "CK_E_WORKSPACE"),
])
def test_c_decode_refuses(bad, code):
    assert _c_decode(**bad) == _codes()[code]


def test_c_decode_workspace_is_the_plans():
    n = ctypes.c_int64(0)
    assert abi.lib().ck_latent_decode_plan(3, 1, 16, 512, ctypes.byref(n)) == 0 and n.value > 0
    assert _c_decode(ws_bytes=n.value - 1) == _codes()["CK_E_WORKSPACE"]
    assert abi.lib().ck_latent_decode_plan(3, 1, 16, 512, None) == _codes()["CK_E_NULL_PTR"]
    assert abi.lib().ck_latent_decode_plan(3, 0, 16, 512, ctypes.byref(n)) == _codes()["CK_E_INVALID_ARG"]
    assert abi.lib().ck_latent_cascade_decode_plan(3, 16, -1, 512, ctypes.byref(n)) == _codes()["CK_E_INVALID_ARG"]
    assert _c_decode(batch=0, ws=None) == 0  # nothing to do


def test_c_cascade_refuses():
    def call(**kw):
        a = dict(q=A, pc=A, pbt=A, pcols=4, plen=A, pblocks=9, sc=A, sbt=A, scols=4, slens=A, sblocks=9, batch=3,
                 heads=16, page=128, dtype=0, scale=0.1, out=A, lse=A, ws=A, ws_bytes=0, stream=None)
        a.update(kw)
        return abi.lib().ck_latent_cascade_decode(*a.values())
    c = _codes()
    assert call() == c["CK_E_WORKSPACE"]
    for bad in (dict(plen=None), dict(pbt=None), dict(pc=None), dict(out=None)):
        assert call(**bad) == c["CK_E_NULL_PTR"], bad
    for bad in (dict(pc=ODD), dict(plen=ODD), dict(pcols=-1), dict(pblocks=-1), dict(scale=-1.0), dict(pcols=2 ** 23 + 1)):
        assert call(**bad) == c["CK_E_INVALID_ARG"], bad
    assert call(dtype=7) == c["CK_E_UNSUPPORTED"]


def test_c_write_refuses():
    def call(**kw):
        a = dict(kv=A, stride=576, gamma=A, cs=A, max_pos=64, pos=A, slots=A, cache=A, blocks=4, tokens=5, dtype=0,
                 eps=1e-6, inter=1, stream=None)
        a.update(kw)
        return abi.lib().ck_latent_cache_write(*a.values())
    c = _codes()
    for bad in (dict(stride=575), dict(stride=580), dict(tokens=-1), dict(eps=0.0), dict(eps=math.inf), dict(kv=ODD),
                dict(cache=ODD), dict(slots=ODD), dict(blocks=-1)):
        assert call(**bad) == c["CK_E_INVALID_ARG"], bad
    for name in ("kv", "gamma", "cs", "pos", "slots", "cache"):
        assert call(**{name: None}) == c["CK_E_NULL_PTR"], name
    assert call(dtype=1) == c["CK_E_UNSUPPORTED"]
    assert call(tokens=0) == 0 and call(blocks=0) == 0


def test_c_prefill_refuses():
    def call(**kw):
        a = dict(q=A, k=A, kts=512, khs=128, kr=A, krs=64, v=A, vts=512, vhs=128, ql=A, kl=A, batch=2, tokens=10,
                 keys=12, heads=4, dtype=0, scale=0.1, causal=1, out=A, lse=A, stream=None)
        a.update(kw)
        return abi.lib().ck_latent_prefill(*a.values())
    c = _codes()
    for bad in (dict(kts=4), dict(khs=-8), dict(vts=2 ** 24 + 8), dict(heads=0), dict(tokens=-1), dict(keys=2 ** 30),
                dict(batch=2 ** 16 + 1), dict(scale=math.nan), dict(scale=3e38), dict(q=ODD), dict(v=ODD), dict(ql=ODD)):
        assert call(**bad) == c["CK_E_INVALID_ARG"], bad
    for name in ("q", "k", "kr", "v", "ql", "kl", "out", "lse"):
        assert call(**{name: None}) == c["CK_E_NULL_PTR"], name
    assert call(dtype=1) == c["CK_E_UNSUPPORTED"]
    assert call(tokens=0) == 0


# ---- the oracle ------------------------------------------------------------------------------------
def test_oracle_is_the_formula():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, d, generator=g, dtype=torch.float64) for n, d in ((3, 8), (5, 8), (5, 4)))
    k[4], v[4] = math.nan, math.inf  # seen by nobody
    o, lse, _, _ = ol.attend(q, k, v, [4, 2, 0], 0.7, torch.bfloat16)
    for i, n in enumerate((4, 2, 0)):
        w = [math.exp(0.7 * float(q[i] @ k[j])) for j in range(n)]
        if n == 0:
            assert torch.equal(o[i], torch.zeros(4, dtype=torch.float64)) and lse[i] == -math.inf
            continue
        assert abs(lse[i].item() - math.log(sum(w))) < 1e-12
        want = sum(w[j] * v[j] for j in range(n)) / sum(w)
        assert (o[i] - want).abs().max() < 1e-12


@pytest.mark.parametrize("interleaved", [True, False])
def test_oracle_rotation_keeps_lengths(interleaved):
    g = torch.Generator().manual_seed(1)
    kv = torch.randn(4, 576, generator=g, dtype=torch.float64)
    ang = torch.rand(9, 32, generator=g, dtype=torch.float64)
    rows = ol.write_rows(kv, torch.ones(512), torch.cat([ang.cos(), ang.sin()], 1), torch.tensor([0, 3, 8, 3]), 1e-6,
                         interleaved)
    assert (rows[:, 512:].norm(dim=1) - kv[:, 512:].norm(dim=1)).abs().max() < 1e-12
    assert (rows[:, :512].pow(2).mean(1) - 1).abs().max() < 1e-4


def test_oracle_bounds_have_teeth():
    g = torch.Generator().manual_seed(2)
    q, x = torch.randn(4, 576, generator=g), torch.randn(70, 576, generator=g)
    ref = ol.attend(q, x, x[:, :512], 70, 0.05, torch.bfloat16)
    ol.close(ref[0].bfloat16(), ref[1], ref)
    with pytest.raises(AssertionError):  # a token left out
        short = ol.attend(q, x[:69], x[:69, :512], 69, 0.05, torch.bfloat16)
        ol.close(short[0].bfloat16(), short[1], ref)
