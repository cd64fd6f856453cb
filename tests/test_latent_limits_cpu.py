"""Sizes that the latent entry points cannot launch are refused on the host (no GPU): at each
limit of cascade_kernels.h, one past it and far past it."""
import ctypes

import pytest

from cascade_amd import abi

A = 4096  # an aligned address that is never followed
TEXT = open(abi._HEADER).read()
INVALID, WORKSPACE = (int(TEXT.split("#define " + n)[1].split()[0].strip("()")) for n in ("CK_E_INVALID_ARG", "CK_E_WORKSPACE"))


def _plan(batch=1, q_len=1, heads=1, kv=128):
    n = ctypes.c_int64(0)
    return abi.lib().ck_latent_decode_plan(batch, q_len, heads, kv, ctypes.byref(n))


def _decode(**kw):
    a = dict(q=A, cache=A, bt=A, cols=1, lens=A, batch=1, q_len=1, heads=1, blocks=9, page=128, dtype=0, scale=0.1,
             out=A, lse=A, ws=A, ws_bytes=0, stream=None)
    a.update(kw)
    return abi.lib().ck_latent_decode(*a.values())


def _cascade(**kw):
    a = dict(q=A, pc=A, pbt=A, pcols=4, plen=A, pblocks=9, sc=A, sbt=A, scols=4, slens=A, sblocks=9, batch=3,
             heads=16, page=128, dtype=0, scale=0.1, out=A, lse=A, ws=A, ws_bytes=0, stream=None)
    a.update(kw)
    return abi.lib().ck_latent_cascade_decode(*a.values())


def _write(**kw):
    a = dict(kv=A, stride=576, gamma=A, cs=A, max_pos=64, pos=A, slots=A, cache=A, blocks=4, tokens=5, dtype=0,
             eps=1e-6, inter=1, stream=None)
    a.update(kw)
    return abi.lib().ck_latent_cache_write(*a.values())


def _prefill(**kw):
    a = dict(q=A, k=A, kts=512, khs=128, kr=A, krs=64, v=A, vts=512, vhs=128, ql=A, kl=A, batch=2, tokens=10,
             keys=12, heads=4, dtype=0, scale=0.1, causal=1, out=A, lse=A, stream=None)
    a.update(kw)
    return abi.lib().ck_latent_prefill(*a.values())


# The fold takes a workgroup of 256 threads for 16 heads of a token; a launch holds 2^32 threads at most.
@pytest.mark.parametrize("ok,past", [
    (dict(batch=2 ** 12 - 1, q_len=2 ** 12), dict(batch=2 ** 12, q_len=2 ** 12)),
    (dict(batch=2 ** 24 - 1), dict(batch=2 ** 24)),
    (dict(batch=2 ** 20 - 1, q_len=16, heads=16), dict(batch=2 ** 20, q_len=16, heads=16)),
    (dict(batch=2 ** 23 - 1, heads=17), dict(batch=2 ** 23, heads=17)),
    (dict(q_len=2 ** 20, heads=128), dict(q_len=2 ** 21, heads=128)),
])
def test_decode_blocks_of_the_fold(ok, past):
    assert _plan(**ok) == 0 and _decode(**ok) == WORKSPACE  # planned; nothing else is wrong with the call
    assert _plan(**past) == INVALID and _decode(**past) == INVALID


def test_cascade_blocks_of_the_fold():
    assert _cascade(batch=2 ** 20 - 1, heads=130) == WORKSPACE
    assert _cascade(batch=2 ** 21, heads=128) == INVALID
    assert _cascade(batch=2 ** 23, heads=32) == INVALID


@pytest.mark.parametrize("cols", [2 ** 23 + 1, 2 ** 56, 2 ** 57, 2 ** 57 + 1, 2 ** 62, -1, -2 ** 57, -2 ** 63])
def test_table_columns_do_not_wrap(cols):
    # 2^57 columns of 128 tokens are 0 in 64 bits
    assert _decode(cols=cols) == INVALID
    assert _cascade(pcols=cols) == INVALID
    assert _cascade(scols=cols) == INVALID


@pytest.mark.parametrize("tokens", [2 ** 26 - 3, 2 ** 26, 2 ** 32, 2 ** 40, 2 ** 63 - 1])
def test_write_tokens(tokens):
    assert _write(tokens=tokens) == INVALID


@pytest.mark.parametrize("bad", [dict(batch=2 ** 16, heads=128), dict(batch=1, tokens=2 ** 29, heads=4),
                                 dict(batch=2 ** 16, tokens=1, heads=2 ** 16), dict(batch=126, tokens=256, heads=2 ** 16)])
def test_prefill_workgroups(bad):
    # 512 threads for 256 rows of a head; every request's last rows may be a part
    assert _prefill(**bad) == INVALID
