"""More of the latent operators at their edges, against the 64-bit definition: largest scores
that the last products decide, fp16 (whose probabilities could overflow) in every form."""
import math

import pytest
import torch

from oracle import latent as ol
from tests.test_gpu_latent import BF, DEV, HF, OPS, SCALE, _check_decode, _check_prefill, _gen, _i64, _pool, _prompt, _randn, _rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import cascade_amd  # noqa: F401
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible to torch")


# ---- one key above all others, by the last rotated dims alone -------------------------------------------
# A reference point of the softmax that missed the last products would be too low by `nats`: in fp16
# probabilities of 2^(7 + 1.44 nats) overflow from 6.2 on.
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("key,nats", [(0, 8.0), (0, 12.0), (2, 10.0), (5, 9.0), (18, 12.0), (40, 12.0)])
def test_prefill_first_keys_are_the_largest(dtype, key, nats):
    g = _gen(50 + key)
    ql, kl = [300, 70, 33], [300, 131, 48]
    q, k, kr, v = _prompt(g, ql, kl, 2, dtype)
    q[..., :128] *= 0.25
    q[..., 128:] = 0
    q[..., 191] = 4
    kr[:, 63] = 0
    for b in range(3):
        kr[sum(kl[:b]) + key, 63] = nats / (4 * SCALE)
    for causal in (True, False):
        out, lse = OPS.latent_prefill(q, k, kr, v, _i64(ql), _i64(kl), SCALE, causal)
        _check_prefill(q, k, kr, v, ql, kl, causal, out, lse)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("key,nats", [(0, 8.0), (0, 12.0), (2, 10.0), (5, 9.0), (18, 12.0)])
@pytest.mark.parametrize("heads", [1, 16, 40])
def test_decode_first_keys_are_the_largest(dtype, heads, key, nats):
    g = _gen(60 + key)
    lens = [20, 32, 64, 300, 1000]
    cache, table = _pool(g, lens, dtype, garbage=False)
    cache[..., 575] = 0
    for b in range(len(lens)):
        cache[table[b, 0].item(), key, 575] = nats / (4 * SCALE)
    q = _randn(g, len(lens), heads, 576, dtype=dtype, scale=0.125)
    q[..., 575] = 4
    out, lse = OPS.latent_decode(q, cache, table, _i64(lens), SCALE)
    _check_decode(q, cache, table, lens, 1, out, lse)
    out, lse = OPS.latent_cascade_decode(q, cache, table[3:4], _i64([300]), cache, table, _i64(lens), SCALE)
    x = _rows(cache, table, 3, 300)
    for b, n in enumerate(lens):
        keys = torch.cat([x, _rows(cache, table, b, n)])
        ol.close(out[b], lse.view(-1, heads)[b], ol.attend(q[b], keys, keys[:, :512], 300 + n, SCALE, dtype))


# ---- the forms in fp16 ------------------------------------------------------------------------------------
@pytest.mark.parametrize("q_len,heads", [(2, 16), (3, 40), (7, 8), (5, 128), (40, 3)])
def test_several_tokens_fp16(q_len, heads):
    lens = [0, 1, q_len - 1, q_len, q_len + 1, 32, 33, 200, 2000]
    g = _gen(70 + q_len)
    cache, table = _pool(g, lens, HF)
    q = _randn(g, len(lens) * q_len, heads, 576, dtype=HF)
    out, lse = OPS.latent_decode(q, cache, table, _i64(lens), SCALE, q_len)
    _check_decode(q, cache, table, lens, q_len, out, lse)


@pytest.mark.parametrize("heads,lens", [(16, [9000]), (128, [4097, 0, 1, 5000]), (2, [1300] * 40)])
def test_cut_requests_fp16(heads, lens):
    g = _gen(71)
    cache, table = _pool(g, lens, HF)
    q = _randn(g, len(lens), heads, 576, dtype=HF, scale=3.0)  # peaked: reference points move late
    out, lse = OPS.latent_decode(q, cache, table, _i64(lens), SCALE)
    _check_decode(q, cache, table, lens, 1, out, lse)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("step", [1 / 64, 1.0, 8.0, -8.0])
def test_rising_and_falling_scores(dtype, step):
    """Each pair of tokens passes the one before it (or is passed): by less than the reference point's slack
    at a time, and by more; over a prefix, its parts, and suffixes that go on rising."""
    g = _gen(72)
    lens = [700, 33, 1]
    cache, table = _pool(g, lens, dtype, garbage=False)
    q = torch.zeros(3, 40, 576, dtype=dtype, device=DEV)
    q[..., 575] = 1
    for b, n in enumerate(lens):
        j = torch.arange(n, device=DEV)
        cache.view(-1, 576)[table[b, j // 128].long() * 128 + j % 128, 575] = (step * (j // 2)).to(dtype)
    out, lse = OPS.latent_decode(q, cache, table, _i64(lens), SCALE)
    _check_decode(q, cache, table, lens, 1, out, lse)
    out, lse = OPS.latent_cascade_decode(q, cache, table[:1], _i64(lens[:1]), cache, table, _i64(lens), SCALE)
    x = _rows(cache, table, 0, 700)
    for b, n in enumerate(lens):
        keys = torch.cat([x, _rows(cache, table, b, n)])
        ol.close(out[b], lse.view(3, 40)[b], ol.attend(q[b], keys, keys[:, :512], 700 + n, SCALE, dtype))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("step", [0.25, 3.0, -3.0])
def test_prefill_rising_and_falling_scores(dtype, step):
    g = _gen(73)
    q, k, kr, v = _prompt(g, [300, 40], [300, 400], 2, dtype)
    q[:] = 0
    q[..., 191] = 1
    kr[:, 63] = (torch.arange(700, device=DEV) * step).to(dtype)
    for causal in (True, False):
        out, lse = OPS.latent_prefill(q, k, kr, v, _i64([300, 40]), _i64([300, 400]), SCALE, causal)
        _check_prefill(q, k, kr, v, [300, 40], [300, 400], causal, out, lse)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_wide_fold_of_prefix_and_suffix_parts(dtype):
    """512 blocks of the fold, each with several parts of the prefix and of a cut suffix."""
    g = _gen(74)
    suffix = [2000 if b % 16 == 0 else (37 * b) % 300 for b in range(64)]
    pcache, ptable = _pool(g, [3000], dtype)
    scache, stable = _pool(g, suffix, dtype)
    q = _randn(g, 64, 128, 576, dtype=dtype, scale=2.0)
    out, lse = OPS.latent_cascade_decode(q, pcache, ptable, _i64([3000]), scache, stable, _i64(suffix), SCALE)
    x = _rows(pcache, ptable, 0, 3000)
    for b, n in enumerate(suffix):
        keys = torch.cat([x, _rows(scache, stable, b, n)])
        ol.close(out[b], lse.view(64, 128)[b], ol.attend(q[b], keys, keys[:, :512], 3000 + n, SCALE, dtype))
