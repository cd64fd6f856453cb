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
