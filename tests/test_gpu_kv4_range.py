"""The 4-bit cache's decode where a group's scale decides: values up to the largest that the cache holds, groups that are not
numbers beside borders of units, and scales that keep to one way through the kernels."""
import math

import pytest
import torch

from oracle import kv4 as o4
from oracle.latent import close
from tests.test_gpu_kv4 import BF, DEV, HF, OPS, SCALE, _check_decode, _gen, _i64, _normal, _tables
from tests.test_gpu_kv4_edges import FORMS, _check_cascade, _scales

pytestmark = pytest.mark.gpu


def _check_groups(q, k, v, sees, scale, rows, got, more=0.0):
    """Rows of a kv head against the definition, 32 dims at a time: what large values may lose (2^-32 of the largest of
    them) does not widen the bound of the other dims. more: added to the bound of out."""
    out, lse = got
    if k.shape[0] == 0:
        assert (out == 0).all() and (lse == -math.inf).all()
        return
    for d in range(0, 128, 32):
        o, l, b_o, b_l = o4.attend(q, k, v[:, d:d + 32], sees, scale, q.dtype, rows)
        close(out[:, d:d + 32], lse, (o, l, b_o + more, b_l))


def _check_decode_groups(q, pool, table, lens, scale, q_len, got, more=0.0):
    kv_heads, n = pool.shape[1], q.shape[1] // pool.shape[1]
    q, out, lse = q.view(-1, q_len, kv_heads, n, 128), got[0].view(-1, q_len, kv_heads, n, 128), got[1].view(-1, q_len, kv_heads, n)
    for b, length in enumerate(lens):
        k, v = o4.cached(pool, table[b], length)
        sees = (length - q_len + 1 + torch.arange(q_len, device=DEV)).repeat_interleave(n)
        for h in range(kv_heads):
            _check_groups(q[b, :, h].reshape(-1, 128), k[:, h], v[:, h], sees, scale, q_len * n,
                          (out[b, :, h].reshape(-1, 128), lse[b, :, h].reshape(-1)), more)


def _check_cascade_groups(q, ppool, ptable, prefix, pool, table, suffixes, scale, got):
    kv_heads, n = pool.shape[1], q.shape[1] // pool.shape[1]
    pk, pv = o4.cached(ppool, ptable[0], prefix)
    for b, length in enumerate(suffixes):
        k, v = (torch.cat(x) for x in zip((pk, pv), o4.cached(pool, table[b], length)))
        for h in range(kv_heads):
            hs = slice(h * n, (h + 1) * n)
            _check_groups(q[b, hs], k[:, h], v[:, h], prefix + length, scale, n * len(suffixes),
                          (got[0][b, hs], got[1].view(-1, q.shape[1])[b, hs]))


# ---- groups that are not numbers ------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("q_len,heads,kv_heads,lens", [
    (3, 8, 2, [65, 66, 130, 194]), (16, 1, 1, [65, 79, 70, 143]), (32, 1, 1, [65, 95, 128 + 20, 80]), (3, 14, 2, [65, 66, 130, 194]),
    (40, 2, 1, [70, 102, 134, 66]), (300, 1, 1, [330, 301, 364, 290])])
def test_groups_that_are_not_numbers_beside_a_border(q_len, heads, kv_heads, lens, dtype):
    """The newest tokens begin a unit (or half of one), so that in the one before, not seen whole by the first of them, the
    last see more tokens than it has. A value's group of scale 255 there makes NaN the group's dims, and no others."""
    g = _gen(21)
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    clean = pool.clone()
    bad = [(b, j, grp) for b, n in enumerate(lens) for j, grp in (((n - 1) // 64 * 64 - 60 + b, b), (5, (b + 2) % 4))]
    for b, j, grp in bad:
        pool[table[b, j // 128].long(), kv_heads - 1, o4.places(_i64([j % 128]))[3][0, grp]] = 255
    q = _normal(g, len(lens) * q_len, heads, 128, dtype=dtype)
    out, lse = OPS.kv4_decode(q, pool, table, _i64(lens), SCALE, q_len)
    nan = torch.zeros(len(lens), q_len, kv_heads, heads // kv_heads, 128, dtype=torch.bool, device=DEV)
    for b, j, grp in bad:
        first = max(0, j + q_len - lens[b])  # token t sees lens[b] - q_len + 1 + t keys
        nan[b, first:, -1, :, 32 * grp:32 * grp + 32] = True
    assert torch.equal(out.isnan(), nan.view(out.shape))
    want, _ = OPS.kv4_decode(q, clean, table, _i64(lens), SCALE, q_len)
    _check_decode(q, clean, table, lens, SCALE, q_len, (torch.where(nan.view(out.shape), want, out), lse))


# ---- values of any size ------------------------------------------------------------------------
def _large(pool, how, gen):
    """Value scales: the largest that are written everywhere; of 32 dims only, others ordinary and of about 2^-100; of
    single tokens' groups; around 2^65."""
    def draw(lo, hi, shape):
        return torch.randint(lo, hi + 1, shape, generator=gen, device=DEV, dtype=torch.uint8)
    for u in (0, 8704):
        at = pool[..., u + 8448:u + 8704].unflatten(-1, (4, 64))  # [group][token]
        if how == "all":
            at.copy_(draw(250, 252, at.shape))
        elif how == "one group":
            at.copy_(draw(120, 127, at.shape))
            at[..., 1, :] = 252
            at[..., 3, :] = draw(20, 30, at[..., 3, :].shape)
        elif how == "some tokens":
            some = torch.rand(at.shape, generator=gen, device=DEV) < 0.01
            at.copy_(torch.where(some, draw(200, 252, at.shape), draw(124, 127, at.shape)))
        else:
            at.copy_(draw(189, 194, at.shape))


@pytest.mark.parametrize("q_len,heads,kv_heads", FORMS)
@pytest.mark.parametrize("how", ["all", "one group", "some tokens", "border"])
def test_values_up_to_the_largest(how, q_len, heads, kv_heads):
    """A mean of finite values is finite, however large they are and however many."""
    g = _gen(22)
    lens = [1, 2, 64, 300, 3000, 0, 129]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    _large(pool, how, g)
    q = _normal(g, len(lens) * q_len, heads, 128)
    _check_decode_groups(q, pool, table, lens, SCALE, q_len, OPS.kv4_decode(q, pool, table, _i64(lens), SCALE, q_len))
    if q_len == 1:
        other = o4.random_pool(g, blocks, kv_heads, DEV)
        for a, b in ((pool, other), (other, pool), (pool, pool)):
            for prefix in (4, 3):
                got = OPS.kv4_cascade_decode(q, a, table[prefix:prefix + 1], _i64([lens[prefix]]), b, table, _i64(lens), SCALE)
                _check_cascade_groups(q, a, table[prefix:prefix + 1], lens[prefix], b, table, lens, SCALE, got)


@pytest.mark.parametrize("q_len,heads,kv_heads", FORMS)
@pytest.mark.parametrize("first", [0, 40])
def test_tiny_values_in_the_dims_of_large_ones(first, q_len, heads, kv_heads):
    """Beside a scale of 2^65 and more those below 2^-79 (byte 48) count as that: a value of at most 6 * 2^-80 is taken as at most
    6 * 2^-79, so that it, and a mean of such, is off by less than 2^-76. Where a large value's code is 0 a dim holds nothing else."""
    g = _gen(25)
    lens = [40, 200, 1000]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    for u in (0, 8704):
        at = pool[..., u + 8448:u + 8704].unflatten(-1, (4, 64))
        some = torch.rand(at.shape, generator=g, device=DEV) < 0.01
        low = torch.randint(max(8, first), first + 16, at.shape, generator=g, device=DEV, dtype=torch.uint8)
        at.copy_(torch.where(some, 252, low))
    q = _normal(g, len(lens) * q_len, heads, 128)
    _check_decode_groups(q, pool, table, lens, SCALE, q_len, OPS.kv4_decode(q, pool, table, _i64(lens), SCALE, q_len), 2.0 ** -76)


@pytest.mark.parametrize("q_len,heads,kv_heads", FORMS)
@pytest.mark.parametrize("step", [1 / 16, 1.0, 8.0, -8.0])
def test_large_values_and_rising_scores(step, q_len, heads, kv_heads):
    """Weights far above the reference point's, and the point moving, with sums near the largest numbers; what was written
    from the largest 16-bit values."""
    g = _gen(23)
    lens = [1500, 300, 70, 33]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    for b, n in enumerate(lens):
        j = torch.arange(n, device=DEV)
        k = torch.zeros(n, kv_heads, 128, device=DEV)
        k[..., 77] = (step * (j // 4))[:, None]
        v = torch.where(torch.rand(n, kv_heads, 128, generator=g, device=DEV) < 0.8, 1.0, -1.0) * torch.finfo(BF).max
        OPS.kv4_cache_write(k.to(BF), v.to(BF), table[b].long()[j // 128] * 128 + j % 128, pool)
    q = _normal(g, len(lens) * q_len, heads, 128)
    q[..., 77] = 1
    _check_decode_groups(q, pool, table, lens, 0.5, q_len, OPS.kv4_decode(q, pool, table, _i64(lens), 0.5, q_len))
    if q_len == 1:
        got = OPS.kv4_cascade_decode(q, pool, table[:1], _i64([1500]), pool, table, _i64(lens), 0.5)
        _check_cascade_groups(q, pool, table[:1], 1500, pool, table, lens, 0.5, got)


# ---- scales that fp16 holds, all of them ----------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("q_len,heads,kv_heads", FORMS)
@pytest.mark.parametrize("key,value", [(107, 107), (113, 113), (110, 135), (135, 110), (135, 135), (120, 104)])
def test_scales_at_the_borders_of_fp16(key, value, q_len, heads, kv_heads, dtype):
    """Every scale byte is in [104, 135], where the forms of more than 16 rows hold values (and an fp16 query's keys) in
    fp16: its subnormal numbers (up to byte 112) and the largest scales, with no unit that takes another way."""
    g = _gen(24)
    lens = [700, 64, 33, 5, 2000]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    _scales(pool, ((key, min(3, key - 104)), (value, min(3, value - 104))), gen=g)
    q = _normal(g, len(lens) * q_len, heads, 128, dtype=dtype)
    scale = SCALE * 2.0 ** (127 - key)
    got = OPS.kv4_decode(q, pool, table, _i64(lens), scale, q_len)
    if dtype == HF and value == 135:  # up to 6 * 2^8 a value: inside fp16's range
        assert math.isfinite(got[0].abs().max().item())
    _check_decode(q, pool, table, lens, scale, q_len, got)
    if q_len == 1:
        got = OPS.kv4_cascade_decode(q, pool, table[:1], _i64([700]), pool, table, _i64(lens), scale)
        _check_cascade(q, pool, table[:1], 700, pool, table, lens, scale, got, dtype)
