"""The 4-bit K/V cache operators on the GPU against the format and formulas in 64 bits."""
import math

import pytest
import torch

import cascade_amd  # noqa: F401
from oracle import kv4 as o4
from oracle.latent import close

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
OPS = torch.ops.npu
BF, HF = torch.bfloat16, torch.float16
SCALE = 128 ** -0.5


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(gen, *shape, dtype=BF, std=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * std).to(dtype)


def _i64(x):
    return torch.tensor(x, dtype=torch.int64, device=DEV)


# ---- write and read -----------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,kv_heads,blocks", [(1, 1, 1), (5, 3, 2), (64, 8, 9), (300, 2, 4), (1025, 5, 11)])
def test_write_is_exact(tokens, kv_heads, blocks, dtype):
    """Every byte of the pool: those of the tokens written, and the others as they were."""
    g = _gen(tokens)
    pool = torch.randint(0, 256, (blocks, kv_heads, o4.PAGE_BYTES), generator=g, device=DEV, dtype=torch.uint8)
    std = torch.exp(torch.randn(tokens, kv_heads, 1, generator=g, device=DEV) * 3)
    k, v = (_normal(g, tokens, kv_heads, 128, dtype=torch.float32) * std for _ in range(2))
    k, v = k.to(dtype), v.to(dtype)
    slots = torch.randperm(blocks * 128, generator=g, device=DEV)[:tokens]
    want = o4.write(pool, k, v, slots)
    OPS.kv4_cache_write(k, v, slots, pool)
    assert torch.equal(pool, want)


def test_write_of_neighbouring_slots():
    """A prompt's tokens, beginning inside a page, rows in a wider matrix; padded with -1 and past the pool."""
    g = _gen(3)
    qkv = _normal(g, 200, 14, 128)
    k, v = qkv[:, 3:5], qkv[:, 9:13:2]
    slots = torch.arange(200, device=DEV) + 37
    slots[150:] = -1
    slots[160:] = 3 * 128
    slots[170:] = 2 ** 62
    pool = torch.zeros(3, 2, o4.PAGE_BYTES, device=DEV, dtype=torch.uint8)
    want = o4.write(pool, k, v, slots)
    OPS.kv4_cache_write(k, v, slots, pool)
    assert torch.equal(pool, want)


def _slots(gen, how, tokens, blocks):
    """Slots of many tokens: anywhere; a prompt from inside a page on, over scattered pages; prompts of other
    alignments one after another, padded with -1 and slots past the pool, the last pages among them."""
    perm = torch.randperm(blocks, generator=gen, device=DEV)
    j = torch.arange(tokens, device=DEV)
    if how == "anywhere":
        return torch.randperm(blocks * 128, generator=gen, device=DEV)[:tokens]
    if how == "prompt":
        return perm[(j + 37) // 128] * 128 + (j + 37) % 128
    parts, at, page = [], 0, 0
    for n, first in ((517, 0), (3, 127), (1, 5), (700, 8), (64, 64), (9, 3), (tokens, 121)):
        n = min(n, tokens - at)
        i = torch.arange(n, device=DEV) + first
        parts.append(perm[page + i // 128] * 128 + i % 128)
        at, page = at + n, page + -(-(n + first) // 128)
    slots = torch.cat(parts)
    slots[100:103], slots[600], slots[-1] = -1, blocks * 128, -9
    return slots


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("how", ["anywhere", "prompt", "mixed"])
@pytest.mark.parametrize("tokens,kv_heads", [(2049, 4), (6144, 8), (16385, 3)])
def test_write_and_read_of_many_tokens(tokens, kv_heads, how, dtype):
    """From 49152 rows on, eight neighbouring tokens are moved together."""
    g = _gen(tokens)
    blocks = tokens // 128 + 12
    slots = _slots(g, how, tokens, blocks)
    pool = torch.randint(0, 256, (blocks, kv_heads, o4.PAGE_BYTES), generator=g, device=DEV, dtype=torch.uint8)
    kv = _normal(g, tokens, 2 * kv_heads, 136, dtype=dtype)[..., :128]
    k, v = kv[:, :kv_heads], kv[:, kv_heads:]
    want = o4.write(pool, k, v, slots)
    OPS.kv4_cache_write(k, v, slots, pool)
    assert torch.equal(pool, want)
    for order in (slots, slots.flip(0).contiguous()):
        for got, ref in zip(OPS.kv4_cache_read(pool, order, dtype), o4.read(pool, order)):
            assert torch.equal(got.double().nan_to_num(7), ref.to(torch.float32).to(dtype).double().nan_to_num(7))


@pytest.mark.parametrize("dtype", [BF, HF])
def test_write_of_special_values(dtype):
    """Each group of one kind: ties, borders of the scale, the type's largest and least numbers, zeros, values
    that are not finite."""
    most, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    halves = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]
    groups = [halves + [-x for x in halves], [7.0, 6.0, -0.25], [7.0625, 3.5, 0.5], [most, -most, most / 2],
              [tiny, tiny / 2, -tiny], [0.0, -0.0], [math.inf, 1.0], [1.0, -math.inf], [math.nan, 2.0], [1.0],
              [1e-30 if dtype == BF else 2.0 ** -24, 0.0], [2.0, -1e-3, 1e-4]]
    x = torch.zeros(len(groups), 32)
    for i, grp in enumerate(groups):
        x[i, :len(grp)] = torch.tensor(grp)
    x = x.reshape(-1, 1, 128).to(dtype).to(DEV)
    pool = torch.zeros(1, 1, o4.PAGE_BYTES, device=DEV, dtype=torch.uint8)
    slots = torch.arange(x.shape[0], device=DEV) * 9
    want = o4.write(pool, x, x.flip(0).contiguous(), slots)
    OPS.kv4_cache_write(x, x.flip(0).contiguous(), slots, pool)
    assert torch.equal(pool, want)
    k, v = OPS.kv4_cache_read(pool, slots, dtype)
    for got, ref in zip((k, v), o4.read(pool, slots)):
        assert torch.equal(got.isnan(), ref.isnan())
        assert torch.equal(got.nan_to_num(0), ref.to(torch.float32).to(dtype).nan_to_num(0))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,kv_heads", [(1, 1), (77, 3), (512, 8)])
def test_read_is_exact(tokens, kv_heads, dtype):
    """Any bytes, all scale bytes among them; slots in any order, twice the same, and outside the pool."""
    g = _gen(tokens)
    pool = torch.randint(0, 256, (6, kv_heads, o4.PAGE_BYTES), generator=g, device=DEV, dtype=torch.uint8)
    slots = torch.randint(0, 6 * 128, (tokens,), generator=g, device=DEV)
    slots[tokens // 2::7] = -1
    slots[tokens // 3 + 1::11] = 6 * 128
    k, v = OPS.kv4_cache_read(pool, slots, dtype)
    assert k.dtype == v.dtype == dtype and k.shape == (tokens, kv_heads, 128)
    for got, ref in zip((k, v), o4.read(pool, slots)):
        ref = ref.to(torch.float32).to(dtype)  # float32 holds every value, subnormal ones too
        assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got.nan_to_num(0), ref.nan_to_num(0))


# ---- attention ----------------------------------------------------------------------
def _tables(gen, lens, spare=1):
    """Scattered pages for the lengths: (block table int32, number of pages)."""
    pages = [max(1, -(-n // 128)) for n in lens]
    total = sum(pages) + spare
    perm = torch.randperm(total, generator=gen, device=DEV)
    table = torch.zeros(len(lens), max(pages), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, total


def _check_decode(q, pool, table, lens, scale, q_len, got):
    out, lse = got
    heads, kv_heads = q.shape[1], pool.shape[1]
    grp = heads // kv_heads
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (q.shape[0] * heads,)
    out, lse = out.view(-1, q_len, kv_heads, grp, 128), lse.view(-1, q_len, kv_heads, grp)
    rows = q.view(-1, q_len, kv_heads, grp, 128)
    for b, n in enumerate(lens):
        k, v = o4.cached(pool, table[b], n)
        sees = (n - q_len + 1 + torch.arange(q_len, device=DEV)).repeat_interleave(grp)
        for h in range(kv_heads):
            ref = o4.attend(rows[b, :, h].reshape(-1, 128), k[:, h], v[:, h], sees, scale, q.dtype, q_len * grp)
            close(out[b, :, h].reshape(-1, 128), lse[b, :, h].reshape(-1), ref)


DECODES = [  # batch lengths, q_len, heads, kv_heads
    ([1], 1, 1, 1), ([64], 1, 4, 1), ([65, 63, 128, 129, 1], 1, 8, 2), ([1300], 1, 32, 8), ([0, 5, 0, 700, 0], 1, 5, 5),
    ([333, 1, 2, 1000], 3, 16, 2), ([100, 3000], 2, 16, 1), ([2, 1, 0, 65], 5, 28, 4), ([500] * 3, 7, 20, 4),
    ([257, 64], 40, 8, 2), ([40 + 13 * i for i in range(70)], 1, 8, 2), ([9000, 20], 1, 14, 2), ([7] * 300, 1, 2, 1),
    ([64 * i % 777 for i in range(513)], 1, 6, 3), ([20000], 1, 128, 8), ([300, 4000, 64], 1, 64, 1)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens,q_len,heads,kv_heads", DECODES, ids=lambda x: str(x)[:24])
def test_decode(lens, q_len, heads, kv_heads, dtype):
    g = _gen(len(lens) + heads)
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    q = _normal(g, len(lens) * q_len, heads, 128, dtype=dtype)
    got = OPS.kv4_decode(q, pool, table, _i64(lens), SCALE, q_len)
    torch.cuda.synchronize()
    _check_decode(q, pool, table, lens, SCALE, q_len, got)


CASCADES = [  # prefix, suffixes, heads, kv_heads
    (1, [1], 1, 1), (0, [5, 0], 4, 2), (300, [0, 0, 0], 8, 8), (0, [0], 2, 1), (2048, [256, 1, 130, 64, 0, 77, 300, 2], 32, 8),
    (129, [10 * i for i in range(33)], 8, 1), (1000, [3] * 100, 14, 2), (5000, [700, 90], 64, 8), (640, [50] * 17, 16, 16)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("prefix,suffixes,heads,kv_heads", CASCADES, ids=lambda x: str(x)[:24])
def test_cascade(prefix, suffixes, heads, kv_heads, dtype):
    g = _gen(prefix + heads)
    both, blocks = _tables(g, [prefix] + suffixes)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    q = _normal(g, len(suffixes), heads, 128, dtype=dtype)
    ptable, table = both[:1].contiguous(), both[1:].contiguous()
    out, lse = OPS.kv4_cascade_decode(q, pool, ptable, _i64([prefix]), pool, table, _i64(suffixes), SCALE)
    torch.cuda.synchronize()
    grp = heads // kv_heads
    pk, pv = o4.cached(pool, ptable[0], prefix)
    for b, n in enumerate(suffixes):
        k, v = o4.cached(pool, table[b], n)
        k, v = torch.cat([pk, k]), torch.cat([pv, v])
        for h in range(kv_heads):
            hs = slice(h * grp, (h + 1) * grp)
            ref = o4.attend(q[b, hs], k[:, h], v[:, h], prefix + n, SCALE, dtype, grp * len(suffixes))
            close(out[b, hs], lse.view(-1, heads)[b, hs], ref)
