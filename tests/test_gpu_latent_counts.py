"""Every tile of a long or cut call of the latent decode and prefill is read once: exact counts
(oracle/latent.py), at lengths where a lost tile is far within the bounds of ordinary inputs."""
import pytest
import torch

from oracle import latent as ol
from tests.test_gpu_latent import BF, DEV, HF, OPS, SCALE, _gen, _i64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import cascade_amd  # noqa: F401
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible to torch")


def _marked(lens, dtype, seed, first_tile=0):
    """A pool of the lens' marked tokens in shuffled pages, and its table."""
    need = [-(-n // 128) for n in lens]
    order = torch.randperm(max(1, sum(need)), generator=_gen(seed), device=DEV)
    cache = torch.empty(order.numel(), 128, 576, dtype=dtype, device=DEV)
    table = torch.zeros(len(lens), max(need + [1]), dtype=torch.int32, device=DEV)
    at = 0
    for b, k in enumerate(need):
        pages = order[at:at + k]
        table[b, :k] = pages.int()
        for lo in range(0, k, 512):  # in parts: the index of a whole long request is large
            rows = torch.empty(min(512, k - lo) * 128, 576, dtype=dtype, device=DEV)
            ol.mark(rows, first_tile + lo * (128 // ol.TILE))
            cache[pages[lo:lo + 512]] = rows.view(-1, 128, 576)
        at += k
    return cache, table


def _check(out, lse, want):
    """Rows [rows, 512] and their lse, all of one count."""
    o, l, b_o, b_l = want
    n = out.shape[0]
    ol.close(out, lse, (o.expand(n, -1), l.expand(n), b_o.expand(n, -1), b_l.expand(n)))


@pytest.mark.parametrize("dtype,q_len,heads,lens", [
    (HF, 1, 16, [9000]),
    (BF, 1, 16, [9000]),
    (HF, 1, 128, [4097, 0, 1, 5000]),
    (HF, 1, 2, [1300] * 40),
    (BF, 1, 40, [31 + 97 * b for b in range(60)]),
    (HF, 3, 40, [20000, 2, 3, 777, 0]),
    (HF, 7, 20, [5000, 4999, 33]),
    (HF, 300, 1, [20011, 300, 40]),     # 75 row tiles: 3 workgroups for each, their lists of several phases
    (HF, 1100, 1, [9000, 700]),         # more row tiles than workgroups
    (BF, 1, 8, [7] * 700 + [3000]),
])
def test_decode_counts(dtype, q_len, heads, lens):
    cache, table = _marked(lens, dtype, len(lens) + heads)
    q = torch.zeros(len(lens) * q_len, heads, 576, dtype=dtype, device=DEV)
    out, lse = OPS.latent_decode(q, cache, table, _i64(lens), SCALE, q_len)
    lse = lse.view(-1, heads)
    for b, n in enumerate(lens):
        for i in range(q_len):
            t = b * q_len + i
            _check(out[t], lse[t], ol.counted(ol.whole(max(0, n - q_len + 1 + i), DEV), dtype))


def test_decode_counts_of_a_long_list():
    """280 tiles a workgroup: more than are described at a time. 2.6 GB of cache."""
    n = 2293777
    cache, table = _marked([n], HF, 3)
    out, lse = OPS.latent_decode(torch.zeros(1, 16, 576, dtype=HF, device=DEV), cache, table, _i64([n]), SCALE)
    _check(out[0], lse, ol.counted(ol.whole(n, DEV), HF))
    # as two requests and their rows of several tokens
    lens = [n - 1000001, 1000001]
    two = torch.zeros(2, table.shape[1], dtype=torch.int32, device=DEV)
    pages = -(-lens[0] // 128)
    two[0, :pages] = table[0, :pages]
    two[1, :-(-lens[1] // 128)] = table[0, :-(-lens[1] // 128)]
    out, lse = OPS.latent_decode(torch.zeros(4, 70, 576, dtype=HF, device=DEV), cache, two, _i64(lens), SCALE, 2)
    lse = lse.view(4, 70)
    for t in range(4):
        _check(out[t], lse[t], ol.counted(ol.whole(lens[t // 2] - 1 + t % 2, DEV), HF))


@pytest.mark.parametrize("dtype,prefix,batch,heads,suffix", [
    (HF, 20000, 2, 7, [65, 0]),
    (BF, 20000, 2, 7, [65, 0]),
    (HF, 8192, 64, 32, [(311 * b) % 1025 for b in range(64)]),
    (HF, 20000, 117, 128, [(37 * b) % 90 for b in range(117)]),  # units longer than described at once
    (HF, 600, 300, 128, [40] * 300),
    (BF, 4097, 40, 16, [0] * 40),
    (HF, 16001, 1, 16, [9000]),
    (HF, 300001, 5, 16, [1, 0, 40, 5000, 33]),
])
def test_cascade_counts(dtype, prefix, batch, heads, suffix):
    pcache, ptable = _marked([prefix], dtype, batch)
    behind = -(-prefix // ol.TILE)  # the suffix's tiles are named after the prefix's
    scache, stable = _marked(suffix, dtype, heads, behind)
    q = torch.zeros(batch, heads, 576, dtype=dtype, device=DEV)
    out, lse = OPS.latent_cascade_decode(q, pcache, ptable, _i64([prefix]), scache, stable, _i64(suffix), SCALE)
    lse = lse.view(batch, heads)
    of = {}
    for b, n in enumerate(suffix):
        if n not in of:
            of[n] = ol.counted(torch.cat([ol.whole(prefix, DEV), ol.whole(n, DEV)]), dtype)
        _check(out[b], lse[b], of[n])


@pytest.mark.parametrize("dtype,heads,causal,ql,kl", [
    (HF, 2, True, [6000], [6000]),
    (HF, 3, True, [32], [8000]),              # a short continuation of a long context
    (BF, 1, False, [1, 300], [20000, 4097]),
    (HF, 2, True, [257, 0, 900, 33], [5000, 64, 900, 16]),
    (HF, 1, False, [70], [131]),
])
def test_prefill_counts(dtype, heads, causal, ql, kl):
    """Every key a query sees is counted once. Value dims: the tile of 64 keys mod 64, and its number / 64."""
    q = torch.zeros(sum(ql), heads, 192, dtype=dtype, device=DEV)
    k, kr = torch.ones(sum(kl), heads, 128, dtype=dtype, device=DEV), torch.ones(sum(kl), 64, dtype=dtype, device=DEV)
    tiles = [torch.arange(n, device=DEV) // 64 for n in kl]
    marks = torch.cat([torch.nn.functional.one_hot(t % 64, 64) for t in tiles]), \
        torch.cat([torch.nn.functional.one_hot(t // 64, 64) for t in tiles])
    v = torch.cat(marks, 1)[:, None].expand(-1, heads, -1).to(dtype)
    out, lse = OPS.latent_prefill(q, k, kr, v, _i64(ql), _i64(kl), SCALE, causal)
    lse, qa = lse.view(-1, heads), 0
    for n, m in zip(ql, kl):
        if n == 0:
            continue
        i = torch.arange(n, device=DEV)
        sees = (m - n + 1 + i).clamp(0, m) if causal else torch.full((n,), m, device=DEV)
        tile = torch.arange(-(-m // 64), device=DEV)
        tokens = (sees[:, None] - 64 * tile).clamp(0, 64).double()
        names = torch.cat([torch.nn.functional.one_hot(tile % 64, 64), torch.nn.functional.one_hot(tile // 64, 64)], 1)
        o = tokens @ names.double() / sees.clamp_min(1)[:, None]
        # the bounds depend on how many tokens were read, not on where
        b_l = torch.stack([ol.counted(x[None], dtype)[3] for x in sees])
        for h in range(heads):
            ol.close(out[qa:qa + n, h], lse[qa:qa + n, h], (o, torch.log(sees.double()), (ol.unit(dtype) + 4 * ol.F32) * o, b_l))
        qa += n
