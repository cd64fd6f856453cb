"""Every unit of a long or cut list of the 4-bit decode is read once, by exact counts, where a lost unit is far within the
bounds of ordinary inputs; and calls that run beside each other on two streams."""
import math

import pytest
import torch

from oracle import kv4 as o4
from oracle.latent import close
from tests.test_gpu_kv4 import BF, DEV, HF, OPS, SCALE, _gen, _i64, _normal, _tables

pytestmark = pytest.mark.gpu


def _marked(gen, lens, kv_heads, scale):
    """A pool whose values are 0 but for a 1 (times 2^(scale - 127)) in one dim of a unit's tokens in one kv head: unit u of a
    request has it in head u % kv_heads, dim u / kv_heads % 128. Its table too."""
    table, blocks = _tables(gen, lens)
    pool = torch.zeros(blocks, kv_heads, o4.PAGE_BYTES, dtype=torch.uint8, device=DEV)
    for at in (8192, 8704 + 8192):
        pool[..., at:at + 256] = 127
        pool[..., at + 256:at + 512] = scale
    codes = o4.places(torch.arange(128, device=DEV))[1].view(2, 64, 64)  # [unit of the page][token][byte]
    for b, n in enumerate(lens):
        u = torch.arange(-(-n // 64), device=DEV)
        head, dim = u % kv_heads, u // kv_heads % 128
        at = codes[u % 2, :, dim // 2]  # [unit][token]
        pool[table[b].long()[u // 2][:, None], head[:, None], at] = (2 << 4 * (dim % 2)).to(torch.uint8)[:, None]
    return pool, table


def _counted(n, head, kv_heads, scale, dtype):
    """(o, lse, bounds) of a row that sees n tokens. With q = 0 every p is one power of two, so that sums of p and of p v are
    whole multiples of it below 2^24: exact. o then passes the joints of its parts, each some roundings, of at most 64 in a
    row, and rounds to its type. lse is ln 2 (log2(sum) + m), log2 good to a step of its result and m >= -7."""
    u = torch.arange(-(-n // 64), device=DEV)
    tokens = torch.where(u % kv_heads == head, (n - 64 * u).clamp(max=64), 0).double()
    o = torch.zeros(128, dtype=torch.float64, device=DEV)
    o.index_add_(0, u // kv_heads % 128, tokens)
    if n == 0:
        z = torch.zeros(1, dtype=torch.float64, device=DEV)
        return o[None], torch.log(z), o[None], z
    o = o / n * 2.0 ** (scale - 127)
    step = 2.0 ** (math.floor(math.log2(math.log2(n) + 7)) - 23)
    lse = torch.full((1,), math.log(n), dtype=torch.float64, device=DEV)
    b_l = math.log(2) * 1.5 * step + 2 * o4.F32 * lse
    return o[None], lse, (torch.finfo(dtype).eps / 2 + 64 * o4.F32) * o[None], b_l


def _check(out, lse, lens, q_len, kv_heads, scale, dtype):
    out, lse = out.view(len(lens), q_len, kv_heads, -1, 128), lse.view(len(lens), q_len, kv_heads, -1)
    for b, n in enumerate(lens):
        for t in {0, q_len // 2, q_len - 1}:
            for h in range(kv_heads):
                ref = _counted(max(0, n - q_len + 1 + t), h, kv_heads, scale, dtype)
                rows = out.shape[3]
                close(out[b, t, h], lse[b, t, h], tuple(x.expand(rows, *x.shape[1:]) for x in ref))


# up to 16 rows a kv head, up to 32, more; single tokens and several, one request and many
COUNTS = [
    (1, 8, 8, [9000]), (1, 64, 2, [5000, 0, 1, 4097]), (1, 20, 1, [3000, 64, 65]), (3, 16, 2, [20011, 2, 777, 0]),
    (1, 128, 2, [5000, 0, 1, 4097]), (1, 64, 1, [1300] * 40), (5, 16, 2, [31 + 97 * b for b in range(60)]),
    (7, 8, 1, [64] * 300), (40, 2, 1, [5000, 4999, 33]), (300, 2, 1, [9011, 300, 40]), (5, 64, 8, [64] * 64),
]


@pytest.mark.parametrize("dtype,scale", [(BF, 127), (HF, 127), (BF, 252)])
@pytest.mark.parametrize("q_len,heads,kv_heads,lens", COUNTS, ids=lambda x: str(x)[:24])
def test_counts(q_len, heads, kv_heads, lens, dtype, scale):
    pool, table = _marked(_gen(31), lens, kv_heads, scale)
    q = torch.zeros(len(lens) * q_len, heads, 128, dtype=dtype, device=DEV)
    out, lse = OPS.kv4_decode(q, pool, table, _i64(lens), SCALE, q_len)
    _check(out, lse, lens, q_len, kv_heads, scale, dtype)


@pytest.mark.parametrize("scale", [127, 252])
def test_counts_of_long_lists(scale):
    """75 units to a wave, which takes 64 at a time, in every form. The lse tells a unit more or less of 19200; of the
    19 units of a head that mark a dim, one missing or another's in its place moves the dim by 5%."""
    kv_heads, n = 8, 19200 * 64 - 37
    pool, table = _marked(_gen(32), [n], kv_heads, scale)
    for dtype in (BF, HF) if scale == 127 else (BF,):
        for group in (1, 20, 40):
            q = torch.zeros(1, group * kv_heads, 128, dtype=dtype, device=DEV)
            out, lse = OPS.kv4_decode(q, pool, table, _i64([n]), SCALE)
            _check(out, lse, [n], 1, kv_heads, scale, dtype)


@pytest.mark.parametrize("dtype,scale", [(BF, 127), (HF, 127), (BF, 252)])
@pytest.mark.parametrize("batch,heads,kv_heads,prefix,suffix", [
    (8, 32, 8, 2048, 256), (3, 4, 1, 9000, 100), (64, 32, 8, 8192, 300), (117, 16, 2, 5000, 70), (5, 40, 2, 3001, 200), (9, 160, 8, 0, 200)])
def test_counts_of_a_shared_prefix(batch, heads, kv_heads, prefix, suffix, dtype, scale):
    """The prefix marks dims as its units, the suffixes count as a request of their own."""
    lens = [suffix * (i % 5) // 4 for i in range(batch)]
    pool, both = _marked(_gen(33), [prefix] + lens, kv_heads, scale)
    q = torch.zeros(batch, heads, 128, dtype=dtype, device=DEV)
    out, lse = OPS.kv4_cascade_decode(q, pool, both[:1].contiguous(), _i64([prefix]), pool, both[1:].contiguous(), _i64(lens), SCALE)
    out, lse = out.view(batch, kv_heads, -1, 128), lse.view(batch, kv_heads, -1)
    for b, n in enumerate(lens):
        for h in range(kv_heads):
            a, s = (_counted(x, h, kv_heads, scale, dtype) for x in (prefix, n))
            _, l, _, b_l = _counted(prefix + n, h, kv_heads, scale, dtype)
            o = (a[0] * prefix + s[0] * n) / max(1, prefix + n)
            rows = out.shape[2]
            ref = o, l, (torch.finfo(dtype).eps / 2 + 64 * o4.F32) * o, b_l
            close(out[b, h], lse[b, h], tuple(x.expand(rows, *x.shape[1:]) for x in ref))


def test_two_streams_beside_each_other():
    """Calls that wait behind long work on two streams and then run beside each other, nothing copied or made between them,
    give what one alone gives, bit for bit."""
    g = _gen(34)
    lens = [3000, 17, 900, 0]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, 2, DEV)
    kv, ptable, plen = _i64(lens), table[:1].contiguous(), _i64([3000])
    qs = [_normal(g, 4, heads, 128) for heads in (16, 64, 128)]
    calls = [c for q in qs for c in (lambda q=q: OPS.kv4_decode(q, pool, table, kv, SCALE),
                                     lambda q=q: OPS.kv4_cascade_decode(q, pool, ptable, plen, pool, table, kv, SCALE))]
    want = [c() for c in calls]
    x = torch.randn(4096, 4096, device=DEV).to(BF)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for r in range(3):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                for _ in range(40):  # some ms
                    x @ x
        for i in range(8 * len(calls)):
            with torch.cuda.stream(streams[i % 2]):
                got.append(calls[(i // 2 + i % 2 * r) % len(calls)]())
        torch.cuda.synchronize()
        for i, (o, l) in enumerate(got):
            w = want[(i // 2 + i % 2 * r) % len(calls)]
            assert torch.equal(o, w[0]) and torch.equal(l, w[1]), (r, i)
