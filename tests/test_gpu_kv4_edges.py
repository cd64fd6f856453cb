"""The 4-bit cache's operators at their edges, against the 64-bit definition: what hidden places hold, scales of
any size, scores that rise, bad pages and lengths, long lists, large pools, streams, graphs, and together."""
import ctypes
import math

import pytest
import torch

from cascade_amd import abi
from oracle import kv4 as o4
from oracle.latent import close
from tests.test_gpu_kv4 import BF, DEV, HF, OPS, SCALE, _check_decode, _gen, _i64, _normal, _tables

pytestmark = pytest.mark.gpu

# (q_len, heads, kv_heads): up to 16 rows a kv head, up to 32, more; one token and several
FORMS = [(1, 8, 2), (3, 8, 2), (1, 24, 1), (3, 14, 2), (1, 64, 1), (7, 24, 3)]


def _scales(pool, base, spread=3, gen=None):
    """Scale bytes of keys and values in [base - spread, base]."""
    for at, (b, s) in zip((8192, 8448), base if isinstance(base, tuple) else ((base, spread),) * 2):
        for u in (0, 8704):
            pool[..., u + at:u + at + 256] = torch.randint(b - s, b + 1, (*pool.shape[:2], 256), generator=gen, device=DEV,
                                                           dtype=torch.uint8)


def _spoil(pool, table, lens, gen):
    """Tokens behind the lengths hold anything, scales of 255 among them."""
    for b, n in enumerate(lens):
        slots = torch.arange(n, max(1, -(-n // 128)) * 128, device=DEV)
        if slots.numel() == 0:
            continue
        page = table[b].long()[slots // 128][:, None]
        for i, at in enumerate(o4.places(slots)):
            for h in range(pool.shape[1]):
                x = torch.randint(0, 256, at.shape, generator=gen, device=DEV, dtype=torch.uint8)
                if i > 1:
                    x[torch.rand(at.shape, generator=gen, device=DEV) < 0.5] = 255
                pool[page, h, at] = x


def _check_cascade(q, ppool, ptable, prefix, pool, table, suffixes, scale, got, dtype):
    out, lse = got
    heads, kv_heads = q.shape[1], pool.shape[1]
    grp = heads // kv_heads
    pk, pv = o4.cached(ppool, ptable[0], prefix)
    for b, n in enumerate(suffixes):
        k, v = o4.cached(pool, table[b], n)
        k, v = torch.cat([pk, k]), torch.cat([pv, v])
        for h in range(kv_heads):
            hs = slice(h * grp, (h + 1) * grp)
            ref = o4.attend(q[b, hs], k[:, h], v[:, h], prefix + n, scale, dtype, grp * len(suffixes))
            close(out[b, hs], lse.view(-1, heads)[b, hs], ref)


# ---- what a row does not see ---------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("q_len,heads,kv_heads", FORMS)
def test_tokens_behind_a_length_may_hold_anything(q_len, heads, kv_heads, dtype):
    g = _gen(1)
    lens = [1, 31, 32, 33, 63, 64, 65, 100, 127, 0, 2000, 129, 3]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    _spoil(pool, table, lens, g)
    q = _normal(g, len(lens) * q_len, heads, 128, dtype=dtype)
    _check_decode(q, pool, table, lens, SCALE, q_len, OPS.kv4_decode(q, pool, table, _i64(lens), SCALE, q_len))
    if q_len == 1:
        got = OPS.kv4_cascade_decode(q, pool, table[7:8], _i64([100]), pool, table, _i64(lens), SCALE)
        _check_cascade(q, pool, table[7:8], 100, pool, table, lens, SCALE, got, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("q_len,heads,kv_heads", FORMS)
@pytest.mark.parametrize("what", ["key", "value"])
def test_groups_that_are_not_numbers(what, q_len, heads, kv_heads, dtype):
    """A group of scale 255 in a token makes NaN what sees it (of a value: in the group's dims) and nothing else:
    here one token that all rows see, and one of the newest, which not all tokens of the request see."""
    g = _gen(2)
    lens = [300, 300, 40, 64]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    clean = pool.clone()
    bad = {0: (17, 1), 1: (299, 2), 3: (64 - min(q_len, 2), 3)}  # request: token, group
    for b, (j, grp) in bad.items():
        at = o4.places(_i64([j % 128]))[2 if what == "key" else 3][0, grp]
        pool[table[b, j // 128].long(), kv_heads - 1, at] = 255
    q = _normal(g, len(lens) * q_len, heads, 128, dtype=dtype)
    out, lse = OPS.kv4_decode(q, pool, table, _i64(lens), SCALE, q_len)
    n = heads // kv_heads
    o, l = out.view(4, q_len, kv_heads, n, 128), lse.view(4, q_len, kv_heads, n)
    nan = torch.zeros(o.shape, dtype=torch.bool, device=DEV)
    for b, (j, grp) in bad.items():
        for t in range(q_len):
            if lens[b] - q_len + 1 + t > j:
                nan[b, t, -1, :, slice(None) if what == "key" else slice(32 * grp, 32 * grp + 32)] = True
    assert torch.equal(o.isnan(), nan)
    assert torch.equal(l.isnan(), nan.all(-1))
    want, wl = OPS.kv4_decode(q, clean, table, _i64(lens), SCALE, q_len)
    _check_decode(q, clean, table, lens, SCALE, q_len, (want, wl))
    # the rest: the groups that hold NaN leave the rows and dims beside them as they were, up to a half unit's
    # other form for more than 16 rows (P then within 2^-17 instead of 2^-11)
    fixed = torch.where(nan.view(out.shape), want, out), torch.where(nan.all(-1).view(-1), wl, lse)
    _check_decode(q, clean, table, lens, SCALE, q_len, fixed)


@pytest.mark.parametrize("q_len,heads,kv_heads", FORMS)
def test_query_rows_that_are_not_numbers(q_len, heads, kv_heads):
    """make NaN their own results only."""
    g = _gen(3)
    lens = [200, 70, 5]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    q = _normal(g, 3 * q_len, heads, 128)
    want = OPS.kv4_decode(q, pool, table, _i64(lens), SCALE, q_len)
    bad = torch.rand(3 * q_len, heads, generator=g, device=DEV) < 0.2
    bad[0, 0] = bad[-1, -1] = True
    x = q.clone()
    x[bad] = torch.where(torch.rand(128, generator=g, device=DEV) < 0.1, math.nan, 1.0).to(BF)
    x[0, 0, 3] = x[-1, -1, 7] = math.nan
    # token t of request b sees lens[b] - q_len + 1 + t keys; one that sees none has nothing to make NaN of
    sees = (_i64(lens)[:, None] - q_len + 1 + torch.arange(q_len, device=DEV)).view(-1, 1)
    bad = x.isnan().any(-1) & (sees > 0)
    out, lse = OPS.kv4_decode(x, pool, table, _i64(lens), SCALE, q_len)
    assert out[bad].isnan().all() and lse.view(bad.shape)[bad].isnan().all()
    _check_decode(q, pool, table, lens, SCALE, q_len,
                  (torch.where(bad[..., None], want[0], out), torch.where(bad.view(-1), want[1], lse)))


# ---- scales ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("q_len,heads,kv_heads", FORMS)
@pytest.mark.parametrize("key,value", [(127, 105), (127, 137), (105, 127), (137, 130), (20, 30), (105, 106), (9, 9), (200, 200)])
def test_scales_of_any_size(key, value, q_len, heads, kv_heads, dtype):
    """Past what fp16 holds, and units on both sides of it (104 to 135); a softmax scale that brings the scores back.
    A quarter of the groups hold zeros with the least scale."""
    if dtype == HF and value > 137:
        pytest.skip("the results pass fp16's range")
    g = _gen(4)
    lens = [700, 64, 33, 5]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    _scales(pool, ((key, 3 if key > 9 else 1), (value, 3 if value > 9 else 1)), gen=g)
    zero = torch.rand(blocks * 128, kv_heads, generator=g, device=DEV) < 0.25
    slots = torch.arange(blocks * 128, device=DEV)
    for h in range(kv_heads):
        s = slots[zero[:, h]]
        kc, vc, ks, vs = o4.places(s)
        for at, x in ((kc[:, :16], 0), (vc[:, 16:32], 0), (ks[:, :1], 8), (vs[:, 1:2], 8)):
            pool[s[:, None] // 128, h, at] = x
    q = _normal(g, len(lens) * q_len, heads, 128, dtype=dtype)
    scale = SCALE * 2.0 ** (127 - key)
    _check_decode(q, pool, table, lens, scale, q_len, OPS.kv4_decode(q, pool, table, _i64(lens), scale, q_len))
    if q_len == 1:
        got = OPS.kv4_cascade_decode(q, pool, table[:1], _i64([700]), pool, table, _i64(lens), scale)
        _check_cascade(q, pool, table[:1], 700, pool, table, lens, scale, got, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("q_len,heads,kv_heads", FORMS)
@pytest.mark.parametrize("step", [1 / 16, 1.0, 8.0, -1.0, -8.0])
def test_rising_and_falling_scores(step, q_len, heads, kv_heads, dtype):
    """Each four tokens pass those before (or are passed): by less than the reference point's slack at a time, and by more."""
    g = _gen(5)
    lens = [1500, 300, 70, 33]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    for b, n in enumerate(lens):
        j = torch.arange(n, device=DEV)
        kv = torch.zeros(n, kv_heads, 128, device=DEV)
        kv[..., 77] = (step * (j // 4))[:, None]
        v = _normal(g, n, kv_heads, 128)
        pool = o4.write(pool, kv.to(BF), v, table[b].long()[j // 128] * 128 + j % 128)
    q = _normal(g, len(lens) * q_len, heads, 128, dtype=dtype)
    q[..., 77] = 1
    _check_decode(q, pool, table, lens, 0.5, q_len, OPS.kv4_decode(q, pool, table, _i64(lens), 0.5, q_len))
    if q_len == 1:
        got = OPS.kv4_cascade_decode(q, pool, table[:1], _i64([1500]), pool, table, _i64(lens), 0.5)
        _check_cascade(q, pool, table[:1], 1500, pool, table, lens, 0.5, got, dtype)


# ---- pages, lengths, lists --------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("q_len,heads,kv_heads", FORMS)
def test_pages_outside_the_pool_read_as_zeros(q_len, heads, kv_heads, dtype):
    g = _gen(6)
    lens = [400, 130, 64, 700]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    table[0, 1], table[0, 3], table[1, 0], table[2, 0], table[3, 5] = -1, blocks, 2 ** 31 - 1, -2 ** 31, -7
    q = _normal(g, 4 * q_len, heads, 128, dtype=dtype)
    _check_decode(q, pool, table, lens, SCALE, q_len, OPS.kv4_decode(q, pool, table, _i64(lens), SCALE, q_len))
    if q_len == 1:
        got = OPS.kv4_cascade_decode(q, pool, table[:1], _i64([400]), pool, table, _i64(lens), SCALE)
        _check_cascade(q, pool, table[:1], 400, pool, table, lens, SCALE, got, dtype)


@pytest.mark.parametrize("q_len,heads,kv_heads", FORMS)
def test_lengths_are_clamped(q_len, heads, kv_heads):
    g = _gen(7)
    table, blocks = _tables(g, [256, 256])
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    q = _normal(g, 2 * q_len, heads, 128)
    lens = _i64([10 ** 12, -5])
    _check_decode(q, pool, table, [256, 0], SCALE, q_len, OPS.kv4_decode(q, pool, table, lens, SCALE, q_len))
    empty = torch.empty(2, 0, dtype=torch.int32, device=DEV)
    for t, p in ((empty, pool), (table, pool[:0]), (empty, pool[:0])):
        out, lse = OPS.kv4_decode(q, p, t, _i64([3, 300]), SCALE, q_len)
        assert (out == 0).all() and (lse == -math.inf).all()
    if q_len == 1:
        got = OPS.kv4_cascade_decode(q, pool, table[:1], _i64([2 ** 62]), pool, table, lens, SCALE)
        _check_cascade(q, pool, table[:1], 256, pool, table, [256, 0], SCALE, got, BF)
        got = OPS.kv4_cascade_decode(q, pool[:0], empty[:1], _i64([9]), pool, table, lens, SCALE)
        _check_cascade(q, pool, table[:1], 0, pool, table, [256, 0], SCALE, got, BF)
        out, lse = OPS.kv4_cascade_decode(q, pool, table[:1], _i64([-1]), pool[:0], empty, lens, SCALE)
        assert (out == 0).all() and (lse == -math.inf).all()


def test_more_row_tiles_than_workgroups():
    """17600 rows a kv head: 275 tiles, one workgroup each."""
    lens, q_len, heads = [2000, 0, 1101], 1100, 16
    g = _gen(8)
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, 1, DEV)
    q = _normal(g, 3 * q_len, heads, 128)
    _check_decode(q, pool, table, lens, SCALE, q_len, OPS.kv4_decode(q, pool, table, _i64(lens), SCALE, q_len))


@pytest.mark.parametrize("q_len,heads,kv_heads,batch", [(5, 8, 1, 700), (1, 40, 2, 1100), (1, 20, 1, 530), (1, 2, 2, 4000)])
def test_many_requests(q_len, heads, kv_heads, batch):
    """Several to each thread that lays out the list."""
    g = _gen(9)
    lens = [(37 * i) % 130 if i % 5 else 0 for i in range(batch)]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    q = _normal(g, batch * q_len, heads, 128)
    got = OPS.kv4_decode(q, pool, table, _i64(lens), SCALE, q_len)
    some = list(range(0, batch, 11)) + [batch - 1]
    rows = torch.tensor([b * q_len + t for b in some for t in range(q_len)], device=DEV)
    part = got[0][rows], got[1].view(-1, heads)[rows].reshape(-1)
    _check_decode(q[rows], pool, table[some], [lens[b] for b in some], SCALE, q_len, part)


@pytest.mark.parametrize("heads,kv_heads,batch", [(40, 2, 700), (20, 1, 3), (64, 1, 40), (33, 3, 2), (16, 1, 600), (48, 6, 48), (40, 20, 90)])
def test_cascade_of_other_groups(heads, kv_heads, batch):
    """Suffixes of more than 16 rows have a launch of their own; and many suffixes."""
    g = _gen(10)
    lens = [(29 * i) % 150 for i in range(batch)]
    both, blocks = _tables(g, [900] + lens)
    pool = o4.random_pool(g, blocks, kv_heads, DEV)
    q = _normal(g, batch, heads, 128)
    ptable, table = both[:1].contiguous(), both[1:].contiguous()
    out, lse = OPS.kv4_cascade_decode(q, pool, ptable, _i64([900]), pool, table, _i64(lens), SCALE)
    some = list(range(0, batch, 13)) + [batch - 1]
    grp = heads // kv_heads
    pk, pv = o4.cached(pool, ptable[0], 900)
    for b in some:
        k, v = (torch.cat([x, y]) for x, y in zip((pk, pv), o4.cached(pool, table[b], lens[b])))
        for h in range(kv_heads):
            hs = slice(h * grp, (h + 1) * grp)
            ref = o4.attend(q[b, hs], k[:, h], v[:, h], 900 + lens[b], SCALE, BF, grp * batch)
            close(out[b, hs], lse.view(-1, heads)[b, hs], ref)


@pytest.mark.parametrize("group", [1, 20, 40])
def test_long_lists(group):
    """More units to a wave than are described at a time. The pages repeat, so that attention over them is
    that over one copy, with lse + log(copies). A term passes at most as many additions as its wave's share has tokens
    (at most 100 units), then those of 2048 parts."""
    g = _gen(11)
    pages, copies, kv_heads = 64, 150, 8
    pool = o4.random_pool(g, pages, kv_heads, DEV)
    table = torch.arange(pages, dtype=torch.int32, device=DEV).repeat(copies)[None].contiguous()
    n = pages * copies * 128
    q = _normal(g, 1, group * kv_heads, 128)
    out, lse = OPS.kv4_decode(q, pool, table, _i64([n]), SCALE)
    k, v = o4.cached(pool, table[0], pages * 128)
    adds = (100 * 64 + 2048) * o4.F32
    for h in range(kv_heads):
        hs = slice(h * group, (h + 1) * group)
        o, l, b_o, b_l = o4.attend(q[0, hs], k[:, h], v[:, h], pages * 128, SCALE, BF, group)
        lost = n * 2.0 ** -32 * v.abs().amax() if group > 16 else 0
        close(out[0, hs], lse[hs], (o, l + math.log(copies), b_o + adds * v[:, h].abs().mean(0) * 4 + lost, b_l + adds))


@pytest.mark.parametrize("kv_heads", [1, 8])
def test_offsets_past_32_bits(kv_heads):
    """Pages beyond 4 GB of a pool, written, read and attended."""
    g = _gen(12)
    blocks = 2 ** 32 // (kv_heads * o4.PAGE_BYTES) + 40
    pool = torch.empty(blocks, kv_heads, o4.PAGE_BYTES, dtype=torch.uint8, device=DEV)
    ids = [blocks - 1, 3, blocks - 2]
    for p in ids:
        pool[p] = 0
    for tokens in (300, 384):
        slots = _i64([p * 128 + j for p in ids for j in range(128)][:tokens])
        k, v = _normal(g, tokens, kv_heads, 128), _normal(g, tokens, kv_heads, 128)
        OPS.kv4_cache_write(k, v, slots, pool)
        want = [o4.values(*o4.quantise(x)) for x in (k, v)]
        for got, ref in zip(OPS.kv4_cache_read(pool, slots), want):
            assert torch.equal(got.double(), ref)
    big = slots.repeat(130)  # eight tokens at a time
    for got, ref in zip(OPS.kv4_cache_read(pool, big), want):
        assert torch.equal(got.double(), ref.repeat(130, 1, 1))
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    for group in (2, 20, 40):
        q = _normal(g, 1, group * kv_heads, 128)
        _check_decode(q, pool, table, [384], SCALE, 1, OPS.kv4_decode(q, pool, table, _i64([384]), SCALE))
        a, b = table[:, :1].contiguous(), table[:, 1:2].contiguous()
        got = OPS.kv4_cascade_decode(q, pool, a, _i64([100]), pool, b, _i64([128]), SCALE)
        _check_cascade(q, pool, a, 100, pool, b, [128], SCALE, got, BF)


# ---- workspaces, streams, graphs -----------------------------------------------------------
@pytest.mark.parametrize("batch,q_len,heads,kv_heads,prefix", [
    (3, 1, 16, 4, None), (40, 2, 24, 2, None), (1, 1, 130, 1, None), (300, 1, 8, 8, None), (2, 300, 16, 1, None), (5, 1, 16, 4, 700),
    (33, 1, 40, 2, 0), (150, 1, 64, 8, 130), (2, 1, 16, 1, 500), (40, 1, 80, 4, 300)])
def test_workspace_is_as_large_as_planned(batch, q_len, heads, kv_heads, prefix):
    """The C entry points write nothing behind the planned workspace, the output or the lse, and what the workspace
    held before does not matter."""
    g = _gen(batch)
    lens = torch.randint(0, 400, (batch,), generator=g, device=DEV).tolist()
    lens[0] = 512
    kv = _i64(lens)
    table = torch.randint(0, 40, (batch, 4), generator=g, device=DEV, dtype=torch.int32)
    pool = o4.random_pool(g, 40, kv_heads, DEV)
    q = _normal(g, batch * q_len, heads, 128)
    n, guard, lib = ctypes.c_int64(0), 4096, abi.lib()
    if prefix is None:
        assert lib.ck_kv4_decode_plan(batch, q_len, heads, kv_heads, 512, ctypes.byref(n)) == 0
    else:
        ptable, plen = torch.arange(6, dtype=torch.int32, device=DEV)[None], _i64([prefix])
        assert lib.ck_kv4_cascade_decode_plan(batch, heads, kv_heads, 6 * 128, 512, ctypes.byref(n)) == 0
    rows = batch * q_len * heads
    sizes = {"ws": n.value, "out": rows * 256, "lse": rows * 4}
    for fill in (0x5a, 0xff):
        room = {k: torch.full((v + guard,), fill, dtype=torch.uint8, device=DEV) for k, v in sizes.items()}
        tail = (room["out"].data_ptr(), room["lse"].data_ptr(), room["ws"].data_ptr(), n.value,
                torch.cuda.current_stream().cuda_stream)
        if prefix is None:
            rc = lib.ck_kv4_decode(q.data_ptr(), pool.data_ptr(), table.data_ptr(), 4, kv.data_ptr(), batch, q_len, heads,
                                   kv_heads, 40, 128, 0, SCALE, *tail)
        else:
            rc = lib.ck_kv4_cascade_decode(q.data_ptr(), pool.data_ptr(), ptable.data_ptr(), 6, plen.data_ptr(), 40,
                                           pool.data_ptr(), table.data_ptr(), 4, kv.data_ptr(), 40, batch, heads, kv_heads,
                                           128, 0, SCALE, *tail)
        assert rc == 0
        torch.cuda.synchronize()
        for k, v in sizes.items():
            assert (room[k][v:] == fill).all(), k
        out = room["out"][:sizes["out"]].view(BF).view(batch * q_len, heads, 128)
        lse = room["lse"][:sizes["lse"]].view(torch.float32)
        want = OPS.kv4_decode(q, pool, table, kv, SCALE, q_len) if prefix is None else \
            OPS.kv4_cascade_decode(q, pool, ptable, plen, pool, table, kv, SCALE)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_streams_and_repeats():
    """Calls on two streams at once, each with its own workspace, give what one alone gives, bit for bit."""
    g = _gen(13)
    lens = [3000, 17, 900, 0]
    table, blocks = _tables(g, lens)
    pool = o4.random_pool(g, blocks, 2, DEV)
    calls = []
    for heads in (16, 64, 128):
        q = _normal(g, 4, heads, 128)
        calls.append(lambda q=q: OPS.kv4_decode(q, pool, table, _i64(lens), SCALE))
        calls.append(lambda q=q: OPS.kv4_cascade_decode(q, pool, table[:1], _i64([3000]), pool, table, _i64(lens), SCALE))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for r in range(3):
        for i in range(len(calls)):
            with torch.cuda.stream(streams[(i + r) % 2]):
                got.append(calls[i]())
    torch.cuda.synchronize()
    for i, (o, l) in enumerate(got):
        assert torch.equal(o, want[i % len(calls)][0]) and torch.equal(l, want[i % len(calls)][1])


def test_graphs_of_a_step():
    """Write, read, decode and shared-prefix decode captured, two graphs of other shapes replayed in turn on other contents,
    lengths and tables, with eager calls between the replays."""
    def inputs(seed, heads, tokens, pages):
        g = _gen(seed)
        table = torch.randperm(pages, generator=g, device=DEV)[:12].view(3, 4).to(torch.int32)
        lens = [[130, 5, 400], [0, 512, 33], [1, 1, 256], [512, 300, 0]][seed % 4]
        slots = torch.randperm(pages * 128, generator=g, device=DEV)[:tokens]
        slots[0] = -1
        if seed % 2:
            slots = slots.sort().values
        return dict(k=_normal(g, tokens, 2, 128), v=_normal(g, tokens, 2, 128), slots=slots, pool=o4.random_pool(g, pages, 2, DEV),
                    table=table, lens=_i64(lens), plen=_i64([[512, 100, 0, 33][seed % 4]]), q=_normal(g, 3, heads, 128),
                    q2=_normal(g, 6, heads, 128))

    def step(t):
        OPS.kv4_cache_write(t["k"], t["v"], t["slots"], t["pool"])
        r = OPS.kv4_cache_read(t["pool"], t["slots"])
        a = OPS.kv4_decode(t["q"], t["pool"], t["table"], t["lens"], SCALE)
        b = OPS.kv4_decode(t["q2"], t["pool"], t["table"], t["lens"], SCALE, 2)
        c = OPS.kv4_cascade_decode(t["q"], t["pool"], t["table"][:1], t["plen"], t["pool"], t["table"], t["lens"], SCALE)
        return r + a + b + c + (t["pool"],)

    shapes = [(16, 3, 24), (48, 24600, 200)]
    statics, graphs, outs = [], [], []
    for shape in shapes:
        static = inputs(0, *shape)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(static)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(static))
        statics.append(static)
        graphs.append(graph)
    filler = torch.randn(512, 512, device=DEV)
    for r in range(1, 6):
        fresh = [inputs(r, *s) for s in shapes]
        for static, new in zip(statics, fresh):
            for name, x in new.items():
                static[name].copy_(x)
        (filler @ filler).sum().item()
        for i in ((0, 1) if r % 2 else (1, 0)):
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            for o, w in zip([o.clone() for o in outs[i]], step(fresh[i])):
                assert torch.equal(o, w), (r, i)


# ---- together --------------------------------------------------------------------------------
def test_a_request_from_prompt_to_decode():
    """A prompt is written, then tokens one by one, each attended; then three at a time; what the cache gives back goes through
    the 16-bit operators; a part of the sequence in 16 bits is merged with the rest in 4."""
    g = _gen(14)
    heads, kv_heads, n = 16, 4, 200
    kv = _normal(g, n + 5, 2 * kv_heads, 128)
    k, v = kv[:, :kv_heads], kv[:, kv_heads:]
    q = _normal(g, n + 5, heads, 128)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=DEV)
    at = lambda p: table[0, p // 128].long() * 128 + p % 128  # noqa: E731
    pos = torch.arange(n + 5, device=DEV)
    pool = torch.full((3, kv_heads, o4.PAGE_BYTES), 255, dtype=torch.uint8, device=DEV)
    OPS.kv4_cache_write(k[:n], v[:n], at(pos[:n]), pool)
    for i in (n, n + 1):
        OPS.kv4_cache_write(k[i:i + 1], v[i:i + 1], at(pos[i:i + 1]), pool)
        _check_decode(q[i:i + 1], pool, table, [i + 1], SCALE, 1, OPS.kv4_decode(q[i:i + 1], pool, table, _i64([i + 1]), SCALE))
    OPS.kv4_cache_write(k[n + 2:], v[n + 2:], at(pos[n + 2:]), pool)
    new, last = q[n + 2:].contiguous(), q[n + 4:].contiguous()
    got = OPS.kv4_decode(new, pool, table, _i64([n + 5]), SCALE, 3)
    _check_decode(new, pool, table, [n + 5], SCALE, 3, got)
    # the 16-bit pools that the cache gives back, through the 16-bit operator
    every = torch.arange(3 * 128, device=DEV)
    pools = [x.nan_to_num(0).view(3, 128, kv_heads, 128) for x in OPS.kv4_cache_read(pool, every)]
    both = OPS.suffix_decode(last, *pools, table, _i64([n + 5]))
    # its P is within 2^-16: inside the bound for more than 16 rows (2^-11)
    x, y = o4.cached(pool, table[0], n + 5)
    for h in range(kv_heads):
        hs = slice(4 * h, 4 * h + 4)
        close(both[0][0, hs], both[1].view(-1)[hs], o4.attend(last[0, hs], x[:, h], y[:, h], n + 5, SCALE, BF, 17))
    # the first page in 4 bits, the rest in 16: each part's rounding, and the merge's own
    a = OPS.kv4_decode(last, pool, table[:, :1].contiguous(), _i64([128]), SCALE)
    b = OPS.suffix_decode(last, *pools, table[:, 1:].contiguous(), _i64([n + 5 - 128]))
    out, lse = OPS.lse_merge_with_lse(a[0], b[0], a[1], b[1].view(-1))
    for h in range(kv_heads):
        hs = slice(4 * h, 4 * h + 4)
        o, l, _, b_l = o4.attend(last[0, hs], x[:, h], y[:, h], n + 5, SCALE, BF, 17)
        p = torch.exp((last[0, hs].double() @ x[:, h].T) * SCALE - l[:, None])
        mean = p @ y[:, h].abs()
        assert ((out[0, hs].double() - o).abs() <= (2 * 2.0 ** -8 + 2.0 ** -10) * mean + 2.0 ** -8 * o.abs()).all()
        assert ((lse.view(-1)[hs].double() - l).abs() <= 3 * b_l).all()


def test_cascade_is_decode_over_prefix_and_suffix():
    """One table of both, where the prefix ends with a page: the same sums, cut elsewhere."""
    g = _gen(15)
    suffixes = [5, 0, 300, 64]
    both, blocks = _tables(g, [384] + suffixes)
    pool = o4.random_pool(g, blocks, 2, DEV)
    q = _normal(g, 4, 16, 128)
    cols = both.shape[1]
    table = torch.cat([both[:1, :3].expand(4, 3), both[1:]], 1).contiguous()
    assert table.shape == (4, 3 + cols)
    lens = [384 + n for n in suffixes]
    _check_decode(q, pool, table, lens, SCALE, 1, OPS.kv4_decode(q, pool, table, _i64(lens), SCALE))
    got = OPS.kv4_cascade_decode(q, pool, both[:1].contiguous(), _i64([384]), pool, both[1:].contiguous(), _i64(suffixes), SCALE)
    _check_cascade(q, pool, both[:1], 384, pool, both[1:], suffixes, SCALE, got, BF)
