"""GPU parity of the latent operators with their 64-bit definition (oracle/latent.py), at the
sizes, masks and memory contents where they can go wrong. Tolerances are the oracle's bounds
of the documented roundings."""
import math

import pytest
import torch

from oracle import latent as ol

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
OPS = torch.ops.npu
BF, HF = torch.bfloat16, torch.float16
SCALE = 1 / math.sqrt(192)


@pytest.fixture(scope="module", autouse=True)
def _lib():
    import cascade_amd  # noqa: F401
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible to torch")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _i64(x):
    return torch.tensor(x, dtype=torch.int64, device=DEV)


def _pool(g, lens, dtype, extra=3, cols=None, garbage=True):
    """A pool with the lens' tokens in shuffled pages; what lies past a length is NaN and inf."""
    need = [-(-n // 128) for n in lens]
    cols = max(need + [1]) if cols is None else cols
    cache = _randn(g, sum(need) + extra, 128, 576, dtype=dtype)
    order = torch.randperm(sum(need) + extra, generator=g, device=DEV).tolist()
    table = torch.full((len(lens), cols), -7, dtype=torch.int32)  # entries past a length are never looked at
    at = 0
    for b, (n, k) in enumerate(zip(lens, need)):
        table[b, :k] = torch.tensor(order[at:at + k], dtype=torch.int32)
        at += k
        if garbage and n % 128:
            cache[order[at - 1], n % 128:] = math.nan
            cache[order[at - 1], n % 128::2] = math.inf
    return cache, table.to(DEV)


def _rows(cache, table, b, n):
    k = -(-n // 128)
    return cache[table[b, :k].long()].reshape(-1, 576)[:n]


def _check_decode(q, cache, table, lens, q_len, out, lse, scale=SCALE):
    heads, lse = q.shape[1], lse.view(q.shape[0], q.shape[1])
    worst = 0.0
    for b, n in enumerate(lens):
        x = _rows(cache, table, b, n)
        for i in range(q_len):
            t = b * q_len + i
            sees = max(0, n - q_len + 1 + i)
            ref = ol.attend(q[t], x, x[:, :512], sees, scale, q.dtype)
            try:
                worst = max(worst, ol.close(out[t], lse[t], ref))
            except AssertionError as e:
                raise AssertionError("request %d of %d tokens, token %d, %d heads: %s" % (b, n, i, heads, e))
    return worst


# ---- cache write ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("tokens,stride", [(1, 576), (5, 584), (129, 2112)])
def test_write(dtype, interleaved, tokens, stride):
    g = _gen(tokens)
    kv = _randn(g, tokens, stride, dtype=dtype, scale=2.0)[:, :576]
    kv[0, :512] = 0  # a norm of nothing: eps alone
    gamma = _randn(g, 512, dtype=dtype)
    ang = torch.rand(40, 32, generator=g, device=DEV) * 6
    cos_sin = torch.cat([ang.cos(), ang.sin()], 1)
    pos = torch.randint(0, 40, (tokens,), generator=g, device=DEV)
    slots = torch.randperm(4 * 128, generator=g, device=DEV)[:tokens]
    if tokens > 4:  # not written: padding, past the pool, positions without an angle
        slots[1], slots[2] = -1, 4 * 128
        pos[3], pos[4] = -1, 40
    cache = _randn(g, 4, 128, 576, dtype=dtype)
    before = cache.clone()
    OPS.latent_cache_write(kv, gamma, cos_sin, pos, slots, cache, 1e-6, interleaved)
    done = (slots >= 0) & (slots < 512) & (pos >= 0) & (pos < 40)
    ref = ol.write_rows(kv[done], gamma, cos_sin, pos[done], 1e-6, interleaved)
    got = cache.view(-1, 576)[slots[done]].double()
    # one rounding (fp16 also loses half of its smallest step), fp32 before: a sum of 512 squares,
    # a root, three products; two products and a sum of the pair (whose size, not the result's, counts)
    u = ol.unit(dtype)
    r = kv[done][:, 512:].double().abs()
    size = ref.abs()
    size[:, 512:] = r.amax(1, keepdim=True) * 2
    assert ((got - ref).abs() <= u * ref.abs() + (512 + 16) * ol.F32 * size + 2.0 ** -25).all()
    keep = torch.ones(512, dtype=torch.bool, device=DEV)
    keep[slots[done]] = False
    assert torch.equal(cache.view(-1, 576)[keep], before.view(-1, 576)[keep])


def test_write_of_nothing():
    cache = torch.ones(2, 128, 576, dtype=BF, device=DEV)
    e = torch.empty(0, 576, dtype=BF, device=DEV)
    OPS.latent_cache_write(e, torch.ones(512, dtype=BF, device=DEV), torch.ones(4, 64, device=DEV), _i64([]), _i64([]), cache)
    assert (cache == 1).all()


# ---- decode -------------------------------------------------------------------------------------------
LENS = [0, 1, 31, 32, 33, 127, 128, 129, 300]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads", [1, 5, 16, 20, 33, 64, 128, 130])
def test_decode_heads(heads, dtype):
    g = _gen(heads)
    cache, table = _pool(g, LENS, dtype)
    q = _randn(g, len(LENS), heads, 576, dtype=dtype)
    out, lse = OPS.latent_decode(q, cache, table, _i64(LENS), SCALE)
    _check_decode(q, cache, table, LENS, 1, out, lse)


@pytest.mark.parametrize("q_len,heads", [(2, 16), (3, 40), (7, 8), (5, 128), (40, 3)])
def test_decode_several_tokens(q_len, heads):
    # lengths below q_len: the request's first tokens see nothing
    lens = [0, 1, q_len - 1, q_len, q_len + 1, 32, 33, 200]
    g = _gen(100 + q_len)
    cache, table = _pool(g, lens, BF)
    for b, n in enumerate(lens):  # the last token's row, which the others do not see, poisons nothing
        if n > 1 and b % 2:
            _rows(cache, table, b, n)  # (a copy: the write below goes to the page)
            cache[table[b, (n - 1) // 128].item(), (n - 1) % 128] = math.nan
    q = _randn(g, len(lens) * q_len, heads, 576)
    out, lse = OPS.latent_decode(q, cache, table, _i64(lens), SCALE, q_len)
    for b, n in enumerate(lens):
        x = _rows(cache, table, b, n)
        for i in range(q_len):
            t = b * q_len + i
            if n > 1 and b % 2 and i == q_len - 1:
                assert out[t].isnan().all()  # it does see it
                continue
            ref = ol.attend(q[t], x, x[:, :512], max(0, n - q_len + 1 + i), SCALE, BF)
            ol.close(out[t], lse.view(-1, heads)[t], ref)


@pytest.mark.parametrize("dtype,batch,heads,most", [(BF, 300, 8, 40), (HF, 700, 3, 5), (BF, 257, 36, 70), (BF, 3, 128, 1)])
def test_decode_many_requests(dtype, batch, heads, most):
    g = _gen(batch)
    lens = torch.randint(0, most + 1, (batch,), generator=g, device=DEV).tolist()
    cache, table = _pool(g, lens, dtype)
    q = _randn(g, batch, heads, 576, dtype=dtype)
    out, lse = OPS.latent_decode(q, cache, table, _i64(lens), SCALE)
    _check_decode(q, cache, table, lens, 1, out, lse)


@pytest.mark.parametrize("heads,lens", [(16, [9000]), (128, [4097, 0, 1, 5000]), (2, [1300] * 40)])
def test_decode_cut_requests(heads, lens):
    g = _gen(heads)
    cache, table = _pool(g, lens, BF)
    q = _randn(g, len(lens), heads, 576, scale=3.0)  # peaked: reference points move late
    out, lse = OPS.latent_decode(q, cache, table, _i64(lens), SCALE)
    _check_decode(q, cache, table, lens, 1, out, lse)


def test_decode_rising_scores():
    """Each tile's scores pass all before it, by little and by much."""
    g = _gen(7)
    cache, table = _pool(g, [700, 700], BF, garbage=False)
    q = torch.zeros(2, 32, 576, dtype=BF, device=DEV)
    q[..., 575] = 1
    for b, step in enumerate((1 / 64, 8.0)):
        for j in range(700):
            cache[table[b, j // 128].item(), j % 128, 575] = step * (j // 2)
    out, lse = OPS.latent_decode(q, cache, table, _i64([700, 700]), SCALE)
    _check_decode(q, cache, table, [700, 700], 1, out, lse)


def test_decode_scores_of_minus_infinity():
    """Visible tokens whose score is -inf, some and all of a row's."""
    g = _gen(8)
    cache, table = _pool(g, [100, 100], BF, garbage=False)
    cache[..., 512:] = 0
    q = _randn(g, 2, 4, 576)
    q[..., 512:] = 1
    for j in range(100):
        cache[table[1, 0].item(), j, 512] = -math.inf
        if j < 60:
            cache[table[0, 0].item(), j, 512] = -math.inf
    out, lse = OPS.latent_decode(q, cache, table, _i64([100, 100]), SCALE)
    x = _rows(cache, table, 0, 100)[60:]
    ol.close(out[0], lse[:4], ol.attend(q[0], x, x[:, :512], 40, SCALE, BF))
    assert (out[1] == 0).all() and (lse[4:] == -math.inf).all()


def test_decode_pages_outside_the_pool_read_as_zeros():
    g = _gen(9)
    lens = [400, 130, 64]
    cache, table = _pool(g, lens, BF)
    table[0, 1], table[0, 3], table[1, 0], table[2, 0] = -1, cache.shape[0], 2 ** 31 - 1, -2 ** 31
    q = _randn(g, 3, 24, 576)
    out, lse = OPS.latent_decode(q, cache, table, _i64(lens), SCALE)
    for b, n in enumerate(lens):
        x = torch.cat([cache[p] if 0 <= p < cache.shape[0] else torch.zeros(128, 576, dtype=BF, device=DEV)
                       for p in table[b, :-(-n // 128)].tolist()])[:n]
        ol.close(out[b], lse.view(3, 24)[b], ol.attend(q[b], x, x[:, :512], n, SCALE, BF))


def test_decode_lengths_are_clamped():
    g = _gen(10)
    cache, table = _pool(g, [256, 256], BF, garbage=False)
    q = _randn(g, 2, 16, 576)
    out, lse = OPS.latent_decode(q, cache, table, _i64([10 ** 12, -5]), SCALE)
    _check_decode(q, cache, table, [256, 0], 1, out, lse)
    out, lse = OPS.latent_decode(q, cache, torch.empty(2, 0, dtype=torch.int32, device=DEV), _i64([3, 0]), SCALE)
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = OPS.latent_decode(q, cache[:0], table, _i64([3, 0]), SCALE)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_decode_more_row_tiles_than_workgroups():
    """1100 tokens a request: 275 row tiles, one workgroup each, whose list takes several phases."""
    lens, q_len = [9000, 0, 700, 1101], 1100
    g = _gen(13)
    cache, table = _pool(g, lens, BF)
    q = _randn(g, len(lens) * q_len, 1, 576)
    out, lse = OPS.latent_decode(q, cache, table, _i64(lens), SCALE, q_len)
    for b, n in enumerate(lens):
        x = _rows(cache, table, b, n)
        i = torch.arange(q_len, device=DEV)
        t = slice(b * q_len, (b + 1) * q_len)
        ol.close(out[t, 0], lse[t], ol.attend(q[t, 0], x, x[:, :512], (n - q_len + 1 + i).clamp(0), SCALE, BF))


@pytest.mark.parametrize("batch,q_len,heads,prefix", [(3, 1, 16, None), (40, 2, 33, None), (1, 1, 130, None), (300, 1, 8, None),
                                                      (5, 1, 16, 700), (33, 1, 40, 0), (150, 1, 128, 130)])
def test_workspace_is_as_large_as_planned(batch, q_len, heads, prefix):
    """The C entry points write nothing behind the planned workspace, the output or the lse."""
    import ctypes

    from cascade_amd import abi
    g = _gen(batch)
    lens = torch.randint(0, 400, (batch,), generator=g, device=DEV).tolist()
    cache, table = _pool(g, lens, BF, cols=4)
    q = _randn(g, batch * q_len, heads, 576)
    n, guard = ctypes.c_int64(0), 4096
    kv = _i64(lens)
    if prefix is None:
        assert abi.lib().ck_latent_decode_plan(batch, q_len, heads, 4 * 128, ctypes.byref(n)) == 0
    else:
        pcache, ptable = _pool(g, [prefix], BF, cols=6)
        plen = _i64([prefix])
        assert abi.lib().ck_latent_cascade_decode_plan(batch, heads, 6 * 128, 4 * 128, ctypes.byref(n)) == 0
    rows = batch * q_len * heads
    sizes = {"ws": n.value, "out": rows * 1024, "lse": rows * 4}
    room = {k: torch.full((v + guard,), 0x5a, dtype=torch.uint8, device=DEV) for k, v in sizes.items()}
    tail = (room["out"].data_ptr(), room["lse"].data_ptr(), room["ws"].data_ptr(), n.value,
            torch.cuda.current_stream().cuda_stream)
    if prefix is None:
        rc = abi.lib().ck_latent_decode(q.data_ptr(), cache.data_ptr(), table.data_ptr(), 4, kv.data_ptr(), batch, q_len, heads,
                                        cache.shape[0], 128, 0, SCALE, *tail)
    else:
        rc = abi.lib().ck_latent_cascade_decode(q.data_ptr(), pcache.data_ptr(), ptable.data_ptr(), 6, plen.data_ptr(),
                                                pcache.shape[0], cache.data_ptr(), table.data_ptr(), 4, kv.data_ptr(),
                                                cache.shape[0], batch, heads, 128, 0, SCALE, *tail)
    assert rc == 0
    torch.cuda.synchronize()
    for k, v in sizes.items():
        assert (room[k][v:] == 0x5a).all(), k
    out = room["out"][:sizes["out"]].view(BF).view(batch * q_len, heads, 512)
    lse = room["lse"][:sizes["lse"]].view(torch.float32)
    want = OPS.latent_decode(q, cache, table, kv, SCALE, q_len) if prefix is None else \
        OPS.latent_cascade_decode(q, pcache, ptable, plen, cache, table, kv, SCALE)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_decode_long_list():
    """More tiles per workgroup than are described at a time. The pages repeat, so that
    attention over them is that over one copy, with lse + log(copies)."""
    g = _gen(11)
    pages, copies = 64, 280
    cache = _randn(g, pages, 128, 576)
    table = torch.arange(pages, dtype=torch.int32, device=DEV).repeat(copies)[None]
    n = pages * copies * 128
    q = _randn(g, 1, 16, 576)
    out, lse = OPS.latent_decode(q, cache, table, _i64([n]), SCALE)
    x = cache.view(-1, 576)
    o, l, b_o, b_l = ol.attend(q[0], x, x[:, :512], pages * 128, SCALE, BF)
    ol.close(out[0], lse, (o, l + math.log(copies), b_o + n * ol.F32 * o.abs(), b_l + n * ol.F32))


def test_offsets_past_32_bits():
    """Pages beyond 4 GB of a pool, written and read."""
    g = _gen(12)
    blocks = 2 ** 32 // (128 * 576 * 2) + 40
    cache = torch.empty(blocks, 128, 576, dtype=BF, device=DEV)
    ids = [blocks - 1, 3, blocks - 2]
    for p in ids:
        cache[p] = 0
    slots = _i64([p * 128 + j for p in ids for j in range(128)][:300])
    kv = _randn(g, 300, 576)
    ang = torch.rand(300, 32, generator=g, device=DEV)
    cs = torch.cat([ang.cos(), ang.sin()], 1)
    gamma = torch.ones(512, dtype=BF, device=DEV)
    OPS.latent_cache_write(kv, gamma, cs, torch.arange(300, device=DEV), slots, cache)
    ref = ol.write_rows(kv, gamma, cs, torch.arange(300, device=DEV), 1e-6, True)
    got = torch.cat([cache[p] for p in ids])[:300]
    assert (got.double() - ref).abs().max() < 0.05
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    q = _randn(g, 1, 128, 576)
    out, lse = OPS.latent_decode(q, cache, table, _i64([300]), SCALE)
    ol.close(out[0], lse, ol.attend(q[0], got, got[:, :512], 300, SCALE, BF))
    # a prefix there, suffixes below
    out, lse = OPS.latent_cascade_decode(q, cache, table[:, :1], _i64([100]), cache, table[:, 1:2], _i64([128]), SCALE)
    x = torch.cat([cache[ids[0]][:100], cache[3]])
    ol.close(out[0], lse, ol.attend(q[0], x, x[:, :512], 228, SCALE, BF))


# ---- shared prefix --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,prefix,batch,heads,suffix", [
    (BF, 0, 3, 16, [0, 5, 129]),
    (BF, 1, 1, 1, [0]),
    (HF, 31, 9, 20, [1, 32, 0, 33, 64, 0, 200, 128, 7]),
    (BF, 129, 5, 128, [10, 0, 0, 300, 1]),
    (HF, 1000, 17, 33, [3] * 17),
    (BF, 4096, 40, 16, [0] * 40),
    (BF, 700, 130, 40, list(range(130))),
    (BF, 600, 300, 128, [40] * 300),
    (BF, 20000, 2, 7, [65, 0]),
])
def test_cascade(dtype, prefix, batch, heads, suffix):
    g = _gen(prefix + batch)
    pcache, ptable = _pool(g, [prefix], dtype)
    scache, stable = _pool(g, suffix, dtype)
    q = _randn(g, batch, heads, 576, dtype=dtype)
    out, lse = OPS.latent_cascade_decode(q, pcache, ptable, _i64([prefix]), scache, stable, _i64(suffix), SCALE)
    x = _rows(pcache, ptable, 0, prefix)
    for b, n in enumerate(suffix):
        keys = torch.cat([x, _rows(scache, stable, b, n)])
        ol.close(out[b], lse.view(batch, heads)[b], ol.attend(q[b], keys, keys[:, :512], prefix + n, SCALE, dtype))


def test_cascade_is_decode_over_prefix_and_suffix():
    """One pool, a table that begins with the shared pages: both calls see the same tokens."""
    g = _gen(20)
    lens = [256 + n for n in (1, 0, 77, 400)]
    cache, table = _pool(g, [256] + [n - 256 for n in lens], BF, cols=4)
    full = torch.cat([table[:1, :2].expand(4, 2), table[1:]], 1).contiguous()
    q = _randn(g, 4, 32, 576)
    a = OPS.latent_cascade_decode(q, cache, table[:1].contiguous(), _i64([256]), cache, table[1:].contiguous(),
                                  _i64([n - 256 for n in lens]), SCALE)
    b = OPS.latent_decode(q, cache, full, _i64(lens), SCALE)
    for o, l in (a, b):
        _check_decode(q, cache, full, lens, 1, o, l)


def test_cascade_bad_pages_and_empty_prefix_table():
    g = _gen(21)
    cache, table = _pool(g, [300, 70], BF)
    bad = table.clone()
    bad[0, 1] = 10 ** 6
    q = _randn(g, 1, 16, 576)
    out, lse = OPS.latent_cascade_decode(q, cache, bad[:1], _i64([300]), cache, table[1:], _i64([70]), SCALE)
    x = torch.cat([cache[table[0, 0]], torch.zeros(128, 576, dtype=BF, device=DEV), cache[table[0, 2]][:44],
                   cache[table[1, 0]][:70]])
    ol.close(out[0], lse, ol.attend(q[0], x, x[:, :512], 370, SCALE, BF))
    none = torch.empty(1, 0, dtype=torch.int32, device=DEV)
    out, lse = OPS.latent_cascade_decode(q, cache, none, _i64([300]), cache, table[1:], _i64([70]), SCALE)
    x = cache[table[1, 0]][:70]
    ol.close(out[0], lse, ol.attend(q[0], x, x[:, :512], 70, SCALE, BF))


def test_cascade_units_longer_than_described_at_once():
    """More tiles in a unit of the prefix than are described at a time: its state goes on over phases."""
    g = _gen(22)
    suffix = [(37 * b) % 90 for b in range(117)]
    pcache, ptable = _pool(g, [20000], BF)
    scache, stable = _pool(g, suffix, BF)
    q = _randn(g, 117, 128, 576)
    out, lse = OPS.latent_cascade_decode(q, pcache, ptable, _i64([20000]), scache, stable, _i64(suffix), SCALE)
    x = _rows(pcache, ptable, 0, 20000)
    for b in (0, 1, 58, 116):
        keys = torch.cat([x, _rows(scache, stable, b, suffix[b])])
        ol.close(out[b], lse.view(117, 128)[b], ol.attend(q[b], keys, keys[:, :512], 20000 + suffix[b], SCALE, BF))


# ---- prefill ----------------------------------------------------------------------------------------------
def _prompt(g, ql, kl, heads, dtype, behind=0, packed=True):
    t, s = sum(ql) + behind, sum(kl)
    q = _randn(g, t, heads, 192, dtype=dtype)
    kv = _randn(g, s, heads, 256, dtype=dtype)
    kr = _randn(g, s, 64 if packed else 576, dtype=dtype)[:, -64:]
    return q, kv[..., :128], kr, kv[..., 128:]


def _check_prefill(q, k, kr, v, ql, kl, causal, out, lse):
    heads, qa, ka = q.shape[1], 0, 0
    lse = lse.view(-1, heads)
    for n, m in zip(ql, kl):
        sees = (m - n + 1 + torch.arange(n, device=DEV)).clamp(0, m) if causal else torch.full((n,), m, device=DEV)
        for h in range(heads):
            keys = torch.cat([k[ka:ka + m, h], kr[ka:ka + m]], 1)
            ol.close(out[qa:qa + n, h], lse[qa:qa + n, h],
                     ol.attend(q[qa:qa + n, h], keys, v[ka:ka + m, h], sees, SCALE, q.dtype))
        qa, ka = qa + n, ka + m
    assert (out[qa:] == 0).all() and (lse[qa:] == -math.inf).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,ql,kl,behind", [
    (1, [1], [1], 0),
    (3, [7, 0, 1, 64], [7, 5, 0, 64], 4),
    (2, [32, 33, 63], [64, 33, 200], 0),
    (2, [257, 100], [257, 3], 300),      # 97 rows of the second see nothing
    (5, [129], [700], 1),
    (1, [600, 31], [600, 1000], 0),
])
def test_prefill(dtype, causal, heads, ql, kl, behind):
    g = _gen(sum(ql))
    q, k, kr, v = _prompt(g, ql, kl, heads, dtype, behind, packed=causal)
    out, lse = OPS.latent_prefill(q, k, kr, v, _i64(ql), _i64(kl), SCALE, causal)
    _check_prefill(q, k, kr, v, ql, kl, causal, out, lse)


def test_prefill_many_requests():
    g = _gen(31)
    ql = torch.randint(0, 4, (600,), generator=g, device=DEV).tolist()
    kl = [n + (i % 3) for i, n in enumerate(ql)]
    q, k, kr, v = _prompt(g, ql, kl, 2, BF)
    out, lse = OPS.latent_prefill(q, k, kr, v, _i64(ql), _i64(kl), SCALE)
    _check_prefill(q, k, kr, v, ql, kl, True, out, lse)


def test_prefill_other_strides():
    """Heads outside tokens, one key head for all, a rotated part inside wider rows."""
    g = _gen(32)
    q = _randn(g, 90, 3, 192)
    k = _randn(g, 3, 90, 128).transpose(0, 1)
    v = _randn(g, 90, 1, 128).expand(90, 3, 128)
    kr = _randn(g, 90, 576)[:, 512:]
    out, lse = OPS.latent_prefill(q, k, kr, v, _i64([90]), _i64([90]), SCALE)
    _check_prefill(q, k, kr, v, [90], [90], True, out, lse)


def test_prefill_lengths_past_the_ends():
    g = _gen(33)
    q, k, kr, v = _prompt(g, [100], [150], 2, BF)
    out, lse = OPS.latent_prefill(q, k, kr, v, _i64([40, 10 ** 15, 5]), _i64([40, 10 ** 15, 5]), SCALE, False)
    _check_prefill(q, k, kr, v, [40, 60, 0], [40, 110, 0], False, out, lse)
    out, lse = OPS.latent_prefill(q, k, kr, v, _i64([-3, 100]), _i64([-3, 150]), SCALE)
    _check_prefill(q, k, kr, v, [0, 100], [0, 150], True, out, lse)
    out, lse = OPS.latent_prefill(q, k[:0], kr[:0], v[:0], _i64([100]), _i64([0]), SCALE)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_prefill_hidden_keys_may_hold_anything(dtype, bad):
    """Keys and values that a query does not see, in its own tiles and in the next request's,
    change nothing of it; those that do see them show it."""
    g = _gen(34)
    ql, kl, at = [100, 70], [100, 70], 65
    q, k, kr, v = _prompt(g, ql, kl, 2, dtype)
    good = OPS.latent_prefill(q, k, kr, v, _i64(ql), _i64(kl), SCALE)
    v[at, 0, 5] = bad
    v[100:, 1] = bad
    k[100:, 1] = bad
    out, lse = OPS.latent_prefill(q, k, kr, v, _i64(ql), _i64(kl), SCALE)
    assert torch.equal(out[:at], good[0][:at]) and torch.equal(lse[:at * 2], good[1][:at * 2])
    assert torch.equal(out[:100, 1], good[0][:100, 1])
    assert not torch.isfinite(out[at:100, 0, 5]).any()
    rest = [d for d in range(128) if d != 5]
    assert torch.equal(out[:100, 0][:, rest], good[0][:100, 0][:, rest])
    if not math.isnan(bad):
        assert (out[at:100, 0, 5] == bad).all()


def test_prefill_rising_scores():
    g = _gen(35)
    q, k, kr, v = _prompt(g, [300], [300], 1, BF)
    q[:] = 0
    q[..., 191] = 1
    kr[:, 63] = torch.arange(300, device=DEV).to(BF) * 3
    out, lse = OPS.latent_prefill(q, k, kr, v, _i64([300]), _i64([300]), SCALE)
    _check_prefill(q, k, kr, v, [300], [300], True, out, lse)


# ---- together, on streams, in graphs -------------------------------------------------------------------
def test_a_request_from_prompt_to_decode():
    """A prompt's tokens are written and attended in the expanded form; the next token is written and
    attended in the absorbed form: what the whole sequence's expanded attention gives its last row."""
    g = _gen(40)
    heads, n = 8, 200
    kv = _randn(g, n + 1, 576)
    gamma = _randn(g, 512)
    ang = torch.rand(n + 1, 32, generator=g, device=DEV) * 6
    cs = torch.cat([ang.cos(), ang.sin()], 1)
    w_k, w_v = (_randn(g, heads, 512, 128, scale=512 ** -0.5) for _ in range(2))
    q = _randn(g, n + 1, heads, 192)
    table = torch.tensor([[2, 0]], dtype=torch.int32, device=DEV)
    slot = lambda p: table[0, p // 128].long() * 128 + p % 128  # noqa: E731
    pos = torch.arange(n + 1, device=DEV)
    cache = torch.full((3, 128, 576), math.nan, dtype=BF, device=DEV)
    OPS.latent_cache_write(kv[:n], gamma, cs, pos[:n], slot(pos[:n]), cache)
    OPS.latent_cache_write(kv[n:], gamma, cs, pos[n:], slot(pos[n:]), cache)
    x = _rows(cache, table, 0, n + 1)
    assert torch.isfinite(x).all()
    c = x[:, :512].float()
    k = torch.stack([c @ w_k[h].float() for h in range(heads)], 1)
    v = torch.stack([c @ w_v[h].float() for h in range(heads)], 1)
    out, lse = OPS.latent_prefill(q, k.to(BF), x[:, 512:], v.to(BF), _i64([n + 1]), _i64([n + 1]), SCALE)
    _check_prefill(q, k.to(BF), x[:, 512:], v.to(BF), [n + 1], [n + 1], True, out, lse)
    absorbed = torch.stack([q[n, h, :128].float() @ w_k[h].float().T for h in range(heads)])
    qa = torch.cat([absorbed, q[n, :, 128:].float()], 1).to(BF)[None]
    o, l = OPS.latent_decode(qa, cache, table, _i64([n + 1]), SCALE)
    _check_decode(qa, cache, table, [n + 1], 1, o, l)
    o = torch.stack([o[0, h].float() @ w_v[h].float() for h in range(heads)])
    # between the two: the rounding of k, of the absorbed query and of v and both results, each
    # 2^-8 of numbers whose products add up like random ones: 2^-8 sqrt(5) of the norm, and half as much
    # again for the scores' part in the weights
    assert (o - out[n].float()).norm() < 2 * 2 ** -8 * math.sqrt(5) * out[n].float().norm()
    assert (l - lse.view(-1, heads)[n]).abs().max() < 0.05


def test_graph_of_a_step():
    """Write, decode, shared-prefix decode and prefill captured once, replayed on other contents, lengths
    and tables, with eager calls (which take workspaces of their own) between the replays."""
    heads = 24

    def inputs(seed):
        g = _gen(seed)
        lens = [[130, 5, 400], [0, 512, 33], [1, 1, 256], [512, 300, 0]][seed % 4]
        cache, table = _pool(g, [512] * 3, BF, garbage=False)
        return dict(kv=_randn(g, 3, 576), gamma=_randn(g, 512), cs=torch.rand(600, 64, generator=g, device=DEV),
                    pos=torch.randint(0, 600, (3,), generator=g, device=DEV),
                    slots=table[:, 0].long() * 128 + torch.tensor([seed % 7, -1, 9], device=DEV), cache=cache, table=table,
                    lens=_i64(lens), plen=_i64([[512, 100, 0, 33][seed % 4]]), q=_randn(g, 3, heads, 576),
                    pq=_randn(g, 80, heads, 192), k=_randn(g, 90, heads, 128), kr=_randn(g, 90, 64), v=_randn(g, 90, heads, 128),
                    ql=_i64([[70, 5], [0, 80], [33, 40], [1, 1]][seed % 4]), kl=_i64([[80, 5], [3, 80], [33, 50], [90, 0]][seed % 4]))

    def step(t):
        OPS.latent_cache_write(t["kv"], t["gamma"], t["cs"], t["pos"], t["slots"], t["cache"])
        a = OPS.latent_decode(t["q"], t["cache"], t["table"], t["lens"], SCALE)
        b = OPS.latent_cascade_decode(t["q"], t["cache"], t["table"][:1], t["plen"], t["cache"], t["table"], t["lens"], SCALE)
        c = OPS.latent_prefill(t["pq"], t["k"], t["kr"], t["v"], t["ql"], t["kl"], SCALE)
        return a + b + c + (t["cache"],)

    static = inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    filler = torch.randn(512, 512, device=DEV)
    for r in range(1, 6):
        fresh = inputs(r)
        for name, x in fresh.items():
            static[name].copy_(x)
        (filler @ filler).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for o, w in zip(got, step(fresh)):
            assert torch.equal(o, w), r


def test_streams_and_repeats():
    """Calls on two streams at once, each with its own workspace, give what one alone gives, bit for bit."""
    g = _gen(41)
    lens = [3000, 17, 900, 0]
    cache, table = _pool(g, lens, BF)
    qs = [_randn(g, 4, 64, 576) for _ in range(2)]
    want = [OPS.latent_decode(q, cache, table, _i64(lens), SCALE) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for r in range(3):
        for q, st in zip(qs, streams):
            with torch.cuda.stream(st):
                got.append(OPS.latent_decode(q, cache, table, _i64(lens), SCALE))
    torch.cuda.synchronize()
    for i, (o, l) in enumerate(got):
        assert torch.equal(o, want[i % 2][0]) and torch.equal(l, want[i % 2][1])
