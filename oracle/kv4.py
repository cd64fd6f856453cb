"""The 4-bit K/V cache in 64 bits (torch, any device): the format, the formulas of its operators and
bounds of what their documented roundings can change.

A page holds 128 tokens of a kv head in two units of 64: e2m1 codes and a scale 2^(e - 127) for each
32 dims of a token. What a token's bytes are is stated here address by address.
"""
import math

import torch

D, GROUP, PAGE, UNIT, PAGE_BYTES = 128, 32, 128, 64, 17408
LOWEST, HIGHEST, BAD = 8, 252, 255
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
F32 = 2.0 ** -24


def places(slots):
    """Where a slot's bytes lie in its page: (key codes [T, 64], value codes [T, 64], key scales [T, 4],
    value scales [T, 4]); byte i of the codes holds dims 2 i and 2 i + 1."""
    t = slots % UNIT
    h, g, j, r = (x[:, None] for x in (t // 32, t // 8 % 4, t // 4 % 2, t % 4))
    unit = (slots % PAGE // UNIT * (PAGE_BYTES // 2))[:, None]
    i, grp = (torch.arange(n, device=slots.device)[None, :] for n in (64, 4))
    # values: dims 8 n + 2 q and the next are byte i = 4 n + q
    return (unit + t[:, None] * 64 + i,
            unit + 4096 + (i % 4) * 1024 + g * 256 + (i // 4) * 16 + h * 8 + 4 * j + r,
            unit + 8192 + grp * 64 + g * 16 + r * 4 + h * 2 + j,
            unit + 8448 + grp * 64 + g * 16 + h * 8 + 4 * j + r)


def quantise(x):
    """[..., 128] -> (codes uint8 [..., 64], scale bytes uint8 [..., 4])."""
    x = x.double().unflatten(-1, (D // GROUP, GROUP))
    finite = torch.isfinite(x).all(-1)
    x = torch.where(finite[..., None], x, 0.0)
    most = x.abs().amax(-1)
    floor = torch.floor(torch.log2(most.clamp_min(2.0 ** -160)))
    # log2 may round up to a whole number just below a power of two
    floor = torch.where(torch.exp2(floor) > most.clamp_min(2.0 ** -160), floor - 1, floor)
    e = floor - 2 + (most > 1.75 * torch.exp2(floor)) + 127
    e = e.clamp(LOWEST, HIGHEST)
    y = x.abs() / torch.exp2(e - 127)[..., None]
    grid = torch.tensor(E2M1, dtype=torch.float64, device=x.device)
    d = (y[..., None] - grid).abs()
    near = d == d.amin(-1, keepdim=True)  # one or two neighbours: of two the even one
    even = (torch.arange(8, device=x.device) % 2 == 0)
    code = torch.where(near.sum(-1) == 2, (near & even).int().argmax(-1), near.int().argmax(-1))
    code = torch.where(finite[..., None], code + 8 * torch.signbit(x), 0).flatten(-2)
    return ((code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8),
            torch.where(finite, e, float(BAD)).to(torch.uint8))


def values(codes, e):
    """The numbers that codes [..., 64] and scale bytes [..., 4] stand for, float64 [..., 128]."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    lut = torch.tensor(E2M1 + tuple(-x for x in E2M1), dtype=torch.float64, device=codes.device)
    scale = torch.where(e == BAD, math.nan, torch.exp2(e.double() - 127))
    return (lut[code].unflatten(-1, (D // GROUP, GROUP)) * scale[..., None]).flatten(-2)


def write(pool, key, value, slots):
    """The pool after a write, a copy."""
    pool = pool.clone()
    ok = (slots >= 0) & (slots < pool.shape[0] * PAGE)
    slots, key, value = slots[ok], key[ok], value[ok]
    kc, vc, ks, vs = places(slots)
    (kq, ke), (vq, ve) = quantise(key), quantise(value)
    for h in range(pool.shape[1]):
        page = slots[:, None] // PAGE
        for at, x in ((kc, kq), (ks, ke), (vc, vq), (vs, ve)):
            pool[page, h, at] = x[:, h]
    return pool


def read(pool, slots):
    """(keys, values) of the slots, float64 [T, KVH, 128]; zeros outside the pool."""
    ok = (slots >= 0) & (slots < pool.shape[0] * PAGE)
    k = torch.zeros(slots.shape[0], pool.shape[1], D, dtype=torch.float64, device=pool.device)
    v = k.clone()
    at = slots[ok]
    kc, vc, ks, vs = places(at)
    page = at[:, None] // PAGE
    for h in range(pool.shape[1]):
        k[ok, h] = values(pool[page, h, kc], pool[page, h, ks])
        v[ok, h] = values(pool[page, h, vc], pool[page, h, vs])
    return k, v


def cached(pool, row, n):
    """(keys, values) of the first n tokens behind a block-table row; a page outside the pool holds zeros."""
    j = torch.arange(n, device=pool.device)
    page = row.long()[j // PAGE]
    ok = (page >= 0) & (page < pool.shape[0])
    return read(pool, torch.where(ok, page * PAGE + j % PAGE, -1))


def random_pool(gen, blocks, kv_heads, device, spread=3):
    """A pool of random codes and scales around 1."""
    pool = torch.randint(0, 256, (blocks, kv_heads, PAGE_BYTES), generator=gen, device=device, dtype=torch.uint8)
    for at in (8192, PAGE_BYTES // 2 + 8192):
        pool[..., at:at + 512] = torch.randint(126 - spread, 127 + 1, (blocks, kv_heads, 512), generator=gen, device=device,
                                               dtype=torch.uint8)
    return pool


def attend(q, k, v, sees, scale, dtype, rows):
    """Rows q [n, 128] over keys and values [m, 128]; row i sees the first sees[i] (a list, or one
    number); the call has `rows` of them a kv head. Returns (o, lse, bound of |out - o|, bound of
    |out lse - lse|).

    out rounds by half a step u |o|, below the least normal number by half the least step: 2^-25 in fp16 (steps of
    2^-14-10), 2^-134 in bf16 (of 2^-126-7). A score is an fp32 sum of 128
    exact products, (128 + 8) roundings of partial sums below sum |q| |k|, times the scale (2 roundings,
    its conversion to log2 among them); an error e of the scores moves a softmax weight by 2 e of it. P enters
    as two bf16 terms, off by 2^-18 of it, or (more than 16 rows a kv head) as an fp16 number, off by 2^-11 of it; 2^7 p
    then loses bits in steps of 2^-24 where the largest weight is 1 or more: 2^-32 of it for each token, and so
    does a value below 2^-14, a scale of 2^-23 or more leaving it its bits. The sums over m tokens are fp32;
    exp2 is good to a few steps."""
    q, k, v = q.double(), k.double(), v.double()
    n, m = q.shape[0], k.shape[0]
    sees = torch.as_tensor(sees, device=q.device).clamp(0, m).expand(n)
    if m == 0:
        z = q.new_zeros(n, D)
        return z, q.new_full((n,), -torch.inf), z, q.new_zeros(n)
    hidden = torch.arange(m, device=q.device)[None, :] >= sees[:, None]
    s = torch.where(hidden, -torch.inf, (q @ k.T) * scale)
    lse = torch.logsumexp(s, 1)
    p = torch.where(torch.isneginf(lse)[:, None], 0.0, torch.exp(s - lse[:, None]))
    o, mean = p @ v, p @ v.abs()
    u = torch.finfo(dtype).eps / 2
    e = (128 + 8 + 2) * F32 * (q.abs() @ k.abs().T).masked_fill(hidden, 0).amax(1) * scale
    sums = (sees + 64) * F32
    p_off, lost = (2.0 ** -18, 0.0) if rows <= 16 else (2.0 ** -11, 2.0 ** -32)
    b_o = u * o.abs() + (1 + u) * ((p_off + 2 * e + sums)[:, None] * mean + (sees * lost)[:, None] * v.abs().amax())
    b_o = b_o + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)
    return o, lse, b_o, e + sums + 8 * F32 * lse.nan_to_num(0, 0, 0).abs()
