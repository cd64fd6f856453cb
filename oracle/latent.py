"""Latent attention in 64 bits (torch, any device): the formulas of the latent operators
and bounds of what their documented roundings can change.

A cache row is x = [c (512) | r (64)]. Roundings that the operators make: results to
their 16-bit type (half a step: relative ``unit``), and each probability to that type
before the second product (again ``unit``, of the sum of p |value|). Scores, the softmax's
statistics and sums are fp32.
"""
import math

import torch

R, P, D, PAGE = 512, 64, 128, 128
F32 = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def write_rows(kv, gamma, cos_sin, positions, eps, interleaved):
    """The cache rows of the tokens, float64 [T, 576]."""
    kv, gamma = kv.double(), gamma.double()
    c = kv[:, :R]
    c = c * torch.rsqrt(c.pow(2).mean(1, keepdim=True) + eps) * gamma
    cs = cos_sin.double()[positions]
    cos, sin = cs[:, :P // 2], cs[:, P // 2:]
    r = kv[:, R:]
    a, b = (r[:, 0::2], r[:, 1::2]) if interleaved else (r[:, :P // 2], r[:, P // 2:])
    x, y = a * cos - b * sin, a * sin + b * cos
    r = torch.stack([x, y], 2).flatten(1) if interleaved else torch.cat([x, y], 1)
    return torch.cat([c, r], 1)


def attend(q, keys, values, sees, scale, dtype):
    """Rows q [n, k] over keys [m, k] and values [m, d]; row i sees the first sees[i] of them
    (a list, or one number). Returns (o, lse, bound of |out - o|, bound of |out lse - lse|).

    With u the type's unit: out rounds by u |o|; each p rounds by u, which moves o by at most
    u sum_j softmax_j |value_j|; an error e of the scores moves a softmax weight by 2 e of it, and
    e is that of an fp32 sum of k products (k + 8 roundings of partial sums that stay below
    sum |q| |key| scale). Sums over m tokens are in fp32 too, exp2 is good to a few steps.
    fp16 probabilities are lifted by 2^7 against a largest weight of 1 or more and lose bits in
    steps of 2^-24: half of one, 2^-25, is 2^-32 of a weight, for each token."""
    q, keys, values = q.double(), keys.double(), values.double()
    n, m, d = q.shape[0], keys.shape[0], values.shape[1]
    sees = torch.as_tensor(sees, device=q.device).clamp(0, m).expand(n)
    o, lse = q.new_zeros(n, d), q.new_full((n,), -torch.inf)
    if m == 0:
        return o, lse, q.new_zeros(n, d), q.new_zeros(n)
    hidden = torch.arange(m, device=q.device)[None, :] >= sees[:, None]
    never = hidden.all(0)  # such tokens may hold anything
    keys, values = (torch.where(never[:, None], 0.0, x) for x in (keys, values))
    s = torch.where(hidden, -torch.inf, (q @ keys.T) * scale)
    lse = torch.logsumexp(s, 1)
    p = torch.where(torch.isneginf(lse)[:, None], 0.0, torch.exp(s - lse[:, None]))
    o, mean = p @ values, p @ values.abs()
    u = unit(dtype)
    e = 2 * (q.shape[1] + 8) * F32 * (q.abs() @ keys.abs().T).masked_fill(hidden, 0).amax(1) * scale
    sums = (sees + 64) * F32
    lost = sees * 2.0 ** -32 * values.abs().amax() if dtype == torch.float16 else 0 * sums
    b_o = u * o.abs() + (1 + u) * ((u + 2 * e + sums)[:, None] * mean + lost[:, None])
    if dtype == torch.float16:
        b_o = b_o + 2.0 ** -25
    return o, lse, b_o, e + sums + 8 * F32 * lse.nan_to_num(0, 0, 0).abs()


def close(out, lse, ref):
    """Asserts that out and lse lie within the bounds of attend(); the largest share used."""
    o, l, b_o, b_l = ref
    out, lse = out.double(), lse.double()
    assert torch.isfinite(out).all()
    assert torch.equal(torch.isneginf(lse), torch.isneginf(l)) and not lse.isnan().any()
    d_o, d_l = (out - o).abs(), (lse - l).abs()[~torch.isneginf(l)]
    assert (d_o <= b_o).all(), "out: %.3g over a bound of %.3g" % max(zip(d_o.flatten().tolist(), b_o.flatten().tolist()), key=lambda t: t[0] - t[1])
    assert (d_l <= b_l[~torch.isneginf(l)]).all(), "lse: off by %.3g" % d_l.max()
    return 0.0 if d_o.numel() == 0 else (d_o / b_o.clamp_min(1e-30)).max().item()


# ---- exact counts: which tiles of a long call were read, and how often -----------------------------------
# With q = 0 every score is 0 and every p is one power of two, so that sums of p are whole
# multiples of it, exact in fp32 below 2^24 tokens, and lse is log(tokens read) but for the last few
# roundings. Cached tokens hold a 1 in two value dims that name their tile of 32: o is then the
# share of each dim's tiles.
TILE = 32


def markers(tile):
    """The two value dims of a tile: its number mod 256, and its number / 256."""
    return tile % 256, 256 + tile // 256 % 256


def mark(rows, first_tile=0):
    """Cached tokens [n, 576] of a request, from its tile first_tile on, in place."""
    rows.zero_()
    tile = torch.arange(rows.shape[0], device=rows.device) // TILE + first_tile
    for d in markers(tile):
        rows.scatter_(1, d[:, None], 1)


def counted(tokens, dtype):
    """(o, lse, bounds) of a row that read tokens[t] tokens of tile t (a tensor), as attend() gives them.
    o rounds to the type behind a division and a product in fp32. lse is ln 2 (log2(sum) - bias), log2 good
    to a step of its result, the difference to half of one (the bias is below it), then a product by a
    rounded constant. fp16 sums are 2^7 as large."""
    tokens = tokens.double()
    n, tile = tokens.sum(), torch.arange(tokens.numel(), device=tokens.device)
    o = tokens.new_zeros(R)
    for d in markers(tile):
        o.index_add_(0, d, tokens)
    if n == 0:
        return o, torch.log(n), o, torch.zeros_like(n)
    o, lse = o / n, torch.log(n)
    log2 = torch.log2(n) + (7 if dtype == torch.float16 else 0)
    step = torch.exp2(torch.floor(torch.log2(log2.clamp_min(1))) - 23)
    return o, lse, (unit(dtype) + 4 * F32) * o, math.log(2) * 1.5 * step + 2 * F32 * lse


def whole(n, device="cpu"):
    """Tokens of each tile of a request of n tokens."""
    tile = torch.arange(-(-n // TILE), device=device)
    return (n - tile * TILE).clamp(max=TILE)
