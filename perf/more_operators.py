"""The 4-bit K/V cache operators as measurable calls.

A pool holds pages of 128 tokens and, per kv head, two units of 64 tokens: keys and values
as 4-bit floats (1 sign, 2 exponent, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) in groups of
32 dims that share a scale 2^(e - 127), one byte. Four operators work on it: quantising a
step's tokens into their slots (``kv4_cache_write``), reading tokens back as 16-bit rows
(``kv4_cache_read``), decode over the pages (``kv4_decode``) and the same for a batch that
shares a prefix (``kv4_cascade_decode``).

``listed()`` names the fixed cases, ``draw()`` gives others of the same ranges,
``prepare()`` builds what a serving process holds before the call, ``run()`` is one
call: in elementary torch operations in 32 bits, or, where ``own`` is set, the
framework's operator. ``exact()`` is the operator's definition in 64 bits.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda:0"
D = 128             # head dim
GROUP = 32          # dims that share a scale
PAGE, UNIT = 128, 64  # tokens per page, per unit of a page
UNIT_BYTES = 2 * UNIT * D // 2 + 2 * UNIT * D // GROUP  # codes, then scales: 8704
TOKEN_BYTES = UNIT_BYTES // UNIT  # 136 of a token and kv head
V_AT, KS_AT, VS_AT = 4096, 8192, 8448  # behind the keys' codes: the values', the scales
LOWEST, HIGHEST = 8, 252  # scale bytes: dequantised values stay normal and finite
SCALE = 1.0 / math.sqrt(D)
MAX_SUFFIX = 4096
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases --------------------------------------------------------------------------
def listed():
    return [
        # One decode step's tokens of 64 sequences, written and read back: all launch latency.
        _store("store-t64", 64, 8, "bf16"),
        # A prefill chunk's tokens, in neighbouring slots; the chunk's attention reads them
        # back, so that it sees what later steps will see.
        _store("store-t8192", 8192, 8, "fp16"),
        # The cached context of a prompt that goes on, as 16-bit rows; a small one.
        _load("load-t777", 777, 4, "bf16"),
        # The pages of a long shared context, for kernels that take a 16-bit pool.
        _load("load-t65536", 65536, 8, "bf16"),
        # One sequence: the smallest attention call.
        _decode("decode-b1-h32", 1, 1, 32, 8, 1300, "bf16"),
        # A decode batch with ragged sequences, 4 query heads a kv head: bound by the cache.
        _decode("decode-b64-h32", 64, 1, 32, 8, 8192, "bf16"),
        # Three tokens a sequence (drafted ones under verification), causal among themselves.
        _decode("decode-b24-h64-q3", 24, 3, 64, 8, 5000, "fp16"),
        # Every query head with a kv head of its own.
        _decode("decode-b5-mha", 5, 1, 20, 20, 20011, "fp16"),
        # Long contexts, 8 query heads a kv head: the largest cache.
        _decode("decode-b16-h64", 16, 1, 64, 8, 65536, "bf16"),
        # A small batch on a short system prompt.
        _cascade("cascade-b8-h32", 8, 32, 8, 2048, 256, "bf16"),
        # 64 sequences on a shared 8192-token prefix, suffixes of mean 512: the batch, heads
        # and lengths of this repository's benchmark.
        _cascade("cascade-b64-h32", 64, 32, 8, 8192, 512, "bf16"),
        # A large batch on a long prefix, no multiples of anything: the most arithmetic.
        _cascade("cascade-b117-h64", 117, 64, 8, 16001, 512, "fp16"),
    ]


def _store(name, tokens, kv_heads, dtype):
    return {"name": name, "op": "store", "tokens": tokens, "kv_heads": kv_heads, "dtype": dtype}


def _load(name, tokens, kv_heads, dtype):
    return {"name": name, "op": "load", "tokens": tokens, "kv_heads": kv_heads, "dtype": dtype}


def _decode(name, batch, q_len, heads, kv_heads, kv, dtype):
    return {"name": name, "op": "decode", "batch": batch, "q_len": q_len, "heads": heads, "kv_heads": kv_heads,
            "kv": kv, "dtype": dtype}


def _cascade(name, batch, heads, kv_heads, prefix, mean, dtype):
    return {"name": name, "op": "cascade", "batch": batch, "heads": heads, "kv_heads": kv_heads, "prefix": prefix,
            "suffix_mean": mean, "dtype": dtype}


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["store", "load", "decode", "decode", "decode", "cascade", "cascade"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8, 16])
    if op == "store":
        c = _store("", log(1, 65536 // kv_heads), kv_heads, dtype)
    elif op == "load":
        c = _load("", log(1, 524288 // kv_heads), kv_heads, dtype)
    else:
        heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8, 8, 16])
        if op == "decode":
            batch, q_len = log(1, 128), rng.choice([1, 1, 1, 2, 3, 5])
            kv = log(1, min(65536, 6000000 // (batch * kv_heads), 400000000 // (batch * q_len * heads)))
            c = _decode("", batch, q_len, heads, kv_heads, kv, dtype)
        else:
            batch = log(1, 117)
            prefix = log(128, min(16000, 100000000 // (batch * heads)))
            c = _cascade("", batch, heads, kv_heads, prefix, log(32, 512), dtype)
    del c["name"]
    return c


# ---- sizes --------------------------------------------------------------------------
def _lens(case):
    """Cache lengths of a decode call's requests, new tokens included: ragged in [kv / 4, kv],
    the longest kv. The same set for every seed."""
    rng = np.random.default_rng(case["batch"] * 8191 + case["kv"])
    lens = rng.integers(max(1, case["kv"] // 4), case["kv"] + 1, size=case["batch"])
    lens[0] = case["kv"]
    return lens.astype(np.int64)


def _suffix_lens(case):
    """Suffix lengths, geometric and clipped; every 17th sequence has not begun its own."""
    rng = np.random.default_rng(case["batch"] * 8191 + case["suffix_mean"])
    lens = np.clip(rng.geometric(1.0 / case["suffix_mean"], size=case["batch"]), 1, MAX_SUFFIX)
    lens[16::17] = 0
    return lens.astype(np.int64)


def _pages(lens):
    return (np.asarray(lens) + PAGE - 1) // PAGE


def work(case):
    op, kvh = case["op"], case["kv_heads"]
    if op in ("store", "load"):
        rows = case["tokens"] * kvh
        if op == "store":  # 16-bit rows in, codes and scales written, 16-bit rows out
            return {"bytes": rows * (2 * 2 * 2 * D + TOKEN_BYTES) + 8 * case["tokens"], "flops": rows * 2 * D * 4}
        return {"bytes": rows * (2 * 2 * D + TOKEN_BYTES) + 8 * case["tokens"], "flops": rows * 2 * D}
    h = case["heads"]
    if op == "decode":
        lens, n = _lens(case), case["q_len"]
        rows = case["batch"] * n * h
        seen = sum(int(np.clip(lens - n + 1 + i, 0, None).sum()) for i in range(n))
        return {"bytes": int(lens.sum()) * kvh * TOKEN_BYTES + rows * (2 * 2 * D + 4) + int(_pages(lens).sum()) * 4
                + case["batch"] * 8, "flops": 4 * D * h * seen}
    lens, p = _suffix_lens(case), case["prefix"]
    return {"bytes": (int(lens.sum()) + p) * kvh * TOKEN_BYTES + case["batch"] * h * (2 * 2 * D + 4)
            + (int(_pages(lens).sum()) + int(_pages(p))) * 4 + (case["batch"] + 1) * 8,
            "flops": 4 * D * h * (int(lens.sum()) + case["batch"] * p)}


# ---- inputs -------------------------------------------------------------------------
class _Gen:
    """Seeded device normals and host permutations."""

    def __init__(self, seed, dtype):
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.rng = np.random.default_rng(seed)
        self.dtype = dtype

    def normal(self, *shape, std=1.0):
        return torch.empty(*shape, device=DEV, dtype=self.dtype).normal_(0.0, std, generator=self.g)


def _dev(x, dtype):
    return torch.from_numpy(np.ascontiguousarray(x)).to(device=DEV, dtype=dtype)


def _tables(gen, lens):
    """Block table of the requests over scattered pages of one pool, and the pool's pages."""
    n = _pages(lens)
    phys = gen.rng.permutation(int(n.sum()))
    table = np.zeros((len(n), max(1, int(n.max()))), dtype=np.int32)
    at = 0
    for b, c in enumerate(n):
        table[b, :c] = phys[at:at + c]
        at += c
    return table, max(1, int(n.sum()))


def _pool(gen, blocks, kv_heads):
    """A pool of quantised tokens [blocks, kv_heads, bytes of a page]; some key dims are
    larger than others, as in trained models."""
    pool = torch.empty(blocks, kv_heads, 2 * UNIT_BYTES, dtype=torch.uint8, device=DEV)
    dims = torch.exp(torch.empty(kv_heads, 1, D, device=DEV).normal_(0.0, 0.5, generator=gen.g))
    step = max(1, (1 << 27) // (kv_heads * PAGE * D))
    for at in range(0, blocks, step):
        part = pool[at:at + step]
        k, v = gen.normal(part.shape[0], kv_heads, PAGE, D).float() * dims, gen.normal(part.shape[0], kv_heads, PAGE, D)
        part.copy_(_to_pages(_quantise(k), _quantise(v)))
    return pool


def prepare(case, seed):
    gen = _Gen(seed, DT[case["dtype"]])
    op, kvh = case["op"], case["kv_heads"]
    s = {"case": case}
    if op in ("store", "load"):
        t = case["tokens"]
        blocks = t // PAGE + 8
        s["cache"] = _pool(gen, blocks, kvh)
        if op == "store" and t < 256:  # a decode step: one token a sequence, anywhere
            slots = gen.rng.permutation(blocks * PAGE)[:t]
        else:  # a request's tokens, from some token of its first page on, over scattered pages
            first = int(gen.rng.integers(0, PAGE)) if op == "store" else 0
            at = first + np.arange(t)
            slots = gen.rng.permutation(blocks)[at // PAGE] * PAGE + at % PAGE
        s["slots"] = _dev(slots, torch.int64)
        if op == "store":  # keys and values as a projection leaves them: queries first, in one row
            qkv = gen.normal(t, 6 * kvh, D)
            s["k"], s["v"] = qkv[:, 4 * kvh:5 * kvh], qkv[:, 5 * kvh:]
        return s
    h = case["heads"]
    if op == "decode":
        lens = gen.rng.permutation(_lens(case))
        table, blocks = _tables(gen, lens)
        s["q"] = gen.normal(case["batch"] * case["q_len"], h, D)
    else:
        lens = gen.rng.permutation(_suffix_lens(case))
        both, blocks = _tables(gen, np.concatenate([[case["prefix"]], lens]))
        s["ptable"] = _dev(both[:1, :int(_pages(case["prefix"]))], torch.int32)
        table = both[1:, :max(1, int(_pages(lens).max()))]
        s["plen"] = torch.tensor([case["prefix"]], dtype=torch.int64, device=DEV)
        s["q"] = gen.normal(case["batch"], h, D)
    s["cache"] = _pool(gen, blocks, kvh)
    s["table"], s["lens"] = _dev(table, torch.int32), _dev(lens, torch.int64)
    return s


# ---- one call -----------------------------------------------------------------------
def run(s):
    return (_run_own if own else _run_plain)(s)


_loaded = False


def _run_own(s):
    global _loaded
    if not _loaded:  # registers torch.ops.npu
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "vllm-hust-cascade-kernel_amd"))
        import cascade_amd  # noqa: F401
        _loaded = True
    case = s["case"]
    op = case["op"]
    if op == "store":
        torch.ops.npu.kv4_cache_write(s["k"], s["v"], s["slots"], s["cache"])
    if op in ("store", "load"):
        return torch.ops.npu.kv4_cache_read(s["cache"], s["slots"], DT[case["dtype"]])
    if op == "decode":
        return torch.ops.npu.kv4_decode(s["q"], s["cache"], s["table"], s["lens"], SCALE, case["q_len"])
    return torch.ops.npu.kv4_cascade_decode(s["q"], s["cache"], s["ptable"], s["plen"], s["cache"], s["table"],
                                            s["lens"], SCALE)


# ---- plain form ---------------------------------------------------------------------
def _run_plain(s):
    case = s["case"]
    return {"store": _plain_store, "load": _plain_load, "decode": _plain_decode,
            "cascade": _plain_cascade}[case["op"]](s, case)


def _quantise(x):
    """[..., 128] -> (codes uint8 [..., 64], the even dim in the low half; scale bytes uint8 [..., 4]).
    The scale puts a group's largest magnitude into (3.5, 7] code units; codes round to nearest, ties
    to the even code. A group with a value that is not finite gets scale byte 255 (not a number)."""
    x = x.float().unflatten(-1, (D // GROUP, GROUP))
    most = x.abs().amax(dim=-1)
    e = ((most.nan_to_num(0, 0).view(torch.int32) + 0x1FFFFF) >> 23).sub_(2).clamp_(LOWEST, HIGHEST)
    bad = ~torch.isfinite(x).all(dim=-1)
    y = x * ((254 - e) << 23).view(torch.float32)[..., None]  # 2^(127 - e), exact
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
            + 8 * (torch.signbit(y))).masked_fill_(bad[..., None], 0).flatten(-2)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), e.masked_fill_(bad, 255).to(torch.uint8)


def _dequantise(codes, e):
    """The inverse: fp32 [..., 128]."""
    codes = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
    m = (codes & 7).float()
    x = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2, 2 * m - 8))
    x = torch.where(codes > 7, -x, x).unflatten(-1, (D // GROUP, GROUP))
    bits = torch.where(e == 255, 0x7FC00000, torch.where(e == 0, 0x00400000, e.int() << 23))  # 0: 2^-127
    return (x * bits.to(torch.int32).view(torch.float32)[..., None]).flatten(-2)


def _to_pages(k, v):
    """Codes and scales [..., 128 tokens, .] of keys and values -> page bytes [..., 17408]."""
    lead = k[0].shape[:-2]
    n = len(lead) + 1  # the units' dim is n - 1

    def put(x, split, order):
        x = x.reshape(*lead, 2, *split)
        return x.permute(*range(n), *[n + i for i in order]).reshape(*lead, 2, -1)

    # a token is (half, g, t) of (2, 4, 8), for the keys' scales t = (j, r) of (2, 4);
    # a byte of the values' codes is (n, q) of (16, 4): dims 8 n + 2 q and the next
    parts = [put(k[0], (64, 64), (0, 1)), put(v[0], (2, 4, 8, 16, 4), (4, 1, 3, 0, 2)),
             put(k[1], (2, 4, 2, 4, 4), (4, 1, 3, 0, 2)), put(v[1], (2, 4, 8, 4), (3, 1, 0, 2))]
    return torch.cat(parts, dim=-1).flatten(-2)


def _from_pages(pages):
    """Page bytes [..., 17408] -> (keys, values) fp32 [..., 128 tokens, 128]."""
    lead = pages.shape[:-1]
    x = pages.reshape(*lead, 2, UNIT_BYTES)
    n = len(lead) + 1

    def get(lo, hi, split, order, last):
        part = x[..., lo:hi].reshape(*lead, 2, *split)
        return part.permute(*range(n), *[n + i for i in order]).reshape(*lead, PAGE, last)

    k = _dequantise(x[..., :V_AT].reshape(*lead, PAGE, 64), get(KS_AT, VS_AT, (4, 4, 4, 2, 2), (3, 1, 4, 2, 0), 4))
    v = _dequantise(get(V_AT, KS_AT, (4, 4, 16, 2, 8), (3, 1, 4, 2, 0), 64),
                    get(VS_AT, UNIT_BYTES, (4, 4, 2, 8), (2, 1, 3, 0), 4))
    return k, v


def _bytes_of(slots, kv_heads):
    """Places in the pool of each (slot, kv head)'s key codes, value codes [T, KVH, 64], key scales
    and value scales [T, KVH, 4]."""
    page, tok = slots // PAGE, slots % UNIT
    base = (page[:, None] * kv_heads + torch.arange(kv_heads, device=DEV)) * 2 + (slots % PAGE // UNIT)[:, None]
    base = (base * UNIT_BYTES)[..., None]
    half, g, t = (tok // 32)[:, None, None], (tok // 8 % 4)[:, None, None], (tok % 8)[:, None, None]
    i, grp = torch.arange(64, device=DEV), torch.arange(4, device=DEV)
    return (base + tok[:, None, None] * 64 + i,
            base + V_AT + (((i % 4 * 4 + g) * 16 + i // 4) * 2 + half) * 8 + t,
            base + KS_AT + ((grp * 16 + g * 4 + t % 4) * 2 + half) * 2 + t // 4,
            base + VS_AT + ((grp * 4 + g) * 2 + half) * 8 + t)


def _plain_store(s, case):
    flat = s["cache"].view(-1)
    for (codes, e), at in zip((_quantise(s["k"]), _quantise(s["v"])), (0, 1)):
        places = _bytes_of(s["slots"], case["kv_heads"])
        flat[places[at]] = codes
        flat[places[at + 2]] = e
    return _plain_load(s, case)


def _plain_load(s, case):
    flat, dtype = s["cache"].view(-1), DT[case["dtype"]]
    kc, vc, ks, vs = _bytes_of(s["slots"], case["kv_heads"])
    return _dequantise(flat[kc], flat[ks]).to(dtype), _dequantise(flat[vc], flat[vs]).to(dtype)


def _rows_of(cache, table):
    """Keys and values fp32 [B, KVH, cols * PAGE, D] of the pages of each request."""
    k, v = _from_pages(cache[table.long()])  # [B, cols, KVH, PAGE, D]
    return tuple(x.transpose(1, 2).reshape(x.shape[0], x.shape[2], -1, D) for x in (k, v))


def _softmax(sc):
    """Scores with -inf where nothing attends -> probabilities (zeros for an empty row) and the
    log of the sum (-inf for an empty row)."""
    m = sc.amax(dim=-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = torch.exp(sc - m)
    z = e.sum(dim=-1, keepdim=True)
    return e / torch.where(z > 0, z, torch.ones_like(z)), (m + torch.log(z)).squeeze(-1)


def _plain_decode(s, case):
    n, h, b, kvh = case["q_len"], case["heads"], case["batch"], case["kv_heads"]
    q = s["q"].float().reshape(b, n, kvh, h // kvh, D).transpose(1, 2).reshape(b, kvh, -1, D)  # rows (token, head)
    cols = s["table"].shape[1]
    step = max(1, (1 << 30) // (cols * PAGE * kvh * D))  # requests at a time: 4 GB of keys
    j = torch.arange(cols * PAGE, device=DEV)
    outs, lses = [], []
    for at in range(0, b, step):
        k, v = _rows_of(s["cache"], s["table"][at:at + step])
        last = s["lens"][at:at + step, None] - n + 1 + torch.arange(n, device=DEV)  # keys that token i sees
        seen = j < last.repeat_interleave(h // kvh, dim=1)[:, None, :, None]
        sc = torch.matmul(q[at:at + step], k.transpose(2, 3)) * SCALE
        p, lse = _softmax(sc.masked_fill_(~seen, -math.inf))
        outs.append(torch.matmul(p, v))
        lses.append(lse)
    o, lse = torch.cat(outs), torch.cat(lses)
    o = o.reshape(b, kvh, n, h // kvh, D).transpose(1, 2).reshape(b * n, h, D)
    return o.to(s["q"].dtype), lse.reshape(b, kvh, n, h // kvh).transpose(1, 2).reshape(-1)


def _plain_cascade(s, case):
    b, h, kvh, p = case["batch"], case["heads"], case["kv_heads"], case["prefix"]
    g = h // kvh
    pk, pv = (x[0, :, :p] for x in _rows_of(s["cache"], s["ptable"]))  # [KVH, p, D]
    k, v = _rows_of(s["cache"], s["table"])
    q = s["q"].float().reshape(b, kvh, g, D)
    s1 = torch.matmul(q.transpose(0, 1).reshape(kvh, b * g, D), pk.transpose(1, 2))
    s1 = s1.reshape(kvh, b, g, p).transpose(0, 1)
    s2 = torch.matmul(q, k.transpose(2, 3))
    hidden = torch.arange(k.shape[2], device=DEV) >= s["lens"][:, None]
    s2 = s2.masked_fill_(hidden[:, None, None, :], -math.inf)
    w, lse = _softmax(torch.cat([s1, s2], dim=3).mul_(SCALE))
    o = torch.matmul(w[..., :p].transpose(0, 1).reshape(kvh, b * g, p), pv).reshape(kvh, b, g, D).transpose(0, 1)
    o = o + torch.matmul(w[..., p:], v)
    return o.reshape(b, h, D).to(s["q"].dtype), lse.reshape(-1)


# ---- the same in 64 bits --------------------------------------------------------------
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _values64(cache, slots, which):
    """Keys (which 0) or values (1) of the tokens at `slots`, float64 [T, KVH, 128], each byte fetched from
    its address."""
    kvh = cache.shape[1]
    d = torch.arange(D, device=DEV)
    row, tok = slots % PAGE // UNIT, slots % UNIT
    if which == 0:
        code_at = tok[:, None] * 64 + d // 2
        lane, tile = tok % 32 // 8 * 4 + tok % 4, tok // 32 * 2 + tok % 8 // 4
        scale_at = KS_AT + (d // GROUP) * 64 + (lane * 4 + tile)[:, None]
    else:
        of8 = tok % 32 // 8 * 256 + tok // 32 * 8 + tok % 8
        code_at = V_AT + (d % 8 // 2) * 1024 + (d // 8) * 16 + of8[:, None]
        scale_at = VS_AT + (d // GROUP) * 64 + (tok % 32 // 8 * 16 + tok // 32 * 8 + tok % 8)[:, None]
    lut = torch.tensor(_E2M1 + [-x for x in _E2M1], dtype=torch.float64, device=DEV)
    out = torch.empty(slots.shape[0], kvh, D, dtype=torch.float64, device=DEV)
    rows = cache.view(-1, UNIT_BYTES)
    for g in range(kvh):
        at = ((slots // PAGE * kvh + g) * 2 + row)[:, None]
        byte = rows[at, code_at].int()
        code = torch.where(d % 2 == 1, byte >> 4, byte & 15)
        e = rows[at, scale_at]
        out[:, g] = lut[code.long()] * torch.where(e == 255, math.nan, torch.exp2(e.double() - 127))
    return out


def _quantised64(x):
    """Float64 [T, KVH, 128] -> what its groups become in 4 bits, float64."""
    x = x.double().reshape(-1, GROUP)
    most = x.abs().amax(dim=1, keepdim=True)
    m, e = torch.frexp(most)  # most = m 2^e, m in [0.5, 1)
    e = torch.where(m > 0.875, e - 2, e - 3)  # 7 code units at most
    step = torch.exp2(torch.where(most > 0, e, -200).clamp(LOWEST - 127, HIGHEST - 127).double())
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    y = (x.abs() / step).clamp(max=6.0)
    hi = torch.searchsorted(grid, y.contiguous()).clamp(max=7)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - y, y - grid[lo]
    i = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return torch.copysign(grid[i] * step, x)


def _slots_of(row, n):
    """Slots of the first n tokens behind a block-table row."""
    j = torch.arange(n, device=DEV)
    return row.long()[j // PAGE] * PAGE + j % PAGE


def _part64(cache, row, n, q, upto):
    """Rows q [r, KVH, D] over the first n tokens behind a table row, row i seeing upto[i] of them ->
    (o [r, KVH, D], lse [r, KVH])."""
    r, kvh = q.shape[0], q.shape[1]
    o = torch.zeros(r, kvh, D, dtype=torch.float64, device=DEV)
    lse = torch.full((r, kvh), -math.inf, dtype=torch.float64, device=DEV)
    if n == 0:
        return o, lse
    slots = _slots_of(row, n)
    k, v = _values64(cache, slots, 0), _values64(cache, slots, 1)
    hidden = torch.arange(n, device=DEV)[None, :] >= upto[:, None]
    some = upto > 0
    for g in range(kvh):
        sc = (q[:, g].double() @ k[:, g].t().contiguous() * SCALE).masked_fill(hidden, -math.inf)
        lse[:, g] = torch.logsumexp(sc, dim=1)
        o[some, g] = torch.exp(sc[some] - lse[some, g][:, None]) @ v[:, g].contiguous()
    return o, lse


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "store":
        return tuple(_quantised64(s[x]).reshape(s[x].shape) for x in ("k", "v"))
    if op == "load":
        return tuple(_values64(s["cache"], s["slots"], x) for x in (0, 1))
    h, kvh = case["heads"], case["kv_heads"]
    g = h // kvh
    outs, lses = [], []
    if op == "decode":
        n = case["q_len"]
        for b, ln in enumerate(s["lens"].tolist()):
            q = s["q"][b * n:(b + 1) * n].reshape(n, kvh, g, D).transpose(1, 2).reshape(n * g, kvh, D)
            upto = (ln - n + 1 + torch.arange(n, device=DEV)).clamp(min=0).repeat_interleave(g)
            o, lse = _part64(s["cache"], s["table"][b], ln, q, upto)
            outs.append(o.reshape(n, g, kvh, D).transpose(1, 2).reshape(n, h, D))
            lses.append(lse.reshape(n, g, kvh).transpose(1, 2).reshape(n, h))
        return torch.cat(outs), torch.cat(lses).reshape(-1)
    batch, p = case["batch"], case["prefix"]
    rows = s["q"].reshape(batch, kvh, g, D).transpose(1, 2).reshape(batch * g, kvh, D)
    o1, l1 = _part64(s["cache"], s["ptable"][0], p, rows, torch.full((batch * g,), p, device=DEV))
    for b, ln in enumerate(s["lens"].tolist()):
        mine = slice(b * g, (b + 1) * g)
        o2, l2 = _part64(s["cache"], s["table"][b], ln, rows[mine], torch.full((g,), ln, device=DEV))
        lse = torch.logaddexp(l1[mine], l2)
        o = o1[mine] * torch.exp(l1[mine] - lse)[..., None] + o2 * torch.exp(l2 - lse)[..., None]
        outs.append(o.transpose(0, 1).reshape(1, h, D))
        lses.append(lse.transpose(0, 1).reshape(1, h))
    return torch.cat(outs), torch.cat(lses).reshape(-1)
