"""The latent-attention operators as measurable calls.

A latent cache holds one row of 576 numbers a token for all heads: a normed latent of
512, from which keys and values are made, and 64 rotated key dims. Four operators work
on it: writing a step's tokens (``latent_cache_write``), attention in the absorbed form
over pages of 128 tokens (``latent_decode``), the same for a batch that shares a prefix
(``latent_cascade_decode``), and the expanded form, with the keys and values of each
head laid out, for prompts (``latent_prefill``).

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
R, P = 512, 64      # latent dims, rotated dims: a cache row is R + P
D = 128             # dims of a head's own key part and of its value, expanded
PAGE = 128          # tokens per page
SCALE = 1.0 / math.sqrt(D + P)
MAX_SUFFIX = 4096
MAX_POS = 32768
EPS = 1e-6
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases --------------------------------------------------------------------------
def listed():
    return [
        # The tokens of one decode step of 64 sequences: all launch latency.
        _write("write-t64", 64, "bf16", True),
        # A prefill chunk's tokens, rotated in halves.
        _write("write-t8192", 8192, "bf16", False),
        # One sequence on a tensor-parallel shard with 16 heads: the smallest attention call.
        _decode("decode-b1-h16", 1, 1, 16, 1300, "bf16"),
        # A shard's decode batch with long, ragged sequences: bound by reading the cache.
        _decode("decode-b48-h16", 48, 1, 16, 12000, "fp16"),
        # Three tokens a sequence (drafted ones under verification), causal among themselves.
        _decode("decode-b24-h32-q3", 24, 3, 32, 5000, "bf16"),
        # Every head of a large model on one GPU: as much arithmetic as memory traffic.
        _decode("decode-b64-h128", 64, 1, 128, 6000, "bf16"),
        # A small batch on a short system prompt.
        _cascade("cascade-b8-h16", 8, 16, 2048, 256, "bf16"),
        # 64 sequences on a shared 8192-token prefix, suffixes of mean 512: the batch and
        # lengths of this repository's benchmark.
        _cascade("cascade-b64-h32", 64, 32, 8192, 512, "bf16"),
        # The largest call: all heads, a batch and a prefix that are no multiples of anything.
        _cascade("cascade-b117-h128", 117, 128, 16001, 512, "fp16"),
        # A short prompt alone.
        _prefill("prefill-t147-h16", 1, 147, 0, 16, True, "bf16"),
        # Ragged prompts that continue cached context, expanded together.
        _prefill("prefill-b13-ragged", 13, 900, 700, 16, True, "fp16"),
        # A long prompt.
        _prefill("prefill-t6000-h32", 1, 6000, 0, 32, True, "bf16"),
    ]


def _write(name, tokens, dtype, interleaved):
    return {"name": name, "op": "write", "tokens": tokens, "dtype": dtype, "interleaved": interleaved}


def _decode(name, batch, q_len, heads, kv, dtype):
    return {"name": name, "op": "decode", "batch": batch, "q_len": q_len, "heads": heads, "kv": kv, "dtype": dtype}


def _cascade(name, batch, heads, prefix, mean, dtype):
    return {"name": name, "op": "cascade", "batch": batch, "heads": heads, "prefix": prefix, "suffix_mean": mean,
            "dtype": dtype}


def _prefill(name, batch, q, context, heads, causal, dtype):
    return {"name": name, "op": "prefill", "batch": batch, "q": q, "context": context, "heads": heads,
            "causal": causal, "dtype": dtype}


def draw(rng):
    """One more case of the ranges the listed ones stand for."""
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["write", "decode", "decode", "decode", "cascade", "cascade", "prefill", "prefill"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    heads = rng.choice([8, 16, 20, 32, 40, 64, 128])
    if op == "write":
        c = _write("", log(1, 8192), dtype, rng.random() < 0.5)
    elif op == "decode":
        batch, q_len = log(1, 256), rng.choice([1, 1, 2, 4, 7])
        c = _decode("", batch, q_len, heads, log(1, min(16384, 400000 // batch)), dtype)
    elif op == "cascade":
        c = _cascade("", log(1, 117), heads, log(128, 16000), log(32, 512), dtype)
    else:
        batch = log(1, 16)
        q = log(1, 6000 // batch)
        c = _prefill("", batch, q, rng.choice([0, 0, log(1, max(1, 8000 // batch))]), min(heads, 32),
                     rng.random() < 0.75, dtype)
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


def _prompt_lens(case):
    """(query lengths, key lengths) of a prefill call's requests: ragged in [q / 4, q], each
    behind up to `context` tokens."""
    rng = np.random.default_rng(case["batch"] * 8191 + case["q"])
    ql = rng.integers(max(1, case["q"] // 4), case["q"] + 1, size=case["batch"])
    ql[0] = case["q"]
    kl = ql + (rng.integers(0, case["context"] + 1, size=case["batch"]) if case["context"] else 0)
    return ql.astype(np.int64), kl.astype(np.int64)


def _pages(lens):
    return (np.asarray(lens) + PAGE - 1) // PAGE


def _pairs(ql, kl, causal):
    """(query, key) pairs that attend, over all requests, of one head."""
    if not causal:
        return int((ql * kl).sum())
    n = 0
    for q, k in zip(ql.tolist(), kl.tolist()):
        first = k - q + 1  # keys that the first query sees; below 1 for queries in front of all keys
        a, b = max(first, 0), max(k, 0)
        n += (b * (b + 1) - a * (a - 1)) // 2 if first >= 0 else b * (b + 1) // 2
    return n


def work(case):
    op = case["op"]
    if op == "write":
        t = case["tokens"]
        return {"bytes": t * (2 * 2 * (R + P) + 4 * P + 16) + 2 * R, "flops": t * (4 * R + 6 * (P // 2))}
    h = case["heads"]
    if op == "decode":
        lens = _lens(case)
        rows = case["batch"] * case["q_len"] * h
        ql = np.full_like(lens, case["q_len"])
        return {"bytes": int(lens.sum()) * 2 * (R + P) + rows * (2 * (R + P) + 2 * R + 4)
                + int(_pages(lens).sum()) * 4 + case["batch"] * 8,
                "flops": 2 * (R + P + R) * h * _pairs(ql, lens, True)}
    if op == "cascade":
        lens, p = _suffix_lens(case), case["prefix"]
        rows = case["batch"] * h
        return {"bytes": (int(lens.sum()) + p) * 2 * (R + P) + rows * (2 * (R + P) + 2 * R + 4)
                + (int(_pages(lens).sum()) + int(_pages(p))) * 4 + (case["batch"] + 1) * 8,
                "flops": 2 * (R + P + R) * h * (int(lens.sum()) + case["batch"] * p)}
    ql, kl = _prompt_lens(case)
    t, s = int(ql.sum()), int(kl.sum())
    return {"bytes": 2 * t * h * (D + P + D) + 4 * t * h + 2 * s * (2 * h * D + P) + 16 * case["batch"],
            "flops": 2 * (D + P + D) * h * _pairs(ql, kl, case["causal"])}


# ---- inputs -------------------------------------------------------------------------
class _Gen:
    """Seeded device normals and host permutations."""

    def __init__(self, seed, dtype):
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.rng = np.random.default_rng(seed)
        self.dtype = dtype

    def normal(self, *shape, dtype=None, std=1.0):
        return torch.empty(*shape, device=DEV, dtype=dtype or self.dtype).normal_(0.0, std, generator=self.g)


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


def _angles():
    """cos | sin of every position and pair, fp32 [MAX_POS, P]."""
    inv = 10000.0 ** (-np.arange(0, P, 2, dtype=np.float64) / P)
    a = np.arange(MAX_POS, dtype=np.float64)[:, None] * inv[None, :]
    return _dev(np.concatenate([np.cos(a), np.sin(a)], axis=1), torch.float32)


def prepare(case, seed):
    gen = _Gen(seed, DT[case["dtype"]])
    op = case["op"]
    s = {"case": case}
    if op == "write":
        t = case["tokens"]
        blocks = t // PAGE + 8
        # the projection's output holds other columns beside the latent's
        s["kv"] = gen.normal(t, R + P + 128, std=0.7)[:, 64:64 + R + P]
        s["gamma"] = (1.0 + gen.normal(R, dtype=torch.float32, std=0.1)).to(gen.dtype)
        s["cos_sin"] = _angles()
        s["positions"] = _dev(gen.rng.permutation(MAX_POS)[:t], torch.int64)
        s["slots"] = _dev(gen.rng.permutation(blocks * PAGE)[:t], torch.int64)
        s["cache"] = gen.normal(blocks, PAGE, R + P)
        return s
    h = case["heads"]
    if op == "prefill":
        ql, kl = _prompt_lens(case)
        order = gen.rng.permutation(case["batch"])
        ql, kl = ql[order], kl[order]
        t, n = int(ql.sum()), int(kl.sum())
        s["q"] = gen.normal(t, h, D + P)
        kv = gen.normal(n, h, 2 * D)  # the up-projection's output: a head's key part, then its value
        s["k"], s["v"] = kv[..., :D], kv[..., D:]
        s["kr"] = gen.normal(n, P)
        s["q_lens"], s["kv_lens"] = _dev(ql, torch.int64), _dev(kl, torch.int64)
        return s
    if op == "decode":
        lens = gen.rng.permutation(_lens(case))
        table, blocks = _tables(gen, lens)
        s["q"] = gen.normal(case["batch"] * case["q_len"], h, R + P)
    else:
        lens = gen.rng.permutation(_suffix_lens(case))
        both, blocks = _tables(gen, np.concatenate([[case["prefix"]], lens]))
        s["ptable"] = _dev(both[:1, :int(_pages(case["prefix"]))], torch.int32)
        table = both[1:, :max(1, int(_pages(lens).max()))]
        s["plen"] = torch.tensor([case["prefix"]], dtype=torch.int64, device=DEV)
        s["q"] = gen.normal(case["batch"], h, R + P)
    s["cache"] = gen.normal(blocks, PAGE, R + P)
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
    if op == "write":
        torch.ops.npu.latent_cache_write(s["kv"], s["gamma"], s["cos_sin"], s["positions"], s["slots"], s["cache"],
                                         EPS, case["interleaved"])
        return s["cache"]
    if op == "decode":
        return torch.ops.npu.latent_decode(s["q"], s["cache"], s["table"], s["lens"], SCALE, case["q_len"])
    if op == "cascade":
        return torch.ops.npu.latent_cascade_decode(s["q"], s["cache"], s["ptable"], s["plen"], s["cache"],
                                                   s["table"], s["lens"], SCALE)
    return torch.ops.npu.latent_prefill(s["q"], s["k"], s["kr"], s["v"], s["q_lens"], s["kv_lens"], SCALE,
                                        case["causal"])


def _run_plain(s):
    case = s["case"]
    return {"write": _plain_write, "decode": _plain_decode, "cascade": _plain_cascade,
            "prefill": _plain_prefill}[case["op"]](s, case)


def _plain_write(s, case):
    x = s["kv"].float()
    c, r = x[:, :R], x[:, R:]
    c = c * torch.rsqrt(c.square().mean(dim=1, keepdim=True) + EPS) * s["gamma"].float()
    cs = s["cos_sin"][s["positions"]]
    cos, sin = cs[:, :P // 2], cs[:, P // 2:]
    if case["interleaved"]:
        a, b = r[:, 0::2], r[:, 1::2]
        r = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).reshape(-1, P)
    else:
        a, b = r[:, :P // 2], r[:, P // 2:]
        r = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=1)
    s["cache"].view(-1, R + P)[s["slots"]] = torch.cat([c, r], dim=1).to(s["cache"].dtype)
    return s["cache"]


def _softmax(sc):
    """Scores with -inf where nothing attends -> probabilities (zeros for an empty row) and the
    log of the sum (-inf for an empty row)."""
    m = sc.amax(dim=-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    e = torch.exp(sc - m)
    z = e.sum(dim=-1, keepdim=True)
    return e / torch.where(z > 0, z, torch.ones_like(z)), (m + torch.log(z)).squeeze(-1)


def _rows_of(cache, table):
    """[B, cols * PAGE, R + P] fp32 of the pages of each request."""
    return cache[table.long()].reshape(table.shape[0], -1, R + P).float()


def _plain_decode(s, case):
    n, h, b = case["q_len"], case["heads"], case["batch"]
    c = _rows_of(s["cache"], s["table"])
    q = s["q"].float().reshape(b, n * h, R + P)
    sc = torch.bmm(q, c.transpose(1, 2)) * SCALE
    j = torch.arange(c.shape[1], device=DEV)
    last = s["lens"][:, None] - n + 1 + torch.arange(n, device=DEV)  # keys that token i sees
    seen = (j < last.repeat_interleave(h, dim=1)[:, :, None])
    p, lse = _softmax(sc.masked_fill_(~seen, -math.inf))
    o = torch.bmm(p, c[..., :R])
    return o.reshape(b * n, h, R).to(s["q"].dtype), lse.reshape(-1)


def _plain_cascade(s, case):
    b, h, p = case["batch"], case["heads"], case["prefix"]
    pre = _rows_of(s["cache"], s["ptable"])[0, :p]
    c = _rows_of(s["cache"], s["table"])
    q = s["q"].float()
    s1 = (q.reshape(b * h, R + P) @ pre.t()).reshape(b, h, p)
    s2 = torch.bmm(q, c.transpose(1, 2))
    j = torch.arange(c.shape[1], device=DEV)
    s2 = s2.masked_fill_((j >= s["lens"][:, None])[:, None, :], -math.inf)
    w, lse = _softmax(torch.cat([s1, s2], dim=2) * SCALE)
    o = (w[..., :p].reshape(b * h, p) @ pre[:, :R]).reshape(b, h, R) + torch.bmm(w[..., p:], c[..., :R])
    return o.to(s["q"].dtype), lse.reshape(-1)


def _padded(x, start, lens, most):
    """Packed rows [T, ...] -> [B, most, ...] fp32; places past a request's end repeat its last row."""
    at = start[:, None] + torch.minimum(torch.arange(most, device=DEV), lens[:, None] - 1)
    return x[at.clamp_min(0)].float()


def _plain_prefill(s, case):
    h = case["heads"]
    ql, kl = s["q_lens"], s["kv_lens"]
    sizes = _prompt_lens(case)  # a serving process knows its requests' lengths on the host too
    qm, km = int(sizes[0].max()), int(sizes[1].max())
    qs, ks = torch.cumsum(ql, 0) - ql, torch.cumsum(kl, 0) - kl
    q = _padded(s["q"], qs, ql, qm).permute(0, 2, 1, 3)  # [B, h, qm, 192]
    k = _padded(s["k"], ks, kl, km).permute(0, 2, 1, 3)
    v = _padded(s["v"], ks, kl, km).permute(0, 2, 1, 3)
    kr = _padded(s["kr"], ks, kl, km)[:, None].expand(-1, h, -1, -1)
    sc = torch.matmul(q, torch.cat([k, kr], dim=3).transpose(2, 3)).mul_(SCALE)
    i, j = torch.arange(qm, device=DEV), torch.arange(km, device=DEV)
    most = (kl - ql)[:, None] + i + 1 if case["causal"] else kl[:, None].expand(-1, qm)
    seen = j < torch.minimum(most, kl[:, None])[:, :, None]
    w, lse = _softmax(sc.masked_fill_(~seen[:, None], -math.inf))
    o = torch.matmul(w, v).permute(0, 2, 1, 3)  # [B, qm, h, D]
    t = torch.arange(s["q"].shape[0], device=DEV)
    b = (t[:, None] >= (qs + ql)[None, :]).sum(dim=1)  # the request of each packed row
    return o[b, t - qs[b]].to(s["q"].dtype), lse.permute(0, 2, 1)[b, t - qs[b]].reshape(-1)


# ---- the same in 64 bits --------------------------------------------------------------
def _attend64(q, k, v, first, causal):
    """q [n, h, a], k [m, h or 1, a], v [m, h or 1, d] -> o [n, h, d], lse [n, h] in fp64; token i sees
    first + i keys when causal, else all."""
    n, h = q.shape[0], q.shape[1]
    o = torch.zeros(n, h, v.shape[2], dtype=torch.float64, device=DEV)
    lse = torch.full((n, h), -math.inf, dtype=torch.float64, device=DEV)
    m = k.shape[0]
    if m == 0:
        return o, lse
    upto = torch.full((n,), m, device=DEV) if not causal else (first + torch.arange(n, device=DEV)).clamp(0, m)
    hidden = torch.arange(m, device=DEV)[None, :] >= upto[:, None]
    for g in range(h):
        kg, vg = k[:, g % k.shape[1]].double(), v[:, g % v.shape[1]].double()
        sc = (q[:, g].double() @ kg.t().contiguous() * SCALE).masked_fill(hidden, -math.inf)
        lse[:, g] = torch.logsumexp(sc, dim=1)
        some = upto > 0
        o[some, g] = torch.exp(sc[some] - lse[some, g][:, None]) @ vg
    return o, lse


def _cached(s, row, n):
    """The first n cached tokens behind a block-table row, [n, 1, R + P]."""
    return s["cache"][row[:(n + PAGE - 1) // PAGE].long()].reshape(-1, 1, R + P)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "write":
        x = s["kv"].double()
        out = s["cache"].double().view(-1, R + P)
        c = x[:, :R]
        out[s["slots"], :R] = c / (c.pow(2).sum(dim=1, keepdim=True) / R + EPS).sqrt() * s["gamma"].double()
        z = torch.complex(*(x[:, R::2], x[:, R + 1::2]) if case["interleaved"]
                          else (x[:, R:R + P // 2], x[:, R + P // 2:]))
        turn = s["cos_sin"][s["positions"]].double()
        z = z * torch.complex(turn[:, :P // 2], turn[:, P // 2:])
        at = torch.arange(P // 2, device=DEV)
        out[s["slots"][:, None], R + (2 * at if case["interleaved"] else at)] = z.real
        out[s["slots"][:, None], R + (2 * at + 1 if case["interleaved"] else at + P // 2)] = z.imag
        return out.view(s["cache"].shape)
    outs = []
    if op == "prefill":
        at_q = at_k = 0
        for n, m in zip(s["q_lens"].tolist(), s["kv_lens"].tolist()):
            k, v, kr = s["k"][at_k:at_k + m], s["v"][at_k:at_k + m], s["kr"][at_k:at_k + m]
            k = torch.cat([k, kr[:, None].expand(-1, case["heads"], -1)], dim=2)
            outs.append(_attend64(s["q"][at_q:at_q + n], k, v, m - n + 1, case["causal"]))
            at_q, at_k = at_q + n, at_k + m
    elif op == "decode":
        n = case["q_len"]
        for b, ln in enumerate(s["lens"].tolist()):
            c = _cached(s, s["table"][b], ln)
            # all heads read the same rows: one product for the rows of every head
            q = s["q"][b * n:(b + 1) * n]
            parts = [_attend64(q[i].unsqueeze(1), c[:max(0, ln - n + 1 + i)], c[:max(0, ln - n + 1 + i), :, :R], 0, False)
                     for i in range(n)]
            outs += [(o.reshape(1, -1, R), lse.reshape(1, -1)) for o, lse in parts]
    else:
        p = case["prefix"]
        o1, l1 = _attend64(s["q"].reshape(-1, 1, R + P), _cached(s, s["ptable"][0], p),
                           _cached(s, s["ptable"][0], p)[..., :R], 0, False)
        o1, l1 = o1.reshape(case["batch"], -1, R), l1.reshape(case["batch"], -1)
        for b, ln in enumerate(s["lens"].tolist()):
            c = _cached(s, s["table"][b], ln)
            o2, l2 = _attend64(s["q"][b].unsqueeze(1), c, c[..., :R], 0, False)
            o2, l2 = o2.reshape(-1, R), l2.reshape(-1)
            lse = torch.logaddexp(l1[b], l2)
            outs.append(((o1[b] * torch.exp(l1[b] - lse)[:, None] + o2 * torch.exp(l2 - lse)[:, None])[None], lse[None]))
    return torch.cat([o for o, _ in outs]), torch.cat([x for _, x in outs]).reshape(-1)
