"""Measured cases of the quantised KV cache and of chunk attention.

Three operators: ``store`` (quantise K/V rows as they are written into the
paged cache, then read them back), ``load`` (read cached rows back to bf16)
and ``attention`` (a chunk of new tokens attends to a paged cache, bf16 or
quantised, followed by the chunk's own fresh rows where they are given).

With ``own`` false the operators run in their plain form: elementary torch
operations in float32, rounded once. With ``own`` true the same inputs go
through this package's entry points.

Quantised rows: one group per (token, kv head) with a power-of-two scale.
With a = the group's largest magnitude and M the format's largest value (448
for e4m3, 127 for int8), e is the smallest integer with a <= M * 2^e (clamped
to a range that keeps every dequantised value a normal bf16), the codes are
x * 2^-e rounded to nearest even, and the byte e + 127 is kept per group.
"""
import math
import os
import random
import sys

import torch

own = False

PAGE = 256          # cache slots per page, as the model runner allocates them
DIM = 128           # head dimension
FORMATS = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
MOST_WORK = 36864 * 32  # (token, kv head) rows of the largest store / load


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one new token of one sequence enters a grouped-query cache: latency only
        {"name": "store_e4m3_token", "op": "store", "format": "e4m3", "tokens": 1, "kv_heads": 4, "lengths": 1},
        # the rows of one dense step (16 sequences of 256-1024 prompt tokens + a 128-token block)
        {"name": "store_int8_step", "op": "store", "format": "int8", "tokens": 11902, "kv_heads": 32, "lengths": 2},
        # every token of 8 long sequences (4096 + 512) at once
        {"name": "store_e4m3_full", "op": "store", "format": "e4m3", "tokens": 36864, "kv_heads": 32, "lengths": 3},
        # the kept rows of 32 grouped-query sequences
        {"name": "load_int8_kept", "op": "load", "format": "int8", "tokens": 11213, "kv_heads": 4, "lengths": 4},
        # the kept rows of 8 long sequences at retention ratio 0.25
        {"name": "load_e4m3_long", "op": "load", "format": "e4m3", "tokens": 9152, "kv_heads": 32, "lengths": 5},
        # one sequence of 96 tokens decodes one token: the smallest attention call
        {"name": "step_bf16_one", "op": "attention", "format": "bf16", "heads": 32, "kv_heads": 32, "batch": 1,
         "q_lo": 1, "q_hi": 1, "c_lo": 96, "c_hi": 96, "fresh": False, "causal": True, "tables": True, "lengths": 6},
        # a batch of 32 grouped-query sequences decodes one token each
        {"name": "step_bf16_batch", "op": "attention", "format": "bf16", "heads": 28, "kv_heads": 4, "batch": 32,
         "q_lo": 1, "q_hi": 1, "c_lo": 128, "c_hi": 1024, "fresh": False, "causal": True, "tables": True, "lengths": 7},
        # 8 sequences decode one token each over long e4m3 caches, the new rows not stored yet
        {"name": "step_e4m3_long", "op": "attention", "format": "e4m3", "heads": 32, "kv_heads": 32, "batch": 8,
         "q_lo": 1, "q_hi": 1, "c_lo": 4096, "c_hi": 32768, "fresh": True, "causal": True, "tables": True,
         "lengths": 8},
        # the reuse step of a diffusion block: 32 block rows over kept cached rows + the block's own rows
        {"name": "reuse_e4m3_long", "op": "attention", "format": "e4m3", "heads": 32, "kv_heads": 32, "batch": 8,
         "q_lo": 32, "q_hi": 32, "c_lo": 1136, "c_hi": 1144, "fresh": True, "causal": False, "tables": False,
         "lengths": 9},
        # the same with grouped-query heads, 32 shorter sequences, int8
        {"name": "reuse_int8_batch", "op": "attention", "format": "int8", "heads": 28, "kv_heads": 4, "batch": 32,
         "q_lo": 32, "q_hi": 32, "c_lo": 176, "c_hi": 496, "fresh": True, "causal": False, "tables": False,
         "lengths": 10},
        # chunked prefill: up to 512 new tokens, already stored, over long bf16 contexts
        {"name": "chunk_bf16", "op": "attention", "format": "bf16", "heads": 28, "kv_heads": 4, "batch": 4,
         "q_lo": 300, "q_hi": 512, "c_lo": 2000, "c_hi": 4608, "fresh": False, "causal": True, "tables": True,
         "lengths": 11},
        # the largest: prefill chunks of up to 2048 tokens behind e4m3 contexts
        {"name": "prefill_e4m3", "op": "attention", "format": "e4m3", "heads": 32, "kv_heads": 32, "batch": 4,
         "q_lo": 1024, "q_hi": 2048, "c_lo": 1024, "c_hi": 6144, "fresh": True, "causal": True, "tables": True,
         "lengths": 12},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("store", "load", "attention", "attention", "attention", "attention"))
    if op != "attention":
        kv_heads = rng.choice((1, 2, 3, 4, 8, 32))
        return {"op": op, "format": rng.choice(("e4m3", "int8")), "tokens": _log(rng, 1, MOST_WORK // max(kv_heads, 4) // 8),
                "kv_heads": kv_heads, "lengths": rng.randrange(1 << 20)}
    heads, kv_heads = rng.choice(((32, 32), (28, 4), (8, 8), (7, 1), (16, 2), (12, 4), (32, 8), (3, 3)))
    kind = rng.choice(("step", "reuse", "chunk", "prefill"))
    q_hi = 1 if kind == "step" else _log(rng, 2, 64) if kind == "reuse" else _log(rng, 65, 512) if kind == "chunk" else _log(rng, 513, 2048)
    c_hi = _log(rng, 1, {"step": 32768, "reuse": 4096, "chunk": 8192, "prefill": 6144}[kind])
    batch = _log(rng, 1, {"step": 64, "reuse": 32, "chunk": 8, "prefill": 4}[kind])
    while batch > 1 and batch * c_hi * kv_heads > 8 * 20000 * 32:
        batch //= 2
    fresh = kind == "reuse" or rng.random() < 0.5
    return {"op": op, "format": rng.choice(("bf16", "e4m3", "int8")), "heads": heads, "kv_heads": kv_heads, "batch": batch,
            "q_lo": max(1, q_hi // rng.choice((1, 2, 7))), "q_hi": q_hi, "c_lo": c_hi // rng.choice((1, 2, 9)), "c_hi": c_hi,
            "fresh": fresh, "causal": kind != "reuse" and rng.random() < 0.8, "tables": kind != "reuse" and rng.random() < 0.7,
            "lengths": rng.randrange(1 << 20)}


def _lengths(case):
    """(query rows, cached rows, fresh rows) per sequence; without fresh rows the
    cached rows count the chunk's own, which were stored before the call."""
    r = random.Random(case["lengths"])
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["batch"])]
    c = [r.randint(case["c_lo"], case["c_hi"]) for _ in range(case["batch"])]
    return q, c, (q if case["fresh"] else [0] * case["batch"])


def _row_bytes(fmt):
    return 2 * DIM if fmt == "bf16" else DIM + 1


def work(case):
    if case["op"] != "attention":
        n, h = case["tokens"], case["kv_heads"]
        wide, narrow = 2 * n * h * DIM * 2, 2 * n * h * (DIM + 1)
        if case["op"] == "load":
            return {"bytes": wide + narrow + 4 * n, "flops": 0}
        return {"bytes": 2 * (wide + narrow) + 4 * n, "flops": 0}  # written, then read back
    q, c, f = _lengths(case)
    pairs = visible = 0
    for nq, nc, nf in zip(q, c, f):
        L = nc + nf
        if case["causal"]:
            pairs += sum(min(L, max(0, L - nq + i + 1)) for i in range(nq))
        else:
            pairs += nq * L
        visible += nc
    b = 2 * sum(q) * case["heads"] * DIM * 2                       # q, o
    b += 2 * visible * case["kv_heads"] * _row_bytes(case["format"])  # cached rows
    b += 2 * sum(f) * case["kv_heads"] * DIM * 2                   # fresh rows
    b += 4 * visible if not case["tables"] else 4 * sum(-(-x // PAGE) for x in c)
    return {"bytes": b, "flops": 4 * case["heads"] * DIM * pairs}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _rows(g, n, heads, dev):
    """K or V rows: normal values, with heads of different size (a factor of up
    to 8 between them) and a few large channels, as projections give them."""
    x = torch.randn(n, heads, DIM, generator=g, device=dev)
    x *= torch.exp2(torch.randint(-1, 3, (1, heads, 1), generator=g, device=dev).float())
    x[:, :, 5::61] *= 3.0
    return x.to(torch.bfloat16)


def _top(fmt):
    return (448.0, 119) if fmt == "e4m3" else (127.0, 121)


def _quantise(x, fmt):
    """Codes and exponent bytes of rows [..., D] (finite values)."""
    most, e_max = _top(fmt)
    a = x.float().abs().amax(-1)
    m, e = torch.frexp(a / most)                    # a / most = m 2^e, m in [0.5, 1)
    e = e - (m == 0.5).to(e.dtype)
    e = torch.where(torch.ldexp(torch.full_like(a, most), e) < a, e + 1, e)       # the quotient was rounded
    e = torch.where(torch.ldexp(torch.full_like(a, most), e - 1) >= a, e - 1, e)
    e = torch.where(a > 0, e, torch.full_like(e, -100)).clamp(-100, e_max)
    y = torch.ldexp(x.float(), -e.unsqueeze(-1)).clamp(-most, most)
    codes = y.to(torch.float8_e4m3fn) if fmt == "e4m3" else torch.round(y).to(torch.int8)
    return codes, (e + 127).to(torch.uint8)


def _cu(lens, dev):
    c = [0]
    for n in lens:
        c.append(c[-1] + n)
    return torch.tensor(c, dtype=torch.int32, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed * 7919 + case["lengths"])
    fmt, hk = case["format"], case["kv_heads"]
    s = {"op": case["op"], "format": fmt}
    if case["op"] != "attention":
        n = case["tokens"]
        pages = (n + PAGE - 1) // PAGE + 2
        slots = torch.randperm(pages * PAGE, generator=g, device=dev)[:n].to(torch.int32)
        slots[7::251] = -1                         # padded entries of a captured batch
        s["slots"] = slots
        s["k_cache"] = torch.zeros(pages, PAGE, hk, DIM, dtype=torch.int8, device=dev).view(FORMATS[fmt])
        s["v_cache"] = torch.zeros_like(s["k_cache"])
        s["k_exp"] = torch.zeros(pages, PAGE, hk, dtype=torch.uint8, device=dev)
        s["v_exp"] = torch.zeros_like(s["k_exp"])
        if case["op"] == "store":
            qkv = torch.empty(n, 3, hk, DIM, dtype=torch.bfloat16, device=dev)  # rows of a fused projection
            qkv[:, 1], qkv[:, 2] = _rows(g, n, hk, dev), _rows(g, n, hk, dev)
            s["key"], s["value"] = qkv[:, 1], qkv[:, 2]
        else:
            for cache, exp in (("k_cache", "k_exp"), ("v_cache", "v_exp")):
                codes, e = _quantise(_rows(g, pages * PAGE, hk, dev), fmt)
                s[cache], s[exp] = codes.view(pages, PAGE, hk, DIM), e.view(pages, PAGE, hk)
        s["key_out"] = torch.empty(n, hk, DIM, dtype=torch.bfloat16, device=dev)
        s["value_out"] = torch.empty_like(s["key_out"])
        return s
    q, c, f = _lengths(case)
    h = case["heads"]
    s["q"] = torch.randn(sum(q), h, DIM, generator=g, device=dev).to(torch.bfloat16)
    s["cu_q"], s["max_q"], s["causal"] = _cu(q, dev), max(q), case["causal"]
    s["k"] = s["v"] = s["cu_k"] = None
    if case["fresh"]:
        s["k"], s["v"], s["cu_k"] = _rows(g, sum(f), hk, dev), _rows(g, sum(f), hk, dev), s["cu_q"]
    pages_of = [(n + PAGE - 1) // PAGE for n in c]
    pages = sum(pages_of) + 1
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    rows = [_rows(g, pages * PAGE, hk, dev).view(pages, PAGE, hk, DIM) for _ in range(2)]
    s["k_exp"] = s["v_exp"] = None
    if fmt == "bf16":
        s["k_cache"], s["v_cache"] = rows
    else:
        (s["k_cache"], s["k_exp"]), (s["v_cache"], s["v_exp"]) = (_quantise(x, fmt) for x in rows)
    s["context"] = torch.tensor(c, dtype=torch.int32, device=dev)
    s["max_context"] = max(c)
    s["tables"] = s["slots"] = s["cu_slots"] = None
    ends = _cu(pages_of, dev).tolist()
    if case["tables"]:
        s["tables"] = torch.full((len(c), max(1, max(pages_of))), -1, dtype=torch.int32, device=dev)
        for b in range(len(c)):
            s["tables"][b, :pages_of[b]] = order[ends[b]:ends[b + 1]]
    else:
        # whole pages in sequence, the way the block manager hands them out; the last sequence's
        # slots are scattered
        every = (order.long().unsqueeze(1) * PAGE + torch.arange(PAGE, device=dev)).view(pages, PAGE)
        lists = [every[ends[b]:ends[b + 1]].reshape(-1)[:c[b]] for b in range(len(c))]
        lists[-1] = lists[-1][torch.randperm(c[-1], generator=g, device=dev)]
        s["slots"], s["cu_slots"] = torch.cat(lists).to(torch.int32), _cu(c, dev)
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _values(codes, exps):
    """What quantised rows stand for, float32."""
    scale = torch.ldexp(torch.ones_like(exps, dtype=torch.float32), exps.int() - 127) * (exps > 0)
    return codes.float() * scale.unsqueeze(-1)


def _plain_store(s):
    fmt, hk = s["format"], s["key"].shape[1]
    kept = s["slots"] >= 0
    at = s["slots"][kept].long()
    for x, cache, exp in (("key", "k_cache", "k_exp"), ("value", "v_cache", "v_exp")):
        codes, e = _quantise(s[x][kept], fmt)
        s[cache].view(torch.int8).view(-1, hk, DIM)[at] = codes.view(torch.int8)
        s[exp].view(-1, hk)[at] = e


def _plain_load(s):
    hk = s["k_exp"].shape[-1]
    kept = (s["slots"] >= 0).view(-1, 1, 1)
    at = s["slots"].clamp(min=0).long()
    out = []
    for cache, exp in (("k_cache", "k_exp"), ("v_cache", "v_exp")):
        codes = s[cache].view(torch.int8).view(-1, hk, DIM)[at].view(FORMATS[s["format"]])
        out.append((_values(codes, s[exp].view(-1, hk)[at]) * kept).to(torch.bfloat16))
    return out


def _cached(s, cache, exp, at):
    """float32 rows of the slots `at` (any shape) of a cache."""
    hk = s[cache].shape[2]
    if s[exp] is None:
        return s[cache].view(-1, hk, DIM)[at].float()
    codes = s[cache].view(torch.int8).view(-1, hk, DIM)[at].view(s[cache].dtype)
    return _values(codes, s[exp].view(-1, hk)[at])


def _plain_attention(s):
    q, ctx = s["q"], s["context"].long()
    dev, heads, hk = q.device, q.shape[1], s["k_cache"].shape[2]
    cu_q = s["cu_q"].long()
    nq = cu_q[1:] - cu_q[:-1]
    B, g = nq.numel(), heads // hk
    pos = torch.arange(s["max_context"], device=dev)
    if s["tables"] is not None:
        page = s["tables"].long().clamp(min=0)[:, pos // PAGE]
        at = page * PAGE + pos % PAGE
    else:
        at = s["slots"].long()[(s["cu_slots"].long()[:-1, None] + pos).clamp(max=s["slots"].numel() - 1)]
    keys, vals = _cached(s, "k_cache", "k_exp", at), _cached(s, "v_cache", "v_exp", at)
    there, place = pos < ctx[:, None], pos.expand(B, -1)
    total = ctx
    row = torch.arange(s["max_q"], device=dev)
    rows = (cu_q[:-1, None] + row).clamp(max=q.shape[0] - 1)
    if s["k"] is not None:
        keys, vals = torch.cat([keys, s["k"].float()[rows]], 1), torch.cat([vals, s["v"].float()[rows]], 1)
        there = torch.cat([there, row < nq[:, None]], 1)
        place = torch.cat([place, ctx[:, None] + row], 1)
        total = ctx + nq
    seen = there[:, None, :].expand(B, s["max_q"], -1)
    if s["causal"]:
        seen = seen & (place[:, None, :] <= (total - nq)[:, None, None] + row[:, None])
    qf = q.float()[rows].view(B, s["max_q"], hk, g, DIM).permute(0, 2, 3, 1, 4).reshape(B, hk, g * s["max_q"], DIM)
    sc = (qf @ keys.permute(0, 2, 3, 1)).view(B, hk, g, s["max_q"], -1) * DIM ** -0.5
    sc = sc.masked_fill(~seen[:, None, None], -math.inf)
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    del sc
    p /= p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = p.view(B, hk, g * s["max_q"], -1) @ vals.transpose(1, 2)
    o = o.view(B, hk, g, s["max_q"], DIM).permute(0, 3, 1, 2, 4).reshape(B, s["max_q"], heads, DIM)
    return o[row < nq[:, None]].to(torch.bfloat16)


def run(s):
    if own:
        return _own(s)
    if s["op"] == "attention":
        return _plain_attention(s)
    if s["op"] == "store":
        _plain_store(s)
    return _plain_load(s)


# ---------------------------------------------------------------------------
# the package's operators
# ---------------------------------------------------------------------------
_OPS = []


def _ops():
    if not _OPS:
        root = os.path.join(os.getcwd(), "dllm-serve_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        from dllmserve_b200 import ops
        _OPS.append(ops)
    return _OPS[0]


def _own(s):
    ops = _ops()
    if s["op"] == "attention":
        return ops.chunk_attention(
            s["q"], s["k_cache"], s["v_cache"], s["cu_q"], s["max_q"], causal=s["causal"], block_tables=s["tables"],
            context_lens=s["context"] if s["tables"] is not None else None, slots=s["slots"],
            cu_seqlens_slots=s["cu_slots"], max_context=s["max_context"], k=s["k"], v=s["v"], cu_seqlens_k=s["cu_k"],
            k_exp=s["k_exp"], v_exp=s["v_exp"])
    if s["op"] == "store":
        ops.store_kvcache_quant(s["key"], s["value"], s["k_cache"], s["v_cache"], s["k_exp"], s["v_exp"], s["slots"])
    ops.load_kvcache_quant(s["key_out"], s["value_out"], s["k_cache"], s["v_cache"], s["k_exp"], s["v_exp"], s["slots"])
    return [s["key_out"], s["value_out"]]


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _round_trip(x, fmt):
    """float64 values that quantised rows [n, heads, D] stand for."""
    most, e_max = (448.0, 119) if fmt == "e4m3" else (127.0, 121)
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    e = torch.full_like(a, -100.0)
    for t in range(-60, 61):          # inputs lie far inside this range
        e = torch.where(a > most * 2.0 ** (t - 1), torch.full_like(e, float(min(t, e_max))), e)
    unit = torch.exp2(e)
    y = x / unit
    if fmt == "int8":
        return torch.round(y).clamp(-127, 127) * unit
    size = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -20))).clamp(min=-6)
    size = torch.where(y.abs() < torch.exp2(size), (size - 1).clamp(min=-6), size)
    step = torch.exp2(size - 3)
    return (torch.round(y / step) * step).clamp(-448, 448) * unit


def _exact_rows(cache, exp, at):
    rows = cache.reshape(-1, cache.shape[2], DIM)
    if exp is None:
        return rows[at].double()
    scale = torch.exp2(exp.reshape(-1, exp.shape[2])[at].double() - 127.0)
    return rows.view(torch.int8)[at].view(cache.dtype).to(torch.float32).double() * scale.unsqueeze(-1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        gone = (s["slots"] < 0).view(-1, 1, 1)
        return [_round_trip(s[x], case["format"]).masked_fill(gone, 0.0) for x in ("key", "value")]
    if case["op"] == "load":
        gone, at = (s["slots"] < 0).view(-1, 1, 1), s["slots"].long().clamp(min=0)
        return [_exact_rows(s[c], s[e], at).masked_fill(gone, 0.0) for c, e in (("k_cache", "k_exp"), ("v_cache", "v_exp"))]
    nq, nc, nf = _lengths(case)
    heads, hk = case["heads"], case["kv_heads"]
    out, start, first = [], 0, 0
    for b in range(case["batch"]):
        if case["tables"]:
            n = torch.arange(nc[b], device="cuda")
            at = s["tables"][b].long()[n // PAGE] * PAGE + n % PAGE
        else:
            at = s["slots"][first:first + nc[b]].long()
        first += nc[b]
        K, V = _exact_rows(s["k_cache"], s["k_exp"], at), _exact_rows(s["v_cache"], s["v_exp"], at)
        Q = s["q"][start:start + nq[b]].double()
        if case["fresh"]:
            K = torch.cat([K, s["k"][start:start + nq[b]].double()])
            V = torch.cat([V, s["v"][start:start + nq[b]].double()])
        L = K.shape[0]
        limit = torch.full((nq[b],), L, device="cuda")
        if case["causal"]:
            limit = torch.arange(nq[b], device="cuda") + (L - nq[b] + 1)
        hidden = torch.arange(L, device="cuda") >= limit[:, None]
        o = torch.empty(nq[b], heads, DIM, dtype=torch.float64, device="cuda")
        for h in range(heads):
            kv = h // (heads // hk)
            a = (Q[:, h] @ K[:, kv].T) / math.sqrt(DIM)
            a.masked_fill_(hidden, -math.inf)
            a = torch.softmax(a, -1)
            a.masked_fill_((limit <= 0)[:, None], 0.0)
            o[:, h] = a @ V[:, kv]
        out.append(o)
        start += nq[b]
    return torch.cat(out)
