"""Plain 64-bit forms of the quantised KV cache and of chunk attention.

Written from the definitions, one sequence and one head at a time, with no
code of the package; the reference has neither (its cache is bf16, and its
regular attention branches call flash-attn, dllmserve/layers/attention.py:121-148).
"""
from __future__ import annotations

import math

import torch

TOP = {"e4m3": (448.0, 119), "int8": (127.0, 121)}


def exponent(row: torch.Tensor, fmt: str) -> int:
    """The smallest e with a <= M * 2^e, a the row's largest finite magnitude."""
    top, e_max = TOP[fmt]
    x = row.double().abs()  # (a row with a NaN has no value of its own: the cache marks it)
    x = x[torch.isfinite(x)]
    a = float(x.max()) if x.numel() else 0.0
    if a == 0.0:
        return -100
    e = math.frexp(a)[1] - math.frexp(top)[1] - 1
    while top * 2.0 ** e < a:
        e += 1
    return min(max(e, -100), e_max)


def round_code(y: torch.Tensor, fmt: str) -> torch.Tensor:
    """Nearest value of the format, ties to even, saturating; float64."""
    y = y.double()
    if fmt == "int8":
        return torch.nan_to_num(torch.round(y), nan=0.0, posinf=127.0, neginf=-127.0).clamp(-127, 127)
    # e4m3: 3 mantissa bits, smallest normal 2^-6
    mag = y.abs().clamp(min=2.0 ** -30, max=1024.0)
    e = torch.floor(torch.log2(mag))
    e = torch.where(torch.exp2(e) > mag, e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= mag, e + 1, e).clamp(min=-6)
    step = torch.exp2(e - 3)
    r = torch.round(y / step) * step
    return torch.where(torch.isnan(y), y, r.clamp(-448, 448))


def quantise(x: torch.Tensor, fmt: str):
    """(code values float64, exponents int) of rows [..., D]."""
    rows = x.reshape(-1, x.shape[-1])
    exps = torch.tensor([exponent(r, fmt) for r in rows], dtype=torch.int64)
    codes = round_code(rows.double() * torch.exp2(-exps.double())[:, None], fmt)
    return codes.reshape(x.shape), exps.reshape(x.shape[:-1])


def values(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    return codes.double() * torch.exp2(exps.double()).unsqueeze(-1)


def chunk_attention(q, keys, vals, scale, causal):
    """One sequence: q [Lq, H, D], keys/vals [L, Hkv, D] (any float type) ->
    (o, sum_j p_ij |v_j|, max_j sum_d |q_d k_jd| scale), all float64."""
    q, keys, vals = q.double(), keys.double(), vals.double()
    Lq, H, D = q.shape
    L, Hk, _ = keys.shape
    o = torch.zeros(Lq, H, D, dtype=torch.float64)
    mag = torch.zeros_like(o)
    big = torch.zeros(Lq, H, dtype=torch.float64)
    for i in range(Lq):
        n = min(L, max(0, L - Lq + i + 1)) if causal else L
        if n == 0:
            continue
        for h in range(H):
            kh, vh = keys[:n, h // (H // Hk)], vals[:n, h // (H // Hk)]
            s = (kh * q[i, h]).sum(-1) * scale
            p = torch.softmax(s, -1)
            o[i, h] = p @ vh
            mag[i, h] = p @ vh.abs()
            big[i, h] = ((kh * q[i, h]).abs().sum(-1) * scale).max()
    return o, mag, big


def small_probability_floor(vals, heads):
    """What a quantised cache's f16 probabilities add to the bound, [heads].

    Over a quantised cache p_j 2^(e_j - E + 15) is rounded to f16, E the largest
    exponent of the values met. Above 2^-14 that is 2^-11 of its value (the
    bound's 2^-8 covers it); below, at most half of f16's smallest step, 2^-25,
    which the product with the code c_j and the unit 2^(E - 15) turns into
    2^-25 |c_j| 2^(E - 15) <= 2^-40 M 2^E. E is the smallest with
    max |v| <= M 2^E, so M 2^E < 2 max |v|: at most 2^-39 max |v| for each of
    the sequence's keys (those a row does not see included: E may be theirs).
    It matters only where the output is that small against the head's largest
    value, as when every key of weight has a zero in that dimension."""
    top = vals.double().abs().amax((0, 2)) * vals.shape[0] * 2.0 ** -39 if vals.shape[0] else torch.zeros(vals.shape[1])
    return top.double().repeat_interleave(heads // vals.shape[1])


def attention_bound(o, mag, big, floor=None):
    """Largest error the operator's roundings explain, per output element.

    Probabilities are rounded to bf16 before the second product (2^-8 of each
    p_j v_j: 2^-8 sum p |v|) and the output once more (2^-8 |o|). The scores
    are float32 sums of 128 products: an error of at most 256 * 2^-24 *
    sum |q k| scale each (twice the usual bound, for accumulation in any order
    with truncation), which changes each probability by that fraction, in the
    numerator and in the normaliser; exponentials, sums and the final division
    add less than 2^-16 relative. ``floor`` [heads]: an absolute part."""
    e32 = 2 * 256 * 2.0 ** -24 * big.unsqueeze(-1) + 2.0 ** -16
    bound = (2.0 ** -8 + e32) * mag * 1.01 + 2.0 ** -8 * o.abs() * 1.01 + 1e-30
    return bound if floor is None else bound + floor.view(1, -1, 1)
