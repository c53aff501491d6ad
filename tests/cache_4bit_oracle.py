"""The 4-bit cache's operators and packed cross-attention restated in 64 bits on the CPU, from
their definitions."""

import math

import torch

SIZES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def nearest_e2m1(x):
    """float64 -> the e2m1 value next to it (ties to the even code, past 6 to 6), as float64."""
    a = x.abs()
    step = torch.where(a <= 2, 0.5, torch.where(a <= 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), x)


def needed_scale(group):
    """The smallest power of two that brings the largest |x| of a group to 6 or less."""
    largest = float(group.abs().max())
    if largest == 0.0:
        return 2.0**-100
    m, e = math.frexp(largest / 6)  # exact powers of two need no step up
    return min(max(2.0 ** (e - (m == 0.5)), 2.0**-100), 2.0**125)


def quantised(x):
    """What a cache holds of [..., D]: float64."""
    dim = x.shape[-1]
    x = torch.nn.functional.pad(x.double().cpu(), (0, -dim % 32)).unflatten(-1, (-1, 32))
    largest = x.abs().amax(dim=-1, keepdim=True)
    m, e = torch.frexp(largest / 6)  # exact powers of two need no step up
    e = (e - (m == 0.5).int()).masked_fill(largest == 0, -100).clamp(-100, 125)
    scale = torch.ldexp(torch.ones_like(largest), e)
    held = (nearest_e2m1(x / scale) * scale).masked_fill(~largest.isfinite(), math.nan)
    return held.flatten(-2)[..., :dim]


def append(values, key, value, slots):
    """Keys and values [NB, H, bs, D] (float64, in place) after the tokens at ``slots``."""
    nb, _, bs, _ = values[0].shape
    kept = [t for t, s in enumerate(slots.tolist()) if 0 <= s < nb * bs]
    for held, x in zip(values, (key, value)):
        q = quantised(x[kept])
        for i, t in enumerate(kept):
            held[int(slots[t]) // bs, :, int(slots[t]) % bs] = q[i]


def same(a, b):
    """Whether two float tensors hold the same values, NaN in the same places."""
    a, b = a.double().cpu(), b.double().cpu()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def softmax_rows(q, k, v, scale):
    """(out, sum_j p_j |v_j|, the largest sum_d |q_d k_jd| * |scale|) of [H, n, D] queries over
    [H, t, D] keys and values, in 64 bits."""
    p = torch.softmax(torch.matmul(q, k.transpose(1, 2)) * scale, dim=-1)
    size = torch.matmul(q.abs(), k.abs().transpose(1, 2)).amax(-1) * abs(scale)
    return torch.matmul(p, v), torch.matmul(p, v.abs()), size


def attend(query, values, lens, tables, scale):
    """``softmax_rows`` of each row [N, H, D] over its pages (rows without tokens: zeros)."""
    k, v = values
    nb, _, bs, _ = k.shape
    out = torch.zeros(query.shape, dtype=torch.float64)
    weight, size = torch.zeros_like(out), torch.zeros(query.shape[:2], dtype=torch.float64)
    for r, n in enumerate(lens):
        n = min(n, len(tables[r]) * bs)
        pages = [(b, min(bs, n - bs * i)) for i, b in enumerate(tables[r]) if bs * i < n]
        pages = [(b, c) for b, c in pages if 0 <= b < nb]
        if not pages:
            continue
        keys, vals = (torch.cat([x[b, :, :c] for b, c in pages], dim=1) for x in (k, v))
        o, w, s = softmax_rows(query[r].double().cpu()[:, None], keys, vals, scale)
        out[r], weight[r], size[r] = o[:, 0], w[:, 0], s[:, 0]
    return out, weight, size


def cross(query, key, value, query_starts, key_starts, scale):
    """The same for packed runs [T, H, D] over [S, H, D]."""
    out = torch.zeros(query.shape, dtype=torch.float64)
    weight, size = torch.zeros_like(out), torch.zeros(query.shape[:2], dtype=torch.float64)
    for a, b, c, d in zip(query_starts, query_starts[1:], key_starts, key_starts[1:]):
        if a == b or c == d:
            continue
        o, w, s = softmax_rows(*(x.double().cpu().transpose(0, 1) for x in
                                 (query[a:b], key[c:d], value[c:d])), scale)
        out[a:b], weight[a:b], size[a:b] = o.transpose(0, 1), w.transpose(0, 1), s.T
    return out, weight, size


def tolerance(dtype, products, longest, kept, out, weight, size):
    """Half a step of the output's type (below its smallest normal number t steps are t eps, whatever
    the value: half of one is t eps / 2, fp16's 2^-14 2^-10 / 2 = 2^-25, and a value that the
    relative half step does not cover is at most that far from the nearest), and of sum p|v|
    what 32-bit sums leave: a score is a sum
    of ``products`` products (and two scalings) of total size ``size``, off by (products + 4) 2^-24
    of it, which moves its weight by that much (numerator and normaliser: twice); weights are
    kept to ``kept`` (the normaliser may sum them unrounded), and their exponential is good to
    2^-22; sums over tokens run in chains of at most longest / 2 products and 64 partial sums
    more, each addition off by 2^-24 of what it adds to, numerator and normaliser."""
    half = torch.finfo(dtype).eps / 2
    inner = (2 * ((products + 4) * 2.0**-24 * size + 2.0**-22) + kept
             + (longest / 2 + 64) * 2.0**-23)
    subnormal = torch.finfo(dtype).tiny * half
    return half * out.abs() + inner[..., None] * weight * (1 + half) + subnormal + 1e-30


def attend_tolerance(dtype, dim, longest, *found):
    """Over a 4-bit cache: queries as one (bf16), two (fp16) or three bf16 terms, weights as two
    (2^-17) or, for fp32, three (2^-25)."""
    terms = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[dtype]
    kept = 2.0**-25 if dtype == torch.float32 else 2.0**-17
    return tolerance(dtype, terms * dim, longest, kept, *found)


def cross_tolerance(dtype, dim, longest, *found):
    """Packed runs: 16-bit operands as they are and weights rounded to their type; fp32 as three
    rounded terms (2^-26 each, twice) with six products, the others 2^-26 of the whole."""
    if dtype == torch.float32:
        return tolerance(dtype, 6 * dim, longest, 3 * 2.0**-26, *found)
    return tolerance(dtype, dim, longest, torch.finfo(dtype).eps / 2, *found)
