"""The 8-bit cache's operators restated in 64 bits on the CPU, from their definitions."""

import math

import torch

E4M3 = torch.float8_e4m3fn


def nearest_e4m3(x):
    """float64 -> the e4m3 value next to it (ties to even), as float64; NaN for non-finite."""
    a = x.abs().clamp(min=2.0**-6)
    mantissa, exponent = torch.frexp(a)  # a = mantissa * 2^exponent, mantissa in [0.5, 1)
    step = torch.ldexp(torch.ones_like(a), exponent - 4)
    return torch.where(x.isfinite(), torch.round(x / step) * step, math.nan)


def needed_scale(x):
    """The smallest power of two that brings the largest finite |x| to 448 or less."""
    finite = x[x.isfinite()]
    largest = float(finite.abs().max()) if finite.numel() else 0.0
    if largest == 0.0:
        return 2.0**-100
    e = math.frexp(largest / 448)
    return max(2.0**-100, 2.0 ** (e[1] - (1 if e[0] == 0.5 else 0)))


class Cache:
    """K and V as float64 quantised values [NB, H, bs, D] in token order, and scales."""

    def __init__(self, k, v, scales):
        self.q = [k.clone(), v.clone()]
        self.scales = scales.double().clone()

    @classmethod
    def of(cls, k_cache, v_cache, scales):
        from vflorence_amd import hip_attn

        return cls(k_cache.cpu().float().double(),
                   hip_attn.v_cache_logical(v_cache.cpu().view(torch.uint8)).view(E4M3).float()
                   .double(), scales.cpu())

    def append(self, key, value, slots):
        nb, heads, bs, _ = self.q[0].shape
        i, slots = 0, slots.tolist()
        while i < len(slots):
            if not 0 <= slots[i] < nb * bs:
                i += 1
                continue
            block, j = slots[i] // bs, i
            while j < len(slots) and 0 <= slots[j] < nb * bs and slots[j] // bs == block:
                j += 1
            taken = {s % bs: t for t, s in enumerate(slots[i:j], i)}  # offset: its last token
            offsets = list(taken)
            for n, x in enumerate((key, value)):
                x = x[list(taken.values())].double().cpu()
                for h in range(heads):
                    old = 0.0 if 0 in offsets else float(self.scales[block, h, n])
                    new = max(old, needed_scale(x[:, h]))
                    q = self.q[n][block, h]
                    q = torch.zeros_like(q) if 0 in offsets else nearest_e4m3(q * (old / new))
                    for o, row in zip(offsets, x[:, h]):
                        q[o] = nearest_e4m3(row / new)
                    self.q[n][block, h] = q
                    self.scales[block, h, n] = new
            i = j

    def values(self):
        s = self.scales[..., None, None]
        return self.q[0] * s[:, :, 0], self.q[1] * s[:, :, 1]


def attend(query, values, lens, tables, scale):
    """(out, sum_j p_j |v_j|, the largest sum_d |q_d k_jd| * |scale|) in 64 bits."""
    k, v = values
    nb, heads, bs, dim = k.shape
    out = torch.zeros(query.shape, dtype=torch.float64)
    weight = torch.zeros_like(out)
    size = torch.zeros(query.shape[:2], dtype=torch.float64)
    for r, n in enumerate(lens):
        n = min(n, len(tables[r]) * bs)
        pages = [(b, min(bs, n - bs * i)) for i, b in enumerate(tables[r]) if bs * i < n]
        pages = [(b, c) for b, c in pages if 0 <= b < nb]
        if not pages:
            continue
        keys = torch.cat([k[b, :, :c] for b, c in pages], dim=1)
        vals = torch.cat([v[b, :, :c] for b, c in pages], dim=1)
        q = query[r].double().cpu()
        p = torch.softmax(torch.einsum("hd,htd->ht", q, keys) * scale, dim=-1)
        out[r] = torch.einsum("ht,htd->hd", p, vals)
        weight[r] = torch.einsum("ht,htd->hd", p, vals.abs())
        size[r] = torch.einsum("hd,htd->ht", q.abs(), keys.abs()).amax(-1) * abs(scale)
    return out, weight, size


def attend_tolerance(dtype, dim, longest, out, weight, size):
    """Half a step of the output's type, and of sum p|v| what fp32 sums leave: a score is a sum
    of `dim` products (and two scalings) of total size `size`, off by (dim + 4) 2^-24 of it,
    which moves its weight by that much (numerator and normaliser: twice); weights are kept
    to 2^-17, or 2^-25 for fp32 outputs, and their exponential is good to 2^-22; the sums over
    tokens run in chains of 32 a lane's share of (longest / 8), 16 and 8 partial sums more."""
    half = torch.finfo(dtype).eps / 2
    kept = 2.0**-25 if dtype == torch.float32 else 2.0**-17
    inner = 2 * ((dim + 4) * 2.0**-24 * size + 2.0**-22) + kept + (longest / 8 + 24) * 2.0**-23
    return half * out.abs() + inner[..., None] * weight * (1 + half) + 1e-30
