"""Attention over 4-bit caches whose scales stand at the ends of their range, against the
definition in 64 bits."""

import pytest
import torch

from tests.cache_4bit_oracle import attend, attend_tolerance
from tests.test_cache_4bit_gpu import DEV, queries, random_cache, run_attention, values_of

pytestmark = pytest.mark.gpu


def cache_of(gen, blocks, heads, bs, dim, low, high):
    """A cache whose values' scales are 2^low to 2^high; its keys' are 2^-4 to 1."""
    cache = random_cache(gen, blocks, heads, bs, dim)
    groups = -(-dim // 32)
    scales = cache.view(blocks, -1)[:, heads * bs * groups * 32:]
    of_values = scales.view(blocks, heads, bs // 16, 4, 2, groups, 4)[:, :, :, :, 1]
    of_values.copy_(torch.randint(127 + low, 128 + high, of_values.shape, generator=gen))
    return cache


def check(query, cache, lens, tables, scale, **kw):
    out = run_attention(query, cache, lens, tables, scale, **kw)
    dim = query.shape[2]
    found = attend(query, values_of(cache, dim), lens, tables, scale)
    # In place of the oracle's allowance for results near 0: weights times V's scale are taken down
    # by 2^-6 and end as multiples of bf16's least number, 2^-133, off by half of one, a code of up
    # to 6 a token; the weights' sum is 1 or more.
    limit = attend_tolerance(query.dtype, dim, max(lens), *found) - 1e-30
    limit += max(lens) * 6 * 2.0**-128
    error = (out.double().cpu() - found[0]).abs()
    assert bool((error <= limit).all()), float((error / limit).max())


SHAPES = [(64, 1, [700, 130], None), (64, 2, [300, 200], [4, 3]), (96, 1, [200, 90], [8, 1]),
          (128, 1, [6000, 80], None), (256, 1, [300, 40], [2, 1]), (512, 1, [150], None)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("low,high", [(125, 125), (118, 125), (-100, -100), (-100, -90),
                                      (-30, 125)])
@pytest.mark.parametrize("dim,heads,lens,groups", SHAPES)
def test_values_at_the_ends_of_the_range(dtype, dim, heads, lens, groups, low, high):
    """Later scores pass the first ones' by up to 2^8 in weight before a reference moves."""
    gen = torch.Generator().manual_seed(dim + high)
    blocks = sum(-(-n // 16) for n in lens) + 2
    cache = cache_of(gen, blocks, heads, 16, dim, low, high)
    ids = torch.randperm(blocks, generator=gen).tolist()
    tables = [[ids.pop() for _ in range(-(-n // 16))] for n in lens]
    rows = [g for g, n in enumerate(groups or [1] * len(lens)) for _ in range(n)]
    for std in (0.5, 2.0):
        check(queries(gen, len(rows), heads, dim, dtype, std), cache, [lens[g] for g in rows],
              [tables[g] for g in rows], dim**-0.5, groups=groups)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("length", [70, 1000, 4000])
def test_equal_weights_of_the_largest_values(dtype, length):
    """A mean of the largest values the cache holds."""
    gen = torch.Generator().manual_seed(length)
    blocks = -(-length // 16)
    cache = cache_of(gen, blocks, 1, 16, 64, 125, 125)
    values = cache.view(blocks, -1)[:, 512:1024]
    values.fill_(0x77)  # 6
    query = torch.zeros(2, 1, 64, dtype=dtype, device=DEV)
    out = run_attention(query, cache, [length] * 2, [list(range(blocks))] * 2, 1.0)
    assert bool((out.double() == 6 * 2.0**125).all()), out
