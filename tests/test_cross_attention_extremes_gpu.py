"""Packed cross-attention of operands at the ends of their types, against the definition in 64
bits."""

import math

import pytest
import torch

from tests.cache_4bit_oracle import cross, cross_tolerance, tolerance
from tests.test_cross_attention_gpu import DEV, inputs, run

pytestmark = pytest.mark.gpu

# heads of one to eight 32 dims, runs in one part and in several, in one key group and in more
SHAPES = [(32, 100), (48, 300), (64, 100), (64, 2500), (80, 2500), (96, 300), (128, 2500),
          (160, 70), (224, 100), (256, 100), (256, 1300)]


def as_defined(out, infinite, starts, keys, finite, finite_keys, scale=0.125):
    """``out`` against the definition: infinities and NaN where the ``infinite`` operands have
    them, the other elements within the bound of the ``finite`` ones."""
    want = cross(*infinite, starts, keys, scale)[0]
    found = cross(*finite, starts, finite_keys, scale)
    longest = max(b - a for a, b in zip(keys, keys[1:]))
    limit = cross_tolerance(out.dtype, out.shape[2], longest, *found)
    got = out.double().cpu()
    fine = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    error = (got - want).abs()[fine]
    assert bool((error <= limit[fine]).all()), float((error / limit[fine]).max())


@pytest.mark.parametrize("dim,keys", SHAPES)
def test_fp32_keys_of_score_minus_infinity(dim, keys):
    """They have no weight, wherever they stand: the whole first 32 keys, a lone one, the last."""
    gen = torch.Generator().manual_seed(dim + keys)
    q, k, v = inputs(gen, [40, 10], [keys, 30], 2, dim, torch.float32)
    q = q.abs() + 0.1
    starts, at = [0, 40, 50], [0, keys, keys + 30]
    for gone in (list(range(32)), [0], [keys - 1], [3, 33, 34, 69], [keys + 7]):
        k2 = k.clone()
        k2[gone] = 0.0
        k2[gone, :, dim - 2] = -math.inf
        keep = torch.ones(keys + 30, dtype=torch.bool)
        keep[gone] = False
        rest = int(keep[:keys].sum())
        out = run(q, k2, v, starts, at, 0.125)
        found = cross(q, k[keep.to(DEV)], v[keep.to(DEV)], starts, [0, rest, int(keep.sum())],
                      0.125)
        limit = cross_tolerance(torch.float32, dim, keys, *found)
        error = (out.double().cpu() - found[0]).abs()
        assert bool((error <= limit).all()), (gone, float((error / limit).max()))


@pytest.mark.parametrize("scale", [0.125, -0.125])
@pytest.mark.parametrize("dim,keys", SHAPES)
def test_fp32_infinite_keys_by_the_query(dim, keys, scale):
    """One key of both signs of score: no weight for a query of one sign, NaN for the other's."""
    gen = torch.Generator().manual_seed(dim + keys + 1)
    q, k, v = inputs(gen, [40, 10], [keys, 30], 2, dim, torch.float32)
    k2 = k.clone()
    k2[5, 1, 3] = math.inf
    starts, at = [0, 40, 50], [0, keys, keys + 30]
    out = run(q, k2, v, starts, at, scale)
    lost = (q[:40, 1, 3] * scale > 0).cpu()
    assert bool(lost.any()) and not bool(lost.all())
    assert out[:40, 1][lost].isnan().all()
    clean = run(q, k, v, starts, at, scale)
    assert torch.equal(out[:, 0], clean[:, 0]) and torch.equal(out[40:], clean[40:])
    keep = torch.arange(keys + 30) != 5
    found = cross(q, k[keep.to(DEV)], v[keep.to(DEV)], starts, [0, keys - 1, keys + 29], scale)
    limit = cross_tolerance(torch.float32, dim, keys, *found)
    error = (out.double().cpu() - found[0]).abs()[:40, 1][~lost]
    assert bool((error <= limit[:40, 1][~lost]).all())


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dim,keys", SHAPES)
def test_fp32_infinite_values(dim, keys, in_place):
    """An infinite value gives infinities of its sign, both signs or a key without weight NaN;
    no other dim, head or sequence changes by a bit."""
    gen = torch.Generator().manual_seed(dim + keys + 2)
    q, k, v = inputs(gen, [40, 33], [keys, 40], 2, dim, torch.float32, std=0.5)
    starts, at = [0, 40, 73], [0, keys, keys + 40]
    clean = run(q, k, v, starts, at, 0.125)
    v2 = v.clone()
    v2[5, 0, 9] = math.inf
    v2[6, 0, 8] = v2[keys - 1, 0, 8] = -math.inf
    v2[7, 0, dim - 1], v2[keys - 2, 0, dim - 1] = math.inf, -math.inf
    v2[8, 1, 17], v2[9, 1, 17] = math.nan, math.inf
    v2[keys + 39, 1, 0] = math.inf
    want = clean.clone()
    want[:40, 0, 9], want[:40, 0, 8] = math.inf, -math.inf
    want[:40, 0, dim - 1] = want[:40, 1, 17] = math.nan
    want[40:, 1, 0] = math.inf
    query = q.clone()
    out = run(query, k, v2, starts, at, 0.125, out=query if in_place else None)
    assert torch.equal(out.isnan(), want.isnan())
    assert torch.equal(out.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))


@pytest.mark.parametrize("dim,keys", [(64, 100), (128, 2500), (256, 100)])
def test_fp32_infinities_together(dim, keys):
    """Of a key of score -inf an infinite value is 0 * inf; infinite queries lose their own row;
    a value beside an infinite key keeps its weight."""
    gen = torch.Generator().manual_seed(dim + keys + 3)
    q, k, v = inputs(gen, [40, 10], [keys, 30], 2, dim, torch.float32)
    q = q.abs() + 0.1
    starts, at = [0, 40, 50], [0, keys, keys + 30]
    q2, k2, v2 = q.clone(), k.clone(), v.clone()
    k2[11] = 0.0
    k2[11, :, 1] = -math.inf
    v2[11, 0, 4] = math.inf  # weight 0
    v2[12, 0, 5] = math.inf
    q2[7, 1, 3] = math.inf
    q3, v3, keep = q2.clone(), v2.clone(), torch.arange(keys + 30, device=DEV) != 11
    q3[7, 1, 3] = v3[12, 0, 5] = 1.0
    as_defined(run(q2, k2, v2, starts, at, 0.125), (q2, k2, v2), starts, at,
               (q3, k[keep], v3[keep]), [0, keys - 1, keys + 29])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("scale", [0.125, 8.0])
@pytest.mark.parametrize("keys", [20, 100, 2500])
def test_rows_of_no_finite_score(dtype, scale, keys):
    """They are 0, beside rows that have one key of a finite score: that key's values.  Of them, in
    16 bits the product with the weight is exact, the reciprocal of the sum and the last product
    round by 2^-24 each and the result by eps / 2: less than eps in all.  In fp32 the product is a
    sum of six, rounded by 2^-24 each time, that leaves out 3 * 2^-26, of a weight kept to 2^-25:
    with the reciprocal and the last product 9.25 * 2^-24, less than 5 eps."""
    gen = torch.Generator().manual_seed(keys)
    q, k, v = inputs(gen, [40], [keys], 2, 64, dtype)
    q, k = q.abs() + 0.1, k.abs()
    k[:, :, 3] = -math.inf
    assert not run(q, k, v, [0, 40], [0, keys], scale).any()
    k[keys - 3, 1, 3] = 0.5
    out = run(q, k, v, [0, 40], [0, keys], scale)
    assert not out[:, 0].any()
    error = (out[:, 1].double() - v[keys - 3, 1].double()).abs()
    steps = 5 if dtype == torch.float32 else 1
    assert bool((error <= v[keys - 3, 1].double().abs() * steps * torch.finfo(dtype).eps).all())


@pytest.mark.parametrize("base", [3000.0, 30000.0, -40000.0, 45410.0, 60000.0])
@pytest.mark.parametrize("dim,queries,keys", [(64, 130, 700), (64, 9, 700), (64, 9, 6000),
                                              (128, 40, 2500), (256, 5, 900)])
def test_fp32_scores_far_from_zero(dim, queries, keys, base):
    """Scores that lie ``base`` from zero and rise by 6, so that references move, are apart in
    the key groups and in the parts: weights follow their differences (on either side of 2^16 in
    log2 units, from where a reference is no whole number, and across it).  Query and key have one
    dim that is not 0, of 22 bits: scores are exact.  A weight's exponent is rounded at 16 to 32
    in size, 2^-20, its exponential is good to 2^-22, a correction between two references adds
    three roundings below 2^-21 (of a difference of at most 9 in log2 units)."""
    gen = torch.Generator().manual_seed(dim + keys)
    q, k, v = inputs(gen, [queries], [keys], 1, dim, torch.float32)
    q.zero_()
    q[:, 0, 7] = 1.0
    steps = torch.randint(-64, 64, (keys,), generator=gen) + torch.linspace(0, 384, keys).long()
    k[:, 0, 7] = (base + steps / 64).to(DEV)
    out = run(q, k, v, [0, queries], [0, keys], 1.0)
    o, weight, size = cross(q, k, v, [0, queries], [0, keys], 1.0)
    limit = tolerance(torch.float32, 0, keys, 3 * 2.0**-26, o, weight, size * 0)
    limit += weight * 2 * (2.0**-20 + 3 * 2.0**-21)
    error = (out.double().cpu() - o).abs()
    assert bool((error <= limit).all()), float((error / limit).max())
