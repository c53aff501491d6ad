"""The 4-bit cache on the GPU: what is appended and read back equals the definition bit for bit,
attention stays within derived bounds of it in 64 bits, and all hold in graphs, on other
streams and far into a large pool."""

import math

import pytest
import torch

from tests.cache_4bit_oracle import (append, attend, attend_tolerance, cross, cross_tolerance,
                                     quantised, same)

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DIMS = [32, 48, 64, 80, 96, 112, 128, 160, 192, 224, 256, 512]


def random_cache(gen, blocks, heads, bs, dim, low=-4, high=0):
    """A cache in use: any codes and scales of 2^low to 2^high."""
    from vflorence_amd import hip_attn

    cache = hip_attn.kv_cache_4bit(blocks, heads, bs, dim, "cpu")
    cache.copy_(torch.randint(0, 256, cache.shape, generator=gen))
    scales = cache.view(blocks, -1)[:, heads * bs * -(-dim // 32) * 32:]
    scales.copy_(torch.randint(127 + low, 128 + high, scales.shape, generator=gen))
    return cache.to(DEV)


def values_of(cache, dim):
    """Keys and values of a device cache, float64 on the host."""
    from vflorence_amd import hip_attn

    return [x.double() for x in hip_attn.kv_cache_4bit_values(cache.cpu(), dim)]


def tokens_of(gen, count, heads, dim, dtype, spread=2.0):
    """Keys and values as views of a fused projection, of mixed sizes."""
    qkv = torch.randn(count, 3, heads, dim, generator=gen)
    qkv *= torch.exp2(torch.randn(count, 1, heads, 1, generator=gen) * spread)
    qkv = qkv.to(dtype).to(DEV)
    return qkv[:, 1], qkv[:, 2]


def read(cache, slots, count, heads, dim, dtype):
    from vflorence_amd import hip_attn

    kv = torch.full((count, 2, heads, dim), 7.0, dtype=dtype, device=DEV)
    hip_attn.gather_cache_4bit(cache, slots, kv[:, 0], kv[:, 1])
    return kv[:, 0], kv[:, 1]


def check_append(cache, dim, key, value, slots):
    """Appends, and compares the whole cache and what is read back with the definition."""
    from vflorence_amd import hip_attn

    nb, heads, bs, _ = cache.shape
    want = values_of(cache, dim)
    hip_attn.reshape_and_cache_4bit(key, value, cache, slots.to(DEV))
    append(want, key, value, slots)
    got = values_of(cache, dim)
    assert same(got[0], want[0]) and same(got[1], want[1])
    back = read(cache, slots.to(DEV), len(slots), heads, dim, key.dtype)
    for x, held in zip(back, want):
        for t, s in enumerate(slots.tolist()):
            row = held[s // bs, :, s % bs] if 0 <= s < nb * bs else torch.zeros(heads, dim)
            assert same(x[t], row.to(key.dtype)), (t, s)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bs,dim", [(16, d) for d in DIMS] + [(32, d) for d in (48, 64, 128, 512)])
def test_append_to_blocks_in_use(dtype, bs, dim):
    gen = torch.Generator().manual_seed(bs + dim)
    heads, blocks = 3, 11
    cache = random_cache(gen, blocks, heads, bs, dim)
    # a lone token, a run, a block's first ones, skipped tokens, a whole block, any order
    slots = [5 * bs + 7, 2 * bs + 3, 2 * bs + 4, 2 * bs + 5, 7 * bs, 7 * bs + 1, -1, blocks * bs,
             4 * bs + bs - 1, *range(9 * bs, 10 * bs), 3 * bs, 2 * bs, -(1 << 40), 1 << 40]
    key, value = tokens_of(gen, len(slots), heads, dim, dtype)
    check_append(cache, dim, key, value, torch.tensor(slots))


@pytest.mark.parametrize("dtype,heads,bs,dim", [
    (torch.bfloat16, 2, 16, 64), (torch.float16, 3, 32, 48), (torch.float32, 1, 16, 32),
    (torch.bfloat16, 1, 16, 96), (torch.float32, 2, 32, 160), (torch.bfloat16, 1, 32, 512)])
def test_append_prompts(dtype, heads, bs, dim):
    """More tokens than a step has: packed prompts that begin anywhere in a block, whole parts
    at every place in a wave's window, runs with a token missing, skipped or out of order."""
    gen = torch.Generator().manual_seed(dim + bs)
    blocks = 80
    cache = random_cache(gen, blocks, heads, bs, dim)
    order = torch.randperm(blocks, generator=gen).tolist()
    slots = []
    for n, start in ((37, 0), (16, 0), (1, 5), (15, 1), (64, 0), (100, 9), (17, 15), (33, 0),
                     (130, 3), (48, 0), (90, 7)):
        ids = [order.pop() for _ in range((start + n - 1) // bs + 1)]
        slots += [ids[(start + i) // bs] * bs + (start + i) % bs for i in range(n)]
    whole = list(range(order[-1] * bs, order[-1] * bs + 16))
    order.pop()
    slots += whole[:7] + whole[8:]  # a part that lacks one
    slots += [-1] * 20
    whole = list(range(order[-1] * bs, order[-1] * bs + 16))
    order.pop()
    slots += whole[::-1]
    whole = list(range(order[-1] * bs, order[-1] * bs + 16))
    slots += whole[:8] + [-5] + whole[8:]
    slots += [blocks * bs] * 3
    assert len(slots) > 512
    key, value = tokens_of(gen, len(slots), heads, dim, dtype)
    check_append(cache, dim, key, value, torch.tensor(slots))


@pytest.mark.parametrize("count", [512, 513])
@pytest.mark.parametrize("dim", [64, 80])
def test_append_either_side_of_a_step(count, dim):
    gen = torch.Generator().manual_seed(count)
    cache = random_cache(gen, 70, 1, 16, dim)
    slots = torch.randperm(70 * 16, generator=gen)[:count]
    key, value = tokens_of(gen, count, 1, dim, torch.bfloat16)
    check_append(cache, dim, key, value, slots)
    cache = random_cache(gen, 70, 1, 16, dim)
    check_append(cache, dim, key, value, torch.arange(5, 5 + count))


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_special_values(dtype, many):
    """Zeros of both signs, every tie, the type's smallest and largest, infinities and NaN."""
    heads, dim, info = 2, 64, torch.finfo(dtype)
    count = 600 if many else 16
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(count, heads, dim, generator=gen)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.0, -0.0])
    x[0, 0, :32] = torch.cat([ties, -ties, ties, torch.ones(2)])
    x[1, 0] = 0.0
    x[2, 0, :32] = info.tiny
    x[3, 0, :32] = info.max
    x[4, 0, 3] = math.inf
    x[5, 0, 40] = -math.inf
    x[6, 1, 63] = math.nan
    x[7, 0, :32], x[7, 0, 5] = info.smallest_normal / 64, -info.tiny
    x[8, 1, :32], x[8, 1, 0] = 1e-6, info.max
    x[9, 0, :32], x[9, 0, 1] = 1.0, 6.0 + 0.0625  # just past 6
    key, value = x.to(dtype).to(DEV), (-x).roll(1, 0).to(dtype).to(DEV)
    cache = random_cache(gen, 64, heads, 16, dim)
    check_append(cache, dim, key, value, torch.arange(count) + 16)


def test_largest_values_stay_finite():
    """fp32 magnitudes that 6 * 2^125 does not reach are held as that; in fp16 what passes its
    range reads as an infinity."""
    from vflorence_amd import hip_attn

    cache = hip_attn.kv_cache_4bit(2, 1, 16, 32, DEV)
    x = torch.zeros(1, 1, 32, device=DEV)
    x[0, 0, :3] = torch.tensor([3.4e38, -3.4e38, 2.0**126])
    hip_attn.reshape_and_cache_4bit(x, x, cache, torch.tensor([3], device=DEV))
    key, value = read(cache, torch.tensor([3], device=DEV), 1, 1, 32, torch.float32)
    assert key[0, 0, :3].tolist() == value[0, 0, :3].tolist() == [6 * 2.0**125, -6 * 2.0**125,
                                                                 2.0**126]
    key, value = read(cache, torch.tensor([3], device=DEV), 1, 1, 32, torch.float16)
    assert key[0, 0, :4].tolist() == value[0, 0, :4].tolist() == [math.inf, -math.inf, math.inf,
                                                                 0.0]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,head_stride,token_stride", [(0, 64, 384), (1, 70, 211),
                                                             (8, 72, 144), (4, 64, 132)])
@pytest.mark.parametrize("count", [7, 600])
def test_strides(dtype, offset, head_stride, token_stride, count):
    """Rows of any strides and alignment, in and out."""
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(count)
    shape, strides = (count, 2, 64), (token_stride, head_stride, 1)
    base = torch.randn(count * token_stride + 512, generator=gen).to(dtype).to(DEV)
    key = base.as_strided(shape, strides, offset)
    value = base.as_strided(shape, strides, offset + 3)
    cache = random_cache(gen, 44, 2, 16, 64)
    slots = torch.arange(20, 20 + count)
    check_append(cache, 64, key, value, slots)
    plain = read(cache, slots.to(DEV), count, 2, 64, dtype)
    to = torch.full((2, count * token_stride + 512), 9.0, dtype=dtype, device=DEV)
    keys, values = (t.as_strided(shape, strides, t.storage_offset() + offset) for t in to)
    hip_attn.gather_cache_4bit(cache, slots.to(DEV), keys, values)
    assert same(keys, plain[0]) and same(values, plain[1])
    left = torch.ones_like(to[0], dtype=torch.bool)
    left.as_strided(shape, strides, offset).fill_(False)
    assert bool((to[:, left] == 9.0).all())


def test_gather_refuses_expanded_rows():
    from vflorence_amd import hip_attn

    cache = hip_attn.kv_cache_4bit(2, 2, 16, 64, DEV)
    out = torch.zeros(3, 2, 64, device=DEV)
    slots = torch.zeros(3, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="expanded"):
        hip_attn.gather_cache_4bit(cache, slots, out, out[:1].expand(3, 2, 64))


def test_gather_refuses_one_tensor_for_both():
    from vflorence_amd import hip_attn

    cache = hip_attn.kv_cache_4bit(2, 2, 16, 64, DEV)
    out = torch.zeros(3, 2, 64, device=DEV)
    slots = torch.zeros(3, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="memory of their own"):
        hip_attn.gather_cache_4bit(cache, slots, out, out)


def test_gather_any_slots():
    """Repeated, skipped and unordered slots; nothing at all; an empty pool."""
    gen = torch.Generator().manual_seed(8)
    cache = random_cache(gen, 40, 3, 16, 48)
    held = values_of(cache, 48)
    for count in (1, 90, 700):
        slots = torch.randint(-40, 40 * 16 + 40, (count,), generator=gen)
        slots[count // 2:] = slots[0].clamp(0, 600) // 16 * 16 + torch.arange(
            count - count // 2) % 32  # whole parts, again and again
        got = read(cache, slots.to(DEV), count, 3, 48, torch.float32)
        inside = (slots >= 0) & (slots < 640)
        for x, y in zip(got, held):
            rows = y.transpose(1, 2).reshape(640, 3, 48)[slots.clamp(0, 639)]
            assert same(x, rows.masked_fill(~inside[:, None, None], 0.0))
    none = read(cache, torch.zeros(0, dtype=torch.int64, device=DEV), 0, 3, 48, torch.float16)
    assert none[0].shape == (0, 3, 48)
    got = read(cache[:0], torch.zeros(5, dtype=torch.int64, device=DEV), 5, 3, 48, torch.float16)
    assert not got[0].any() and not got[1].any()


def test_copied_blocks():
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(4)
    cache = random_cache(gen, 6, 3, 16, 96)
    before = cache.clone()
    src, dst = torch.tensor([1, 4], device=DEV), torch.tensor([0, 3], device=DEV)
    hip_attn.copy_blocks([cache], src, dst)
    assert torch.equal(cache[[0, 3]], before[[1, 4]])
    assert torch.equal(cache[[1, 2, 4, 5]], before[[1, 2, 4, 5]])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def run_attention(query, cache, lens, tables, scale, groups=None, order=None, most=None, out=None,
                  bs=None):
    """The operator on host lists; ``groups``: rows of each group, sharing a table."""
    from vflorence_amd import hip_attn

    width = max(max(map(len, tables)), 1)
    table = torch.tensor([t + [10**6] * (width - len(t)) for t in tables], dtype=torch.int32,
                         device=DEV)
    meta = None
    if groups is not None:
        starts = torch.tensor([0] + groups).cumsum(0).int().to(DEV)
        if order is not None:
            order = torch.tensor(order, dtype=torch.int32, device=DEV)
        meta = hip_attn.get_scheduler_metadata(
            num_reqs=query.shape[0], num_heads=query.shape[1], num_kv_heads=query.shape[1],
            head_dim=query.shape[2], dtype=query.dtype, block_size=cache.shape[2],
            group_start=starts, group_order=order, max_group_size=most or max(groups))
    if out is None:
        out = torch.full(query.shape, 5.0, dtype=query.dtype, device=DEV)
    hip_attn.attention_with_kv_cache_4bit(
        query, cache, out, torch.tensor(lens, dtype=torch.int32, device=DEV), scale=scale,
        block_table=table, scheduler_metadata=meta)
    return out


def check_attention(query, cache, lens, tables, scale, **kw):
    out = run_attention(query, cache, lens, tables, scale, **kw)
    dim = query.shape[2]
    found = attend(query, values_of(cache, dim), lens, tables, scale)
    limit = attend_tolerance(query.dtype, dim, max(lens, default=0), *found)
    error = (out.double().cpu() - found[0]).abs()
    assert bool((error <= limit).all()), float((error / limit).max())
    return out


def queries(gen, rows, heads, dim, dtype, std=1.0):
    return (torch.randn(rows, heads, dim, generator=gen) * std).to(dtype).to(DEV)


LENS = [0, 1, 15, 16, 17, 63, 64, 65, 130, 300, 33]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bs,dim", [(16, d) for d in DIMS] + [(32, d) for d in (48, 64, 128, 512)])
def test_attention_rows(dtype, bs, dim):
    gen = torch.Generator().manual_seed(bs + dim)
    cache = random_cache(gen, 60, 2, bs, dim)
    tables = [torch.randperm(60, generator=gen)[: -(-n // bs)].tolist() for n in LENS]
    check_attention(queries(gen, len(LENS), 2, dim, dtype), cache, LENS, tables, dim**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bs,dim", [(16, 64), (32, 64), (16, 96), (16, 128), (32, 256), (16, 512)])
@pytest.mark.parametrize("most", [None, 8, 1])
def test_attention_groups(dtype, bs, dim, most):
    """Groups of one to eight rows, more than are taken together among them, in another order,
    one of them past the groups there are."""
    gen = torch.Generator().manual_seed(bs + dim)
    groups, lens = [4, 1, 8, 3, 5, 2, 4, 6], [70, 300, 64, 0, 129, 1, 17, 250]
    cache = random_cache(gen, 60, 3, bs, dim)
    tables = [torch.randperm(60, generator=gen)[: -(-n // bs)].tolist() for n in lens]
    rows = [g for g, n in enumerate(groups) for _ in range(n)]
    check_attention(queries(gen, len(rows), 3, dim, dtype), cache, [lens[g] for g in rows],
                    [tables[g] for g in rows], dim**-0.5, groups=groups,
                    order=[5, 2, 7, 0, 1, 6, 3, 4], most=most)


@pytest.mark.parametrize("dtype,bs,dim,heads,lens,groups", [
    (torch.bfloat16, 16, 64, 2, [9000, 1], None), (torch.float32, 32, 64, 1, [5003], None),
    (torch.float16, 32, 128, 2, [4097, 64], [3, 2]), (torch.bfloat16, 16, 256, 1, [3000], [8]),
    (torch.float32, 16, 512, 1, [2500], [4]), (torch.float16, 16, 32, 1, [0], None)])
def test_attention_long_contexts(dtype, bs, dim, heads, lens, groups):
    """Contexts that several workgroups split."""
    gen = torch.Generator().manual_seed(dim)
    blocks = 700
    cache = random_cache(gen, blocks, heads, bs, dim)
    tables = [torch.randint(0, blocks, (-(-max(n, 9000 // dim) // bs) or 1,),
                            generator=gen).tolist() for n in lens]
    rows = [g for g, n in enumerate(groups or [1] * len(lens)) for _ in range(n)]
    check_attention(queries(gen, len(rows), heads, dim, dtype), cache, [lens[g] for g in rows],
                    [tables[g] for g in rows], dim**-0.5, groups=groups)


@pytest.mark.parametrize("rows", [3000, 20000])
def test_attention_few_rows_among_many(rows):
    """A padded call: the context is split while its rows leave memory for four parts."""
    gen = torch.Generator().manual_seed(rows)
    cache = random_cache(gen, 200, 2, 16, 256)
    table = torch.randperm(200, generator=gen)[:188].tolist()
    query = queries(gen, rows, 2, 256, torch.bfloat16)
    out = run_attention(query, cache, [3000] * rows, [table] * rows, 0.07, groups=[3])
    found = attend(query[:3], values_of(cache, 256), [3000] * 3, [table] * 3, 0.07)
    limit = attend_tolerance(query.dtype, 256, 3000, *found)
    assert bool(((out[:3].double().cpu() - found[0]).abs() <= limit).all())
    assert bool((out[3:] == 5.0).all())


@pytest.mark.parametrize("bs", [16, 32])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_ignores_what_lies_behind(dtype, bs):
    """NaN scales behind the last token, ids outside the pool inside and behind the context."""
    gen = torch.Generator().manual_seed(bs)
    heads, dim, groups = 2, 96, 3
    cache = random_cache(gen, 40, heads, bs, dim)
    scales = cache.view(40, -1)[:, heads * bs * groups * 32:]
    scales = scales.view(40, heads, bs // 16, 4, 2, groups, 4)
    lens = [5, 16, 37, 70, 100]
    tables = []
    for i, n in enumerate(lens):
        pages = list(range(7 * i, 7 * i + -(-n // bs)))
        tables.append(pages)
        if n % bs:
            for t in range(n % bs, bs):
                scales[pages[-1], :, t // 16, t % 16 // 4, :, :, t % 4] = 255
    scales[39] = 255
    query = queries(gen, len(lens), heads, dim, dtype)
    check_attention(query, cache, lens, tables, dim**-0.5)
    for bad in (-1, 40, 2**31 - 1, -(2**31)):
        holes = [list(t) for t in tables]
        holes[3][1], holes[4][0], holes[2][-1] = bad, bad, bad
        check_attention(query, cache, lens, holes, dim**-0.5)
    alone = run_attention(query, cache, lens, [[-1] * len(t) for t in tables], dim**-0.5)
    assert not alone.any()


def test_attention_keeps_nan():
    """A NaN group of a token in the context: of K every output, of V its dims; a context longer
    than its table, a negative length."""
    gen = torch.Generator().manual_seed(2)
    for value in (0, 1):
        cache = random_cache(gen, 4, 1, 16, 64)
        scales = cache.view(4, -1)[:, 16 * 64:].view(4, 1, 1, 4, 2, 2, 4)
        scales[1, 0, 0, 2, value, 1, 3] = 255  # token 11 of block 1, dims 32 to 63
        out = run_attention(queries(gen, 2, 1, 64, torch.bfloat16), cache, [28, 27],
                            [[0, 1], [0, 1]], 0.125)
        if value:
            assert out[0, 0, 32:].isnan().all() and out[0, 0, :32].isfinite().all()
        else:
            assert out[0].isnan().all()
        assert out[1].isfinite().all()
    query = queries(gen, 3, 1, 64, torch.float32)
    cache = random_cache(gen, 4, 1, 16, 64)
    check_attention(query, cache, [1000, 33, 2**31 - 1], [[0], [1, 2], [3, 2]], 0.125)
    out = run_attention(query, cache, [-5, 0, -(2**31)], [[0], [1], [2]], 0.125)
    assert not out.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("std,scale,low,high", [(0.01, 1.0, -4, 0), (8.0, 0.25, -2, 2),
                                                (1.0, -0.125, -4, 0), (1.0, 0.0, 0, 3),
                                                (30.0, 20.0, 3, 6), (1.0, 1e-30, -2, 2)])
def test_attention_scores_of_any_size(dtype, std, scale, low, high):
    gen = torch.Generator().manual_seed(6)
    cache = random_cache(gen, 40, 2, 16, 64, low, high)
    lens = [200, 77, 310]
    tables = [torch.randperm(40, generator=gen)[: -(-n // 16)].tolist() for n in lens]
    check_attention(queries(gen, 3, 2, 64, dtype, std), cache, lens, tables, scale)


def test_attention_strides_in_place_and_tables():
    gen = torch.Generator().manual_seed(12)
    cache = random_cache(gen, 40, 2, 16, 48)
    lens, tables = [40, 90, 3], [[1, 2, 3], [4, 5, 6, 7, 8, 9], [10]]
    for dtype in DTYPES:
        fused = torch.randn(3, 500, generator=gen).to(dtype).to(DEV)
        query = fused.as_strided((3, 2, 48), (500, 51, 1), 5)
        a = check_attention(query, cache, lens, tables, 0.2)
        both = query.contiguous()
        assert torch.equal(run_attention(both, cache, lens, tables, 0.2, out=both), a)
        assert both.data_ptr() != query.data_ptr() and torch.equal(both, a)


def test_far_into_a_pool():
    """Blocks past 4 GiB: appended, read back and attended to."""
    from vflorence_amd import hip_attn

    heads, dim, bs = 16, 256, 32
    block_bytes = heads * bs * 34 * 8
    blocks = (5 << 30) // block_bytes
    cache = hip_attn.kv_cache_4bit(blocks, heads, bs, dim, DEV)
    gen = torch.Generator().manual_seed(1)
    ids = [blocks - 1, 3, blocks - 7]
    slots = torch.tensor([b * bs + t for b in ids for t in range(bs)])
    key, value = tokens_of(gen, len(slots), heads, dim, torch.bfloat16)
    hip_attn.reshape_and_cache_4bit(key, value, cache, slots.to(DEV))
    got = read(cache, slots.to(DEV), len(slots), heads, dim, torch.bfloat16)
    held = [quantised(x) for x in (key, value)]
    assert same(got[0], held[0]) and same(got[1], held[1])
    query = queries(gen, 1, heads, dim, torch.bfloat16)
    out = run_attention(query, cache, [90], [ids], dim**-0.5)
    pages = [x.view(3, bs, heads, dim).transpose(1, 2) for x in held]
    found = attend(query, pages, [90], [[0, 1, 2]], dim**-0.5)
    limit = attend_tolerance(torch.bfloat16, dim, 90, *found)
    assert bool(((out.double().cpu() - found[0]).abs() <= limit).all())
    # a prompt's path, past 512 tokens
    slots = torch.arange((blocks - 20) * bs, blocks * bs)
    key, value = tokens_of(gen, len(slots), heads, dim, torch.bfloat16)
    hip_attn.reshape_and_cache_4bit(key, value, cache, slots.to(DEV))
    got = read(cache, slots.to(DEV), len(slots), heads, dim, torch.bfloat16)
    assert same(got[0], quantised(key)) and same(got[1], quantised(value))


def test_over_nothing():
    from vflorence_amd import hip_attn

    cache = hip_attn.kv_cache_4bit(0, 2, 16, 64, DEV)
    query = torch.ones(2, 2, 64, device=DEV)
    out = run_attention(query, cache, [5, 0], [[0], [1]], 0.125)
    assert not out.any()
    full = hip_attn.kv_cache_4bit(3, 2, 16, 64, DEV)
    out = torch.ones_like(query)
    hip_attn.attention_with_kv_cache_4bit(
        query, full, out, torch.tensor([4, 4], dtype=torch.int32, device=DEV), scale=1.0,
        block_table=torch.zeros(2, 0, dtype=torch.int32, device=DEV))
    assert not out.any()
    hip_attn.attention_with_kv_cache_4bit(
        query[:0], full, out[:0], torch.zeros(0, dtype=torch.int32, device=DEV), scale=1.0,
        block_table=torch.zeros(0, 2, dtype=torch.int32, device=DEV))
    hip_attn.reshape_and_cache_4bit(query[:0], query[:0], full,
                                    torch.zeros(0, dtype=torch.int64, device=DEV))
    hip_attn.reshape_and_cache_4bit(query, query, cache,
                                    torch.zeros(2, dtype=torch.int64, device=DEV))
    assert not full.any()


@pytest.mark.parametrize("lens,groups", [([100, 37], [2, 1]), ([6000], None)])
def test_graph_of_a_step(lens, groups):
    """Append and attention captured together and replayed over new inputs, with eager work
    between the replays; two graphs at once have workspaces of their own."""
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(3)
    heads, dim, bs = 2, 64, 16
    rows = [g for g, n in enumerate(groups or [1] * len(lens)) for _ in range(n)]
    width = -(-max(lens) // bs)
    table = torch.stack([torch.randperm(width * 2, generator=gen)[:width] for _ in lens])
    tables = table[rows].int().to(DEV)
    lengths = torch.tensor([lens[g] for g in rows], dtype=torch.int32, device=DEV)
    meta = hip_attn.get_scheduler_metadata(
        num_reqs=len(rows), num_heads=heads, num_kv_heads=heads, head_dim=dim,
        dtype=torch.bfloat16, block_size=bs, max_group_size=max(groups or [1]),
        group_start=torch.tensor([0] + groups).cumsum(0).int().to(DEV) if groups else None)
    slots = torch.tensor([int(table[i, (n - 1) // bs]) * bs + (n - 1) % bs
                          for i, n in enumerate(lens)], device=DEV)

    def step(s):
        hip_attn.reshape_and_cache_4bit(s["key"], s["value"], s["cache"], slots)
        hip_attn.attention_with_kv_cache_4bit(s["query"], s["cache"], s["out"], lengths,
                                              scale=0.125, block_table=tables,
                                              scheduler_metadata=meta)

    states, graphs = [], []
    for _ in range(2):
        cache = random_cache(gen, width * 2, heads, bs, dim)
        key, value = (x.contiguous() for x in tokens_of(gen, len(lens), heads, dim,
                                                        torch.bfloat16))
        states.append(dict(cache=cache, key=key, value=value,
                           query=queries(gen, len(rows), heads, dim, torch.bfloat16),
                           out=torch.zeros(len(rows), heads, dim, dtype=torch.bfloat16,
                                           device=DEV)))
        step(states[-1])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(states[-1])
        graphs.append(graph)
    for turn in range(4):
        for s in states:
            s["query"].copy_(queries(gen, len(rows), heads, dim, torch.bfloat16))
            s["key"].copy_(tokens_of(gen, len(lens), heads, dim, torch.bfloat16)[0])
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s in states:
            got, held = s["out"].clone(), s["cache"].clone()
            step(s)
            assert torch.equal(s["out"], got) and torch.equal(s["cache"], held), turn


def test_other_stream_gradients_and_versions():
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(5)
    cache = random_cache(gen, 8, 2, 16, 64)
    key, value = tokens_of(gen, 20, 2, 64, torch.bfloat16)
    slots, query = torch.arange(20, device=DEV), queries(gen, 1, 2, 64, torch.bfloat16)
    want = cache.clone()
    hip_attn.reshape_and_cache_4bit(key, value, want, slots)
    out = run_attention(query, want, [20], [[0, 1]], 0.125)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        hip_attn.reshape_and_cache_4bit(key, value, cache, slots)
        again = run_attention(query, cache, [20], [[0, 1]], 0.125)
        back = read(cache, slots, 20, 2, 64, torch.bfloat16)
    stream.synchronize()
    assert torch.equal(cache, want) and torch.equal(out, again)
    assert same(back[0], quantised(key)) and same(back[1], quantised(value))

    leaf = key.float().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        hip_attn.reshape_and_cache_4bit(leaf, leaf, cache, slots)
    with pytest.raises(RuntimeError, match="no gradient"):
        hip_attn.gather_cache_4bit(cache, slots, leaf, leaf)
    asked = query.float().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        run_attention(asked, cache, [20], [[0, 1]], 0.125)
    with torch.no_grad():
        hip_attn.reshape_and_cache_4bit(leaf, leaf, cache, slots)
    for t, write in ((cache, lambda: hip_attn.reshape_and_cache_4bit(key, value, cache, slots)),
                     (out, lambda: run_attention(query, cache, [3], [[0]], 1.0, out=out))):
        version = t._version
        write()
        assert t._version > version


def test_serving_together():
    """As a server uses them: prompts' encoder states written in 4 bits, a decode step of beams
    over the pages, the pages read back for a given text of several tokens, whose attention
    over them equals that over the same values packed."""
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(21)
    heads, dim, bs, lens, beams, text = 4, 64, 16, [90, 17, 300, 128], 4, [5, 1, 40, 9]
    blocks = [-(-n // bs) for n in lens]
    ids = torch.randperm(sum(blocks) + 3, generator=gen).tolist()
    tables, at = [], 0
    for n in blocks:
        tables.append(ids[at: at + n])
        at += n
    slots = torch.tensor([t[i // bs] * bs + i % bs for t, n in zip(tables, lens)
                          for i in range(n)])
    cache = hip_attn.kv_cache_4bit(sum(blocks) + 3, heads, bs, dim, DEV)
    key, value = tokens_of(gen, len(slots), heads, dim, torch.bfloat16, spread=0.5)
    hip_attn.reshape_and_cache_4bit(key, value, cache, slots.to(DEV))
    held = quantised(key), quantised(value)
    # a step of beams
    rows = [g for g in range(len(lens)) for _ in range(beams)]
    query = queries(gen, len(rows), heads, dim, torch.bfloat16)
    check_attention(query, cache, [lens[g] for g in rows], [tables[g] for g in rows], dim**-0.5,
                    groups=[beams] * len(lens))
    # the states read back, in packed rows
    kv = torch.empty(len(slots), 2, heads, dim, dtype=torch.bfloat16, device=DEV)
    hip_attn.gather_cache_4bit(cache, slots.to(DEV), kv[:, 0], kv[:, 1])
    assert same(kv[:, 0], held[0]) and same(kv[:, 1], held[1])
    # given texts over them
    starts = [torch.tensor([0] + n).cumsum(0) for n in (text, lens)]
    query = queries(gen, sum(text), heads, dim, torch.bfloat16)
    out = torch.empty_like(query)
    hip_attn.packed_cross_attention(query, kv[:, 0], kv[:, 1], out,
                                    *(s.int().to(DEV) for s in starts), scale=dim**-0.5,
                                    max_query_len=max(text), max_key_len=max(lens))
    found = cross(query, *held, *(s.tolist() for s in starts), dim**-0.5)
    limit = cross_tolerance(torch.bfloat16, dim, max(lens), *found)
    assert bool(((out.double().cpu() - found[0]).abs() <= limit).all())
    # a text's first token, attended through the pages, is the same row within both bounds
    first = starts[0][:-1].tolist()
    step = run_attention(query[first].contiguous(), cache, lens, tables, dim**-0.5)
    both = limit[first] + attend_tolerance(torch.bfloat16, dim, max(lens),
                                           *(x[first] for x in found))
    assert bool(((step.double().cpu() - out[first].double().cpu()).abs() <= both).all())


def test_either_binding(monkeypatch):
    """Through ctypes the calls give what they give through the extension module."""
    from vflorence_amd import hip_attn
    from vflorence_amd._lib import lib

    gen = torch.Generator().manual_seed(31)
    key, value = tokens_of(gen, 40, 2, 64, torch.bfloat16)
    slots, query = torch.arange(40, device=DEV), queries(gen, 3, 2, 64, torch.bfloat16)

    def step():
        cache = hip_attn.kv_cache_4bit(3, 2, 16, 64, DEV)
        hip_attn.reshape_and_cache_4bit(key, value, cache, slots)
        out = run_attention(query, cache, [40] * 3, [[0, 1, 2]] * 3, 0.125)
        starts = [torch.tensor(s, dtype=torch.int32, device=DEV) for s in ([0, 3], [0, 40])]
        across = torch.empty_like(query)
        hip_attn.packed_cross_attention(query, key, value, across, *starts, scale=0.125,
                                        max_query_len=3, max_key_len=40)
        return cache, out, across, *read(cache, slots, 40, 2, 64, torch.bfloat16)

    want = step()
    monkeypatch.setattr(hip_attn, "calls", lib)
    assert all(torch.equal(a, b) for a, b in zip(step(), want))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,groups", [([70, 300], [4, 3]), ([300, 70], [8, 1]), ([6000], None)])
def test_attention_nan_query_stays_in_its_row(dtype, lens, groups):
    gen = torch.Generator().manual_seed(33)
    cache = random_cache(gen, 400, 2, 16, 64)
    tables = [torch.randperm(400, generator=gen)[: -(-n // 16)].tolist() for n in lens]
    rows = [g for g, n in enumerate(groups or [1] * len(lens)) for _ in range(n)]
    args = ([lens[g] for g in rows], [tables[g] for g in rows], 0.125)
    query = queries(gen, len(rows), 2, 64, dtype)
    want = run_attention(query, cache, *args, groups=groups)
    for bad in (math.nan, math.inf):
        query[0, 1, 5] = bad
        out = run_attention(query, cache, *args, groups=groups)
        assert out[0, 1].isnan().all()
        out[0, 1] = want[0, 1]
        assert torch.equal(out, want)


def test_values_of_a_device_cache():
    from vflorence_amd import hip_attn

    cache = random_cache(torch.Generator().manual_seed(34), 5, 3, 32, 96)
    for a, b in zip(hip_attn.kv_cache_4bit_values(cache, 96), values_of(cache, 96)):
        assert a.is_cuda and same(a, b)


def test_two_streams_at_once():
    """Calls that split their contexts, on two streams at once, have parts of their own."""
    gen = torch.Generator().manual_seed(35)
    cache = random_cache(gen, 400, 2, 16, 64)
    tables = [torch.randperm(400, generator=gen)[:375].tolist()]
    streams = [torch.cuda.Stream() for _ in range(2)]
    query = [queries(gen, 1, 2, 64, torch.bfloat16) for _ in streams]
    want = [run_attention(q, cache, [6000], tables, 0.125) for q in query]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for q, s in zip(query, streams):
            with torch.cuda.stream(s):
                got.append(run_attention(q, cache, [6000], tables, 0.125))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
