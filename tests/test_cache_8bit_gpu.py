"""The 8-bit cache on the GPU: appended caches equal the definition bit for bit, attention
stays within derived bounds of it in 64 bits, and both hold in graphs, on other streams and
far into a large pool."""

import pytest
import torch

from tests.cache_8bit_oracle import Cache, attend, attend_tolerance

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DIMS = [32, 48, 64, 80, 96, 112, 128, 160, 192, 224, 256, 512]


def random_cache(gen, blocks, heads, bs, dim, low=-9, high=-6):
    """A cache in use: e4m3 values and power-of-two scales."""
    k, v = ((torch.randn(blocks, heads, bs, dim, generator=gen) * 100).clamp(-448, 448).to(E4M3)
            for _ in range(2))
    e = torch.randint(low, high + 1, (blocks, heads, 2), generator=gen)
    return k.to(DEV), v.to(DEV), torch.exp2(e.double()).float().to(DEV)


def same_cache(cache, got):
    """The device cache holds the oracle's values (a NaN where it has one) and scales."""
    have = Cache.of(*got)
    for a, b in zip(have.q, cache.q):
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.nan_to_num(1e9), b.nan_to_num(1e9))
    assert torch.equal(have.scales, cache.scales)


def tokens_of(gen, count, heads, dim, dtype, spread=2.0):
    """Keys and values as views of a fused projection, of mixed sizes."""
    qkv = torch.randn(count, 3, heads, dim, generator=gen)
    qkv *= torch.exp2(torch.randn(count, 1, heads, 1, generator=gen) * spread)
    qkv = qkv.to(dtype).to(DEV)
    return qkv[:, 1], qkv[:, 2]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bs,dim", [(16, d) for d in DIMS] + [(32, d) for d in (48, 64, 128, 512)])
def test_append_to_blocks_in_use(dtype, bs, dim):
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(bs + dim)
    heads, blocks = 3, 11
    cache = random_cache(gen, blocks, heads, bs, dim)
    want = Cache.of(*cache)
    # a lone token, a run inside a block, one that starts its block over, skipped tokens,
    # a run over a block's end, a whole block
    slots = [5 * bs + 7, 2 * bs + 3, 2 * bs + 4, 2 * bs + 5, 7 * bs, 7 * bs + 1, -1, blocks * bs,
             4 * bs + bs - 1, *range(9 * bs, 10 * bs), 3 * bs]
    key, value = tokens_of(gen, len(slots), heads, dim, dtype)
    slots = torch.tensor(slots)
    hip_attn.reshape_and_cache_8bit(key, value, *cache, slots.to(DEV))
    want.append(key, value, slots)
    same_cache(want, cache)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_prompts_then_steps(dtype):
    """Packed prompts of odd lengths, then a decode step per token: every block grows in
    turn."""
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(3)
    heads, dim, bs, lens = 2, 64, 16, [1, 15, 16, 17, 40, 3]
    starts = [3 * i for i in range(len(lens))]  # three blocks a sequence, filled in order
    cache = random_cache(gen, 18, heads, bs, dim)
    want = Cache.of(*cache)
    slots = torch.tensor([starts[i] * bs + t for i, n in enumerate(lens) for t in range(n)])
    key, value = tokens_of(gen, len(slots), heads, dim, dtype)
    hip_attn.reshape_and_cache_8bit(key, value, *cache, slots.to(DEV))
    want.append(key, value, slots)
    same_cache(want, cache)
    for step in range(8):
        slots = torch.tensor([starts[i] * bs + n + step for i, n in enumerate(lens)])
        key, value = tokens_of(gen, len(slots), heads, dim, dtype, spread=3.0)
        hip_attn.reshape_and_cache_8bit(key, value, *cache, slots.to(DEV))
        want.append(key, value, slots)
        same_cache(want, cache)


@pytest.mark.parametrize("count,bs,dim", [(1, 16, 64), (511, 16, 64), (512, 16, 64), (513, 16, 64),
                                          (1100, 16, 192), (5000, 16, 64), (5000, 32, 64)])
def test_append_many_runs(count, bs, dim):
    """Calls from one token to many, runs at every place of the call, an odd head count."""
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(count)
    heads = 5
    slots, block = [], 0
    while len(slots) < count:
        n = int(torch.randint(1, 3 * bs, (1,), generator=gen))
        first = int(torch.randint(0, bs, (1,), generator=gen))
        slots += [block * bs + first + t for t in range(n)]
        block += (first + n + bs - 1) // bs
        if int(torch.randint(0, 4, (1,), generator=gen)) == 0:
            slots.append(-1)
    slots = torch.tensor(slots[:count])
    cache = random_cache(gen, block, heads, bs, dim)
    want = Cache.of(*cache)
    key, value = tokens_of(gen, count, heads, dim, torch.bfloat16)
    hip_attn.reshape_and_cache_8bit(key, value, *cache, slots.to(DEV))
    want.append(key, value, slots)
    same_cache(want, cache)


@pytest.mark.parametrize("dtype", DTYPES)
def test_append_special_values(dtype):
    """Zeros, infinities, NaN, the type's largest and smallest values, ties, a slot twice."""
    from vflorence_amd import hip_attn

    info = torch.finfo(dtype)
    gen = torch.Generator().manual_seed(1)
    cache = random_cache(gen, 8, 1, 16, 64)
    want = Cache.of(*cache)
    key = torch.randn(7, 1, 64, generator=gen)
    value = torch.randn(7, 1, 64, generator=gen)
    key[0], value[0] = 0.0, -0.0
    key[1, 0, 5], key[1, 0, 6], value[1, 0, 63] = float("inf"), float("-inf"), float("nan")
    key[2] = float("nan")
    key[3, 0, 0], value[3, 0, 0] = info.max / 4, info.tiny
    value[4] = info.tiny
    key[4] = torch.arange(64) * 0.0625 + 17.0  # ties of the two neighbours at 2^4
    key[4, 0, 63] = 448.0
    slots = torch.tensor([0, 16, 32, 48, 64, 83, 83])
    key, value = key.to(dtype).to(DEV), value.to(dtype).to(DEV)
    hip_attn.reshape_and_cache_8bit(key, value, *cache, slots.to(DEV))
    want.append(key, value, slots)
    same_cache(want, cache)


@pytest.mark.parametrize("dim,bs", [(64, 16), (128, 32), (48, 16)])
def test_append_out_of_order_and_repeated_slots(dim, bs):
    """A run in any order, longer than a wave, with slots that come again: the later token is
    taken, the earlier one does not count for the scale either."""
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(dim)
    cache = random_cache(gen, 5, 2, bs, dim)
    want = Cache.of(*cache)
    blocks = [(2, torch.randint(1, bs, (9,), generator=gen)),
              (0, torch.randint(0, bs, (150,), generator=gen)), (4, torch.arange(bs).flip(0)),
              (1, torch.tensor([3, 3, 5, 3]))]
    slots = torch.cat([b * bs + o for b, o in blocks])
    key, value = tokens_of(gen, len(slots), 2, dim, torch.bfloat16)
    key[-3] *= 64.0  # overwritten by the last token
    hip_attn.reshape_and_cache_8bit(key, value, *cache, slots.to(DEV))
    want.append(key, value, slots)
    same_cache(want, cache)


@pytest.mark.parametrize("bs,dim,dtype", [(16, 64, torch.bfloat16), (32, 64, torch.float16),
                                          (16, 192, torch.float32)])
@pytest.mark.parametrize("tail", [0, 600])
def test_append_skips_tokens_inside_runs(bs, dim, dtype, tail):
    """Skipped tokens are as if they were not in the call: inside a block's run, before its first
    and after its last token, more of them than a wave sees at once, and between tokens out of
    order.  (Were each side of a gap a run of its own, both would write the block's scale.)"""
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(bs + dim + tail)
    blocks, heads = 60, 3
    past = blocks * bs + 5
    slots = [-1, past, 0, 1, -1, 2, 5 * bs + 1, -1, past, 5 * bs + 2, -7, 3 * bs]
    for gap in (1, 14, 15, 16, 17, 62, 63, 64, 65, 127, 128, 200):
        block = 6 + len(slots) % 3 + 3 * (gap % 7)
        offsets = torch.randperm(bs, generator=gen)[:5].tolist()
        if gap % 2:
            offsets.sort()
        if any(s // bs == block for s in slots):
            block = next(b for b in range(30, blocks) if all(s // bs != b for s in slots))
        slots += [block * bs + offsets[0]] + [-1] * gap + [block * bs + o for o in offsets[1:3]]
        slots += [past] * (gap % 20) + [block * bs + o for o in offsets[3:]]
    slots += [-1] * 70
    if tail:
        slots = [-1] * tail + slots + [blocks * bs] * tail
    slots = torch.tensor(slots)
    cache = random_cache(gen, blocks, heads, bs, dim)
    want = Cache.of(*cache)
    key, value = tokens_of(gen, len(slots), heads, dim, dtype, spread=3.0)
    for t in range(4):  # whole calls of a few tokens, ends skipped or not
        part = slice(3 * t + tail, 3 * t + 3 + tail)
        few, mine = slots[part].clone(), [t.clone() for t in cache]
        hip_attn.reshape_and_cache_8bit(key[part], value[part], *mine, few.to(DEV))
        other = Cache.of(*cache)
        kept = (few >= 0) & (few < blocks * bs)
        other.append(key[part][kept.to(DEV)], value[part][kept.to(DEV)], few[kept])
        same_cache(other, mine)
    hip_attn.reshape_and_cache_8bit(key, value, *cache, slots.to(DEV))
    kept = (slots >= 0) & (slots < blocks * bs)
    want.append(key[kept.to(DEV)], value[kept.to(DEV)], slots[kept])
    same_cache(want, cache)


@pytest.mark.parametrize("bs", [16, 32])
@pytest.mark.parametrize("gap", [448, 479, 480, 481, 511, 512, 513, 543, 544, 1055, 1056, 5000])
def test_append_runs_over_long_gaps(bs, gap):
    """Runs and ends of runs on either side of more skipped tokens than one look ahead covers, and
    a call that ends with them."""
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(gap)
    slots = [-1] * gap + [2 * bs + 3] + [-1] * gap + [2 * bs + 9, 2 * bs + 1] + [-1] * gap
    slots += [5 * bs + 4, 7 * bs] + [-1] * gap + [7 * bs + 1, 3 * bs + 2] + [-1] * gap
    slots = torch.tensor(slots)
    cache = random_cache(gen, 9, 2, bs, 64)
    want = Cache.of(*cache)
    key, value = tokens_of(gen, len(slots), 2, 64, torch.bfloat16, spread=3.0)
    hip_attn.reshape_and_cache_8bit(key, value, *cache, slots.to(DEV))
    kept = slots >= 0
    want.append(key[kept.to(DEV)], value[kept.to(DEV)], slots[kept])
    same_cache(want, cache)


@pytest.mark.parametrize("count,bs", [(300, 16), (511, 16), (2000, 16), (2000, 32)])
def test_append_padded_prompts(count, bs):
    """A padded batch: every prompt's tokens followed by skipped ones, some inside it as well;
    the same cache as of the call without them, and on every run."""
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(count + bs)
    heads, dim, slots, block = 5, 64, [], 0
    while len(slots) < count:
        n, first, gap = (int(torch.randint(lo, hi, (1,), generator=gen))
                         for lo, hi in ((1, 5 * bs), (0, bs), (0, 150)))
        for t in range(n):
            slots += [-1] * int(torch.rand(1, generator=gen) < 0.2) + [block * bs + first + t]
        slots += [-1] * gap
        block += (first + n + bs - 1) // bs
    slots = torch.tensor(slots[:count])
    cache = random_cache(gen, block, heads, bs, dim)
    key, value = tokens_of(gen, count, heads, dim, torch.bfloat16, spread=3.0)
    kept = slots >= 0
    packed = [t.clone() for t in cache]
    hip_attn.reshape_and_cache_8bit(key[kept.to(DEV)], value[kept.to(DEV)], *packed,
                                    slots[kept].to(DEV))
    want = Cache.of(*cache)
    want.append(key[kept.to(DEV)], value[kept.to(DEV)], slots[kept])
    same_cache(want, packed)
    for _ in range(3):
        padded = [t.clone() for t in cache]
        hip_attn.reshape_and_cache_8bit(key, value, *padded, slots.to(DEV))
        for a, b in zip(padded, packed):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset,head_stride,token_stride", [(0, 96, 200), (1, 65, 131),
                                                             (3, 64, 129)])
def test_append_strides(dtype, offset, head_stride, token_stride):
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(9)
    cache = random_cache(gen, 6, 2, 16, 64)
    want = Cache.of(*cache)
    base = torch.randn(2, offset + 20 * token_stride + 200, generator=gen).to(dtype).to(DEV)
    key, value = (b.as_strided((20, 2, 64), (token_stride, head_stride, 1), offset) for b in base)
    slots = torch.arange(20) + 23
    hip_attn.reshape_and_cache_8bit(key, value, *cache, slots.to(DEV))
    want.append(key, value, slots)
    same_cache(want, cache)


def test_append_and_attend_far_into_a_pool():
    """Blocks whose bytes lie past 2^32 of a pool, and scales past 2^22 of theirs."""
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(2)
    heads, bs, dim, blocks = 16, 16, 64, (1 << 18) + 70  # 2^32 bytes and some a pool
    k, v, scales = hip_attn.kv_cache_8bit(blocks, heads, bs, dim, DEV)
    ids = [blocks - 1, 5, blocks - 2]
    key, value = tokens_of(gen, 40, heads, dim, torch.bfloat16, spread=0.5)
    slots = torch.tensor([ids[t // bs] * bs + t % bs for t in range(40)])
    hip_attn.reshape_and_cache_8bit(key, value, k, v, scales, slots.to(DEV))
    few = torch.tensor(sorted(ids))
    part = [t.view(torch.uint8)[few.to(DEV)].view(E4M3) for t in (k, v)]
    want = Cache(*(torch.zeros(3, heads, bs, dim, dtype=torch.float64) for _ in range(2)),
                 torch.zeros(3, heads, 2))
    place = {b: i for i, b in enumerate(sorted(ids))}
    near = torch.tensor([place[ids[t // bs]] * bs + t % bs for t in range(40)])
    want.append(key, value, near)
    same_cache(want, (*part, scales[few.to(DEV)]))
    query = tokens_of(gen, 1, heads, dim, torch.bfloat16, spread=0.0)[0].contiguous()
    out = torch.empty_like(query)
    hip_attn.attention_with_kv_cache_8bit(
        query, k, v, scales, out, torch.tensor([40], dtype=torch.int32, device=DEV), scale=0.125,
        block_table=torch.tensor([ids], dtype=torch.int32, device=DEV))
    close(query, out, want, [40], [[place[b] for b in ids]], 0.125)


def close(query, out, cache, lens, tables, scale):
    want, weight, size = attend(query, cache.values(), lens, tables, scale)
    tol = attend_tolerance(query.dtype, query.shape[2], max(max(lens), 1), want, weight, size)
    got = out.cpu().double()
    assert got.isfinite().all()
    worst = ((got - want).abs() / tol).max()
    print(f"error / bound {float(worst):.3f}", flush=True)
    assert worst <= 1, float(worst)


def paged_case(seed, dtype, dim, bs, lens, beams=1, heads=2, std=1.0):
    """A random cache and `lens` groups of `beams` rows over it: (query, cache, lens and tables
    of the rows, their device copies, group starts)."""
    gen = torch.Generator().manual_seed(seed)
    width = max(1, max(-(-n // bs) for n in lens))
    blocks = sum(-(-n // bs) for n in lens) + 3
    cache = random_cache(gen, blocks, heads, bs, dim)
    ids, tables, at = torch.randperm(blocks, generator=gen).tolist(), [], 0
    for n in lens:
        count = -(-n // bs)
        tables.append(ids[at: at + count] + [0] * (width - count))
        at += count
    rows = len(lens) * beams
    query = (torch.randn(rows, heads, dim, generator=gen) * std).to(dtype).to(DEV)
    row_lens = [n for n in lens for _ in range(beams)]
    row_tables = [t for t in tables for _ in range(beams)]
    device = (torch.tensor(row_lens, dtype=torch.int32, device=DEV),
              torch.tensor(row_tables, dtype=torch.int32, device=DEV))
    starts = torch.arange(0, rows + 1, beams, dtype=torch.int32, device=DEV)
    return query, cache, row_lens, row_tables, device, starts


def metadata(query, bs, beams=1, starts=None, order=None, **more):
    from vflorence_amd import hip_attn

    rows, heads, dim = query.shape
    return hip_attn.get_scheduler_metadata(
        num_reqs=rows, num_heads=heads, num_kv_heads=heads, head_dim=dim, dtype=query.dtype,
        block_size=bs, group_start=starts, group_order=order, max_group_size=beams, **more)


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 47, 100, 0, 255, 256, 257, 300]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bs,dim", [(16, d) for d in DIMS] + [(32, d) for d in DIMS])
def test_attention_rows(dtype, bs, dim):
    """Rows of their own, every length around the tiles' edges, empty ones among them."""
    from vflorence_amd import hip_attn

    query, cache, lens, tables, dev, _ = paged_case(dim + bs, dtype, dim, bs, LENS)
    out = torch.full_like(query, 7.0)
    hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=dim**-0.5,
                                          block_table=dev[1])
    close(query, out, Cache.of(*cache), lens, tables, dim**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("beams", [2, 3, 4, 5, 8])
@pytest.mark.parametrize("bs,dim", [(16, 64), (32, 128), (16, 80)])
def test_attention_groups(dtype, beams, bs, dim):
    """Groups that share a table, in a dispatch order of their own, and the same rows with
    tables of their own."""
    from vflorence_amd import hip_attn

    query, cache, lens, tables, dev, starts = paged_case(beams, dtype, dim, bs, LENS, beams)
    order = torch.arange(len(LENS) - 1, -1, -1, dtype=torch.int32, device=DEV)
    for meta in (metadata(query, bs, beams, starts, order),
                 metadata(query, bs, beams, starts, own_tables=True)):
        out = torch.full_like(query, 7.0)
        hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=dim**-0.5,
                                              block_table=dev[1], scheduler_metadata=meta)
        close(query, out, Cache.of(*cache), lens, tables, dim**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bs,dim,lens,beams", [
    (16, 64, [20011], 1), (16, 64, [5003, 9000, 1], 4), (32, 128, [12345, 40], 1),
    (16, 512, [3001], 2), (32, 48, [7777, 0], 3)])
def test_attention_long_contexts(dtype, bs, dim, lens, beams):
    """Few rows over long contexts: the work of a row is split."""
    from vflorence_amd import hip_attn

    query, cache, row_lens, tables, dev, starts = paged_case(len(lens), dtype, dim, bs, lens,
                                                             beams)
    out = torch.full_like(query, 7.0)
    hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=dim**-0.5,
                                          block_table=dev[1],
                                          scheduler_metadata=metadata(query, bs, beams, starts))
    close(query, out, Cache.of(*cache), row_lens, tables, dim**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bs,dim,heads,lens,beams", [
    (16, 64, 1, [2555], 1), (16, 64, 5, [20011], 1), (16, 48, 1, [7000, 33, 0], 1),
    (32, 80, 3, [9001], 3), (16, 128, 1, [5001], 5)])
def test_attention_odd_number_of_parts(dtype, bs, dim, heads, lens, beams):
    """Rows x heads x parts of a context odd: the workspace keeps its vectors aligned."""
    from vflorence_amd import hip_attn
    from vflorence_amd._lib import lib

    query, cache, row_lens, tables, dev, starts = paged_case(dim, dtype, dim, bs, lens, beams,
                                                             heads)
    need = lib.vfl_attention_8bit_workspace(len(row_lens), len(lens), heads, dim, bs,
                                            dev[1].shape[1])
    parts = need // (4 * dim + 8)
    assert parts % 2 and parts > len(row_lens) * heads
    out = torch.full_like(query, 7.0)
    hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=dim**-0.5,
                                          block_table=dev[1],
                                          scheduler_metadata=metadata(query, bs, beams, starts))
    close(query, out, Cache.of(*cache), row_lens, tables, dim**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bs", [16, 32])
def test_attention_ignores_what_lies_behind(dtype, bs):
    """NaN elements and NaN scales behind a row's last token, in its last block and in
    blocks that it lists past it, ids outside the pool, a table wider than any row."""
    from vflorence_amd import hip_attn

    lens = [1, 18, 33, 64, 70]
    query, cache, _, tables, dev, _ = paged_case(4, dtype, 64, bs, lens)
    clean = Cache.of(*cache)
    logical = hip_attn.v_cache_logical(cache[1].view(torch.uint8)).contiguous()
    keys = cache[0].view(torch.uint8)
    used = set()
    for n, table in zip(lens, tables):
        last = table[(n - 1) // bs]
        keys[last, :, (n - 1) % bs + 1:] = 0x7F
        logical[last, :, (n - 1) % bs + 1:] = 0xFF
        used |= set(table[: -(-n // bs)])
    for b in set(range(keys.shape[0])) - used:
        keys[b], logical[b], cache[2][b] = 0x7F, 0x7F, float("nan")
    values = hip_attn.v_cache_from_logical(logical.view(E4M3))
    bad = next(b for b in range(keys.shape[0]) if b not in used)
    wide = torch.full((len(lens), 9), bad, dtype=torch.int32, device=DEV)
    for r, n in enumerate(lens):
        count = -(-n // bs)
        wide[r, :count] = dev[1][r, :count]
    far = [list(t) for t in wide.tolist()]
    far[4][1] = 1 << 30  # contributes nothing
    far[2][0] = -5
    table = torch.tensor(far, dtype=torch.int32, device=DEV)
    out = torch.full_like(query, 7.0)
    hip_attn.attention_with_kv_cache_8bit(query, cache[0], values, cache[2], out, dev[0],
                                          scale=0.125, block_table=table[:, :7])
    close(query, out, clean, lens, far, 0.125)


def test_attention_keeps_nan_and_clamps():
    """A NaN among a row's own tokens reaches its output alone; a length past the table is
    the table's."""
    from vflorence_amd import hip_attn

    query, cache, lens, tables, dev, _ = paged_case(5, torch.bfloat16, 64, 16, [40, 40, 1000])
    table = dev[1].clone()[:, :4]
    cache[0].view(torch.uint8)[tables[0][1], 0, 3, 9] = 0x7F
    out = torch.zeros_like(query)
    hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=0.125,
                                          block_table=table)
    assert out[0, 0].isnan().all() and out[0, 1].isfinite().all() and out[1].isfinite().all()
    close(query[1:], out[1:], Cache.of(*cache), lens[1:], table[1:].tolist(), 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("std,low,high", [(30.0, -9, -6), (1e-3, -40, 30), (1.0, -100, -90)])
def test_attention_scales_and_peaks(dtype, std, low, high):
    """One-hot softmaxes and scales far apart from block to block."""
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(8)
    query, _, lens, tables, dev, _ = paged_case(6, dtype, 64, 16, [300, 64, 17], std=std)
    k, v, _ = random_cache(gen, 30, 2, 16, 64)
    scales = torch.exp2(torch.randint(low, high + 1, (30, 2, 2), generator=gen).double())
    scales[..., 0] = 2.0**-7 if std >= 1 else scales[..., 0].clamp(max=1.0)
    scales = scales.float().to(DEV)
    if dtype == torch.float16:
        scales[..., 1].clamp_(max=1.0)
    out = torch.empty_like(query)
    hip_attn.attention_with_kv_cache_8bit(query, k, v, scales, out, dev[0], scale=0.125,
                                          block_table=dev[1])
    cache = Cache.of(k, v, scales)
    want, weight, size = attend(query, cache.values(), lens, tables, 0.125)
    tol = attend_tolerance(dtype, 64, 300, want, weight, size)
    # below the type's smallest normal value a step no longer shrinks
    tol = tol + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    assert ((out.cpu().double() - want).abs() <= tol).all()


def test_attention_strided_query_and_rows_left_alone():
    """A query that is a view of a fused projection, metadata that covers part of the rows."""
    from vflorence_amd import hip_attn

    query, cache, lens, tables, dev, _ = paged_case(7, torch.bfloat16, 64, 16, [50, 60, 70, 80])
    wide = torch.randn(4, 200, device=DEV, dtype=torch.bfloat16)
    view = wide.as_strided((4, 2, 64), (200, 71, 1), 3)
    view.copy_(query)
    starts = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=DEV)
    out = torch.full_like(query, 7.0)
    hip_attn.attention_with_kv_cache_8bit(view, *cache, out, dev[0], scale=0.125,
                                          block_table=dev[1],
                                          scheduler_metadata=metadata(query, 16, 1, starts))
    assert (out[3] == 7.0).all()  # no group names it
    close(query[:3], out[:3], Cache.of(*cache), lens[:3], tables[:3], 0.125)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.125, 1e-6])
def test_attention_any_finite_scale(dtype, scale):
    from vflorence_amd import hip_attn

    query, cache, lens, tables, dev, _ = paged_case(13, dtype, 80, 16, [0, 1, 37, 260])
    out = torch.empty_like(query)
    hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=scale,
                                          block_table=dev[1])
    close(query, out, Cache.of(*cache), lens, tables, scale)
    for bad in (float("nan"), float("inf")):
        with pytest.raises(RuntimeError, match="scale"):
            hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=bad,
                                                  block_table=dev[1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_largest_queries(dtype):
    """One dim of a query at its type's largest value, of either sign, over small keys: the weight
    lies on the tokens whose key has the largest product with it, which share it."""
    from vflorence_amd import hip_attn

    query, cache, lens, tables, dev, _ = paged_case(17, dtype, 64, 16, [300, 64, 17, 1])
    gen = torch.Generator().manual_seed(17)
    query.zero_()
    query[:, :, 5] = torch.finfo(dtype).max
    query[1, :, 5] *= -1
    cache[0].copy_(torch.randint(-4, 5, cache[0].shape, generator=gen).float().to(E4M3))
    cache[2][..., 0] = 2.0**-8  # (fp16: products a hundred apart and more)
    out = torch.empty_like(query)
    hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=1.0,
                                          block_table=dev[1])
    want, weight, size = attend(query, Cache.of(*cache).values(), lens, tables, 1.0)
    tol = attend_tolerance(dtype, 64, 300, want, weight, torch.zeros_like(size))
    assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("length", [45, 6000])
def test_attention_in_place_and_broadcast_tables(length):
    """The output written over the query; rows that share one expanded table and length; a
    single row whose strides say nothing."""
    from vflorence_amd import hip_attn

    query, cache, lens, tables, dev, _ = paged_case(14, torch.bfloat16, 64, 16, [length], 3)
    want = Cache.of(*cache)
    table = dev[1][:1].expand(3, -1)
    out = query.clone()
    hip_attn.attention_with_kv_cache_8bit(out, *cache, out, dev[0][:1].expand(3), scale=0.125,
                                          block_table=table)
    close(query, out, want, lens, tables, 0.125)
    one = query[:1].as_strided((1, 2, 64), (7, 64, 1))
    out = torch.empty_like(query[:1])
    hip_attn.attention_with_kv_cache_8bit(
        one, *cache, out, dev[0][:1], scale=0.125,
        block_table=dev[1][:1].as_strided((1, dev[1].shape[1]), (0, 1)))
    close(query[:1], out, want, lens[:1], tables[:1], 0.125)


def test_attention_over_nothing():
    """A table without columns, a pool without blocks: rows of zeros."""
    from vflorence_amd import hip_attn

    query, cache, lens, _, dev, _ = paged_case(15, torch.bfloat16, 64, 16, [20, 3])
    out = torch.full_like(query, 7.0)
    hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=0.125,
                                          block_table=dev[1][:, :0])
    assert (out == 0).all()
    empty = hip_attn.kv_cache_8bit(0, 2, 16, 64, DEV)
    out = torch.full_like(query, 7.0)
    hip_attn.attention_with_kv_cache_8bit(query, *empty, out, dev[0], scale=0.125,
                                          block_table=dev[1])
    assert (out == 0).all()
    key = torch.ones(2, 2, 64, device=DEV)
    hip_attn.reshape_and_cache_8bit(key, key, *empty, torch.tensor([0, 5], device=DEV))


@pytest.mark.parametrize("lens,beams", [([700, 20, 333], 4), ([9001], 2)])
def test_graph_of_append_and_attention(lens, beams):
    """Captured once, replayed over new tokens with eager work of the same kind between:
    every replay equals the eager calls; two graphs keep apart."""
    from vflorence_amd import hip_attn

    dtype, bs = torch.bfloat16, 16
    query, cache, row_lens, tables, dev, starts = paged_case(9, dtype, 64, bs, lens, beams)
    meta = metadata(query, bs, beams, starts)
    gen = torch.Generator().manual_seed(10)
    key, value = (t.contiguous() for t in tokens_of(gen, len(lens), 2, 64, dtype))
    slots = torch.tensor([tables[i * beams][(n - 1) // bs] * bs + (n - 1) % bs
                          for i, n in enumerate(lens)], device=DEV)
    outs = [torch.empty_like(query) for _ in range(3)]
    queries = [query, (query * 0.5).contiguous()]

    def step(q, out):
        hip_attn.reshape_and_cache_8bit(key, value, *cache, slots)
        hip_attn.attention_with_kv_cache_8bit(q, *cache, out, dev[0], scale=0.125,
                                              block_table=dev[1], scheduler_metadata=meta)

    before = [t.clone() for t in cache]
    step(query, outs[2])  # initialises what a first call does
    graphs = []
    for q, out in zip(queries, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(q, out)
        graphs.append(graph)
    for old, now in zip(before, cache):
        now.view(torch.uint8).copy_(old.view(torch.uint8))
    want = Cache.of(*cache)
    for turn in range(4):
        new = tokens_of(gen, len(lens), 2, 64, dtype)
        key.copy_(new[0])
        value.copy_(new[1])
        want.append(key, value, slots.cpu())
        graphs[turn % 2].replay()
        torch.cuda.synchronize()
        same_cache(want, cache)
        step(queries[turn % 2], outs[2])  # the slots' tokens once more: the same cache
        torch.cuda.synchronize()
        same_cache(want, cache)
        assert torch.equal(outs[turn % 2], outs[2])
        close(queries[turn % 2], outs[2], want, row_lens, tables, 0.125)
    graphs[0].replay()
    graphs[1].replay()
    first = outs[0].clone(), outs[1].clone()
    graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(first[0], outs[0]) and torch.equal(first[1], outs[1])


def test_other_stream_and_gradients():
    from vflorence_amd import hip_attn

    query, cache, lens, tables, dev, _ = paged_case(11, torch.float16, 64, 16, [90, 5000])
    out = torch.empty_like(query)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=0.125,
                                              block_table=dev[1])
    side.synchronize()
    close(query, out, Cache.of(*cache), lens, tables, 0.125)
    query.requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=0.125,
                                              block_table=dev[1])
    with torch.no_grad():
        hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=0.125,
                                              block_table=dev[1])
    empty = torch.empty(0, 2, 64, dtype=torch.float16, device=DEV)
    hip_attn.attention_with_kv_cache_8bit(
        empty, *cache, empty.clone(), torch.empty(0, dtype=torch.int32, device=DEV), scale=1.0,
        block_table=torch.empty(0, 3, dtype=torch.int32, device=DEV))
    hip_attn.reshape_and_cache_8bit(empty, empty, *cache,
                                    torch.empty(0, dtype=torch.int64, device=DEV))


def test_decode_together():
    """As a decoder uses them: prompts paged in 8 bits, then steps in which two requests of
    three beams append, fork with copied blocks and scales, attend to themselves and to their
    prompt, and have their tokens scored."""
    from vflorence_amd import decoder_ops, hip_attn

    gen = torch.Generator().manual_seed(12)
    heads, dim, bs, beams, dtype, vocab = 4, 64, 16, 3, torch.bfloat16, 1003
    prompts = [37, 50]
    cross = hip_attn.kv_cache_8bit(8, heads, bs, dim, DEV)
    want_cross = Cache.of(*cross)
    pages = [[6, 1, 3], [0, 7, 2, 5]]
    slots = torch.tensor([pages[i][t // bs] * bs + t % bs
                          for i, n in enumerate(prompts) for t in range(n)])
    key, value = tokens_of(gen, len(slots), heads, dim, dtype, 0.5)
    hip_attn.reshape_and_cache_8bit(key, value, *cross, slots.to(DEV))
    want_cross.append(key, value, slots)
    rows = 2 * beams
    row_lens = [n for n in prompts for _ in range(beams)]
    row_pages = [p + [0] * (4 - len(p)) for p in pages for _ in range(beams)]
    starts = torch.tensor([0, 3, 6], dtype=torch.int32, device=DEV)
    own = hip_attn.kv_cache_8bit(24, heads, bs, dim, DEV)
    want_own = Cache.of(*own)
    head = torch.randn(heads * dim, vocab, generator=gen).to(dtype).to(DEV) / 8
    tables = [[4 * r] for r in range(rows)]
    for step in range(36):
        if step % bs == 0 and step:
            for r in range(rows):
                tables[r] = tables[r] + [4 * r + step // bs]
        if step in (5, 20):  # the second row of each request goes on from the first
            src = [tables[r][-1] for r in (0, 3)]
            dst = [tables[r][-1] for r in (1, 4)]
            for r in (0, 3):
                tables[r + 1] = tables[r][:-1] + tables[r + 1][-1:]
            args = [torch.tensor(t, device=DEV) for t in (src, dst)]
            hip_attn.copy_blocks([own[0], own[1]], *args)
            hip_attn.copy_blocks([own[2]], *args)
            for q in (*want_own.q, want_own.scales):
                q[dst] = q[src]
        qkv = torch.randn(rows, 3, heads, dim, generator=gen).to(dtype).to(DEV)
        slots = torch.tensor([tables[r][step // bs] * bs + step % bs for r in range(rows)])
        hip_attn.reshape_and_cache_8bit(qkv[:, 1], qkv[:, 2], *own, slots.to(DEV))
        want_own.append(qkv[:, 1], qkv[:, 2], slots)
        lens = torch.full((rows,), step + 1, dtype=torch.int32, device=DEV)
        mid = torch.empty(rows, heads, dim, dtype=dtype, device=DEV)
        hip_attn.attention_with_kv_cache_8bit(
            qkv[:, 0], *own, mid, lens, scale=0.125,
            block_table=torch.tensor(tables, dtype=torch.int32, device=DEV))
        out = torch.empty_like(mid)
        hip_attn.attention_with_kv_cache_8bit(
            mid, *cross, out, torch.tensor(row_lens, dtype=torch.int32, device=DEV), scale=0.125,
            block_table=torch.tensor(row_pages, dtype=torch.int32, device=DEV),
            scheduler_metadata=metadata(mid, bs, beams, starts))
        logits = out.flatten(1) @ head
        tokens = torch.randint(0, vocab, (rows,), generator=gen).to(DEV)
        logprobs, entropy, top, ids = decoder_ops.token_logprobs(logits, tokens, 3)
        same_cache(want_own, own)
        close(qkv[:, 0], mid, want_own, [step + 1] * rows, tables, 0.125)
        close(mid, out, want_cross, row_lens, row_pages, 0.125)
        logp = torch.log_softmax(logits.double(), dim=1)
        # a sum of 1003 exponentials in fp32, each good to 2^-21, over chains of four or so
        assert (logprobs.double() - logp.gather(1, tokens[:, None])[:, 0]).abs().max() < 4e-6
        assert (entropy.double() + (logp.exp() * logp).sum(1)).abs().max() < 2e-5
        order = torch.sort(logits, dim=1, descending=True, stable=True).indices
        assert torch.equal(ids, order[:, :3])
        assert (top.double() - logp.gather(1, ids)).abs().max() < 4e-6
    same_cache(want_cross, cross)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,beams,dim", [([300, 64, 17, 1, 0], 1, 64), ([5003], 3, 64),
                                            ([90, 33], 4, 128)])
@pytest.mark.parametrize("power,scale", [(10, 0.125), (26, 0.125), (34, -0.3), (60, 0.125),
                                         (100, -0.3), (0, 1e30), (0, -3e38), (100, 1e-35),
                                         (110, 0.0), (118, 1e-42)])
def test_attention_scores_of_any_size(dtype, lens, beams, dim, power, scale):
    """Scores so large that their product with log2 e holds no units, whole and split: whole
    numbers times 2^power, which fp32 sums hold exactly (below 2^24 and 2^128), so that equal
    ones share the weight and a score's own error (the bound's `size`) is 0.  A difference times
    the scale is rounded twice, 2^-23 of an exponent that adds weight only below 32."""
    from vflorence_amd import hip_attn

    query, cache, row_lens, tables, dev, starts = paged_case(power, dtype, dim, 16, lens, beams)
    gen = torch.Generator().manual_seed(power)
    query.copy_(torch.randint(-2, 3, query.shape, generator=gen))
    cache[0].copy_(torch.randint(-4, 5, cache[0].shape, generator=gen).float().to(E4M3))
    cache[2][..., 0] = 2.0**power
    cache[2][::3, :, 0] = 2.0**(power - 1)
    out = torch.full_like(query, 7.0)
    hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=scale,
                                          block_table=dev[1],
                                          scheduler_metadata=metadata(query, 16, beams, starts))
    want, weight, size = attend(query, Cache.of(*cache).values(), row_lens, tables, scale)
    tol = attend_tolerance(dtype, dim, max(lens), want, weight, torch.zeros_like(size))
    tol = tol + 32 * 2.0**-22 * weight
    worst = ((out.cpu().double() - want).abs() / tol).max()
    print(f"error / bound {float(worst):.3f}", flush=True)
    assert worst <= 1, float(worst)


def test_refuses_gradients_of_the_cache_and_counts_writes():
    """Pools and scales that require gradients are refused as queries, keys and values are; what
    a call writes counts as written, so that autograd sees a saved tensor change."""
    from vflorence_amd import hip_attn

    query, cache, _, _, dev, _ = paged_case(16, torch.bfloat16, 64, 16, [20, 40])
    key = torch.ones(2, 2, 64, device=DEV)
    slots = torch.tensor([3, 20], device=DEV)

    def attend_into(out):
        hip_attn.attention_with_kv_cache_8bit(query, *cache, out, dev[0], scale=0.125,
                                              block_table=dev[1])

    def append():
        hip_attn.reshape_and_cache_8bit(key, key, *cache, slots)

    out = torch.empty_like(query)
    for call, written in ((append, cache), (lambda: attend_into(out), (out,))):
        before = [t._version for t in written]
        call()
        assert all(t._version > v for t, v in zip(written, before))
    for t in cache:
        t.requires_grad_(True)
        for call in (append, lambda: attend_into(out)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
            with torch.no_grad():
                call()
        t.requires_grad_(False)
    x = torch.ones(query.shape, device=DEV, requires_grad=True)
    saved = torch.empty(query.shape, device=DEV)
    loss = (x * saved).sum()  # saves `saved`
    hip_attn.attention_with_kv_cache_8bit(query.float(), *cache, saved, dev[0], scale=0.125,
                                          block_table=dev[1])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():  # (whose own tensors count no versions)
        held = hip_attn.kv_cache_8bit(4, 2, 16, 64, DEV)
        hip_attn.reshape_and_cache_8bit(key, key, *held, slots)
        other = torch.empty_like(query)
        attend_into(other)


@pytest.mark.parametrize("rows", [3000, 20000])
def test_attention_few_rows_among_many(rows):
    """A padded call: the context is split while its rows leave memory for four parts."""
    from vflorence_amd import hip_attn

    query, cache, lens, tables, _, starts = paged_case(17, torch.bfloat16, 256, 16, [3000], 3)
    many = torch.randn(rows, 2, 256, generator=torch.Generator().manual_seed(rows))
    many = many.to(torch.bfloat16).to(DEV)
    many[:3] = query
    out = torch.full_like(many, 7.0)
    hip_attn.attention_with_kv_cache_8bit(
        many, *cache, out, torch.tensor(lens[:1], dtype=torch.int32, device=DEV).expand(rows),
        scale=256**-0.5,
        block_table=torch.tensor(tables[:1], dtype=torch.int32, device=DEV).expand(rows, -1),
        scheduler_metadata=metadata(many, 16, 3, starts))
    close(query, out[:3], Cache.of(*cache), lens, tables, 256**-0.5)
    assert bool((out[3:] == 7.0).all())
