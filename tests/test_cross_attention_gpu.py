"""Packed cross-attention on the GPU against its definition in 64 bits, within derived bounds."""

import math

import pytest
import torch

from tests.cache_4bit_oracle import cross, cross_tolerance

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
DIMS = [32, 48, 64, 80, 96, 112, 128, 160, 192, 224, 256]


def starts_of(lens):
    return [0] + torch.tensor(lens).cumsum(0).tolist()


def inputs(gen, queries, keys, heads, dim, dtype, std=1.0):
    q = (torch.randn(sum(queries), heads, dim, generator=gen) * std).to(dtype).to(DEV)
    kv = torch.randn(sum(keys), 2, heads, dim, generator=gen).to(dtype).to(DEV)
    return q, kv[:, 0], kv[:, 1]


def run(q, k, v, query_starts, key_starts, scale, longest=None, out=None):
    from vflorence_amd import hip_attn

    if longest is None:
        longest = [max((b - a for a, b in zip(s, s[1:])), default=0)
                   for s in (query_starts, key_starts)]
    if out is None:
        out = torch.full(q.shape, 5.0, dtype=q.dtype, device=DEV)
    at = [torch.tensor(s, dtype=torch.int32, device=DEV) for s in (query_starts, key_starts)]
    hip_attn.packed_cross_attention(q, k, v, out, *at, scale=scale, max_query_len=longest[0],
                                    max_key_len=longest[1])
    return out


def check(q, k, v, query_starts, key_starts, scale, **kw):
    out = run(q, k, v, query_starts, key_starts, scale, **kw)
    found = cross(q, k, v, query_starts, key_starts, scale)
    most = max((b - a for a, b in zip(key_starts, key_starts[1:])), default=0)
    limit = cross_tolerance(q.dtype, q.shape[2], most, *found)
    a, b = query_starts[0], query_starts[-1]
    error = (out.double().cpu() - found[0]).abs()[a:b]
    assert bool((error <= limit[a:b]).all()), float((error / limit[a:b]).max())
    return out


QUERIES = [1, 33, 0, 128, 5, 31, 70, 2]
KEYS = [64, 1, 40, 65, 0, 200, 31, 129]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", DIMS)
def test_ragged_runs(dtype, dim):
    gen = torch.Generator().manual_seed(dim)
    q, k, v = inputs(gen, QUERIES, KEYS, 2, dim, dtype)
    check(q, k, v, starts_of(QUERIES), starts_of(KEYS), dim**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("queries,keys", [
    ([1] * 9, [1, 63, 64, 65, 128, 129, 256, 300, 0]),  # single tokens
    ([20] * 40, [90] * 40),  # runs of one tile, many of them
    ([50, 64, 33] * 8, [300, 17, 128] * 8),  # two tiles of 32
    ([200, 129] * 20, [140, 77] * 20),  # tiles of 128, and a ragged one
])
def test_launch_shapes(dtype, dim, queries, keys):
    gen = torch.Generator().manual_seed(dim + len(queries))
    q, k, v = inputs(gen, queries, keys, 3, dim, dtype, std=2.0)
    check(q, k, v, starts_of(queries), starts_of(keys), dim**-0.5)


@pytest.mark.parametrize("dtype,dim,heads,queries,keys", [
    (torch.bfloat16, 64, 2, [9], [5000]), (torch.float16, 128, 1, [17, 33], [4097, 2600]),
    (torch.float32, 64, 1, [3, 40, 1], [2500, 100, 0]), (torch.float32, 256, 1, [1], [3001]),
    (torch.bfloat16, 256, 2, [130], [2100]), (torch.float32, 96, 2, [70, 2], [2400, 2100])])
def test_long_keys(dtype, dim, heads, queries, keys):
    """Runs of keys that several workgroups split."""
    gen = torch.Generator().manual_seed(dim)
    q, k, v = inputs(gen, queries, keys, heads, dim, dtype)
    check(q, k, v, starts_of(queries), starts_of(keys), dim**-0.5)


@pytest.mark.parametrize("longest", [(0, 0), (1, 1), (1, 100000), (40, 64), (100000, 100000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_stated_lengths_change_no_result(dtype, longest):
    gen = torch.Generator().manual_seed(7)
    queries, keys = [300, 3, 70], [90, 2600, 300]
    q, k, v = inputs(gen, queries, keys, 1, 64, dtype)
    check(q, k, v, starts_of(queries), starts_of(keys), 0.125, longest=longest)


def test_rows_of_no_sequence_are_left_alone():
    gen = torch.Generator().manual_seed(9)
    for dtype in DTYPES:
        for keys in ([3, 60, 2300], [3, 60, 100]):
            q, k, v = inputs(gen, [80], [sum(keys) + 9], 2, 64, dtype)
            qs, ks = [4, 9, 50, 77], [5, 5 + keys[0], 5 + keys[0] + keys[1], sum(keys) + 5]
            k[:5] = v[:5] = k[sum(keys) + 5:] = v[sum(keys) + 5:] = math.nan
            out = check(q, k, v, qs, ks, 0.125)
            assert bool((out[:4] == 5).all()) and bool((out[77:] == 5).all())


@pytest.mark.parametrize("rows", [40000, 300000, 700000])
def test_few_queries_among_many_rows(rows):
    """A padded call: the keys are split over as many parts as its rows leave memory for."""
    gen = torch.Generator().manual_seed(rows)
    q, k, v = inputs(gen, [rows], [5000, 1200], 1, 32, torch.bfloat16)
    first = rows - 40
    out = run(q, k, v, [first, first + 9, first + 30], [0, 5000, 6200], 0.2)
    found = cross(q[first:], k, v, [0, 9, 30], [0, 5000, 6200], 0.2)
    limit = cross_tolerance(q.dtype, 32, 5000, *found)
    error = (out[first:].double().cpu() - found[0]).abs()[:30]
    assert bool((error <= limit[:30]).all())
    assert bool((out[:first] == 5.0).all()) and bool((out[first + 30:] == 5.0).all())


def test_offsets_past_the_rows_are_limited():
    """Starts outside the tensors, falling ones, no sequences, no rows, no keys at all."""
    gen = torch.Generator().manual_seed(10)
    q, k, v = inputs(gen, [40], [50], 2, 64, torch.bfloat16)
    out = run(q, k, v, [-7, 20, 1000], [-3, 30, 2000], 0.125, longest=(40, 50))
    want = run(q, k, v, [0, 20, 40], [0, 30, 50], 0.125)
    assert torch.equal(out, want)
    out = run(q, k, v, [10, 5, 20], [20, 10, 40], 0.125, longest=(40, 50))
    want = run(q[5:20], k[10:40], v[10:40], [0, 15], [0, 30], 0.125)
    assert torch.equal(out[5:20], want) and bool((out[:5] == 5).all())
    assert bool((run(q, k, v, [0], [0], 0.125) == 5).all())
    assert run(q[:0], k, v, [0, 0], [0, 50], 0.125).shape == (0, 2, 64)
    assert not run(q, k[:0], v[:0], [0, 40], [0, 0], 0.125).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    gen = torch.Generator().manual_seed(11)
    for offset, head, token in ((0, 64, 256), (1, 65, 333), (8, 72, 200), (4, 64, 132)):
        bases = [torch.randn(n * token + 900, generator=gen).to(dtype).to(DEV) for n in (45, 99, 99)]
        q, k, v = (b.as_strided((n, 2, 64), (token, head, 1), offset)
                   for b, n in zip(bases, (45, 99, 99)))
        check(q, k, v, [0, 40, 45], [0, 9, 99], 0.125)
        buffer = torch.empty(45 * 128 + 3, dtype=dtype, device=DEV)
        out = buffer[3:].view(45, 2, 64)
        check(q, k, v, [0, 40, 45], [0, 9, 99], 0.125, out=out)
    # broadcast keys and heads, the output in the query's place
    q, k, v = inputs(gen, [45], [99], 1, 64, dtype)
    k, v = k[:1].expand(99, 3, 64), v.expand(99, 3, 64)
    q = q.repeat(1, 3, 1)
    a = check(q, k, v, [0, 40, 45], [0, 9, 99], 0.125)
    assert torch.equal(run(q, k, v, [0, 40, 45], [0, 9, 99], 0.125, out=q), a)
    assert torch.equal(q, a)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("std,scale", [(0.01, 1.0), (8.0, 1.0), (1.0, -0.125), (1.0, 0.0),
                                       (300.0, 30.0), (1.0, 1e-30), (1.0, 1e30), (100.0, -1e4)])
def test_scores_of_any_size(dtype, std, scale):
    gen = torch.Generator().manual_seed(13)
    queries, keys = [40, 150], [200, 77]
    q, k, v = inputs(gen, queries, keys, 2, 64, dtype, std)
    if abs(scale) * std <= 100:
        check(q, k, v, starts_of(queries), starts_of(keys), scale)
        return
    # the largest score takes all of the weight where the next is 2^-8 of it away
    out = run(q, k, v, starts_of(queries), starts_of(keys), scale)
    for a, b, c, d in ((0, 40, 0, 200), (40, 190, 200, 277)):
        x = [t.double().cpu().transpose(0, 1) for t in (q[a:b], k[c:d], v[c:d])]
        top, at = (torch.matmul(x[0], x[1].transpose(1, 2)) * math.copysign(1, scale)).topk(2, -1)
        clear = top[..., 0] - top[..., 1] > top[..., 0].abs() / 256
        want = torch.gather(x[2], 1, at[..., :1].expand(-1, -1, 64)).transpose(0, 1)
        got = out[a:b].double().cpu()
        assert bool(clear.any())
        assert torch.equal(got[clear.T], want[clear.T])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("keys", [100, 2500])
def test_infinities_and_nan(dtype, keys):
    """NaN stays in its own sequence, query and head; a key of score -inf has no weight."""
    gen = torch.Generator().manual_seed(14)
    q, k, v = inputs(gen, [40, 10], [keys, 30], 2, 64, dtype)
    clean = run(q, k, v, [0, 40, 50], [0, keys, keys + 30], 0.125)
    q2 = q.clone()
    q2[7, 1, 3] = math.nan
    out = run(q2, k, v, [0, 40, 50], [0, keys, keys + 30], 0.125)
    assert out[7, 1].isnan().all()
    out[7, 1] = clean[7, 1]
    assert torch.equal(out, clean)
    v2 = v.clone()
    v2[5, 0, 9] = math.nan
    out = run(q, k, v2, [0, 40, 50], [0, keys, keys + 30], 0.125)
    assert out[:40, 0, 9].isnan().all()
    out[:40, 0, 9] = clean[:40, 0, 9]
    assert torch.equal(out, clean)
    k2, q2 = k.clone(), q.abs() + 0.1
    k2[3] = 0.0
    k2[3, :, 0] = -math.inf
    if dtype != torch.float32:  # (an fp32 infinity is not a sum of finite terms)
        out = run(q2, k2, v, [0, 40, 50], [0, keys, keys + 30], 0.125)
        rest = [torch.cat([t[:3], t[4:]]) for t in (k2, v)]
        found = cross(q2, *rest, [0, 40, 50], [0, keys - 1, keys + 29], 0.125)
        limit = cross_tolerance(dtype, 64, keys, *found)
        assert bool(((out.double().cpu() - found[0]).abs() <= limit).all())


def test_largest_operands():
    """fp32 operands next to the type's largest stay finite."""
    q = torch.zeros(3, 1, 64, device=DEV)
    q[:, 0, 0] = torch.tensor([3.4e38, -3.4e38, 1.0])
    k = torch.zeros(4, 1, 64, device=DEV)
    k[:, 0, 0] = torch.tensor([1e-38, 2e-38, -1e-38, 0.0])
    v = torch.full((4, 1, 64), 3.4e38, device=DEV)
    check(q, k, v, [0, 3], [0, 4], 1.0)


@pytest.mark.parametrize("keys", [70, 5000])
def test_graphs(keys):
    """Captured and replayed over new inputs and lengths, two graphs at once, with eager work
    between the replays."""
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(15)
    states, graphs = [], []

    def call(s):
        hip_attn.packed_cross_attention(s["q"], s["k"], s["v"], s["out"], s["qs"], s["ks"],
                                        scale=0.125, max_query_len=40, max_key_len=keys)

    for _ in range(2):
        q, k, v = inputs(gen, [40], [keys], 2, 64, torch.bfloat16)
        s = dict(q=q, k=k, v=v, out=torch.zeros_like(q),
                 qs=torch.tensor([0, 10, 40], dtype=torch.int32, device=DEV),
                 ks=torch.tensor([0, 30, keys], dtype=torch.int32, device=DEV))
        call(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(s)
        states.append(s)
        graphs.append(graph)
    for turn in range(4):
        for s in states:
            s["q"].normal_()
            s["ks"][1] = 3 + 11 * turn
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s in states:
            got = s["out"].clone()
            call(s)
            assert torch.equal(s["out"], got), turn


def test_other_stream_gradients_and_versions():
    gen = torch.Generator().manual_seed(16)
    q, k, v = inputs(gen, [40], [90], 2, 64, torch.float32)
    want = run(q, k, v, [0, 40], [0, 90], 0.125)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        out = run(q, k, v, [0, 40], [0, 90], 0.125)
    stream.synchronize()
    assert torch.equal(out, want)
    leaf = q.clone().requires_grad_()
    for args in ((leaf, k, v), (q, leaf[:1].expand(90, 2, 64), v)):
        with pytest.raises(RuntimeError, match="no gradient"):
            run(*args, [0, 40], [0, 90], 0.125)
    with torch.no_grad():
        assert torch.equal(run(leaf, k, v, [0, 40], [0, 90], 0.125), want)
    version = out._version
    run(q, k, v, [0, 40], [0, 90], 0.125, out=out)
    assert out._version > version


@pytest.mark.parametrize("which", ["query", "key", "value", "far"])
def test_a_misaligned_tensor_is_copied_alone(which):
    """One operand at an odd element or, ``far``, of a token stride past the kernel's: of the
    others nothing is copied."""
    gen = torch.Generator().manual_seed(19)
    sizes = dict(query=9, key=5000, value=5000)
    at = {}
    for name, rows in sizes.items():
        odd = int(name == which)
        base = torch.randn(rows * 128 + odd, generator=gen).to(torch.bfloat16).to(DEV)
        at[name] = base[odd:].view(rows, 2, 64)
    if which == "far":
        base = torch.zeros(40, (1 << 22) + 8, dtype=torch.bfloat16, device=DEV)
        base[:, :128].copy_(at["key"][:40].flatten(1))
        at["key"], at["value"] = base[:, :128].view(40, 2, 64), at["value"][:40]
    keys = at["key"].shape[0]
    aligned = [x.clone(memory_format=torch.contiguous_format) for x in at.values()]
    want = check(*aligned, [0, 9], [0, keys], 0.125, longest=(9, 64))  # (one part: no workspace)
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    assert torch.equal(run(*at.values(), [0, 9], [0, keys], 0.125, longest=(9, 64), out=out), want)
    used = torch.cuda.max_memory_allocated() - before
    copied = at.get(which, at["key"]).numel() * 2
    assert copied <= used <= copied + (1 << 14), (used, copied)


def test_refuses_its_keys_or_values_as_the_output():
    gen = torch.Generator().manual_seed(20)
    q, _, _ = inputs(gen, [40], [1], 2, 64, torch.float32)
    k, v = torch.ones_like(q), torch.zeros_like(q)
    for args, out in (((q, k, v), k), ((q, k, v), v), ((q, q, q), q)):
        with pytest.raises(ValueError, match="memory of its own"):
            run(*args, [0, 40], [0, 40], 0.125, out=out)
    assert bool((k == 1).all()) and not v.any() and q.any()
    assert not run(q, k, v, [0, 40], [0, 40], 0.125, out=q).any()
    # (no queries, or no keys, no address to share)
    run(q[:0], k, v, [0, 0], [0, 40], 0.125)
    run(q, k[:0], v[:0], [0, 40], [0, 0], 0.125)


@pytest.mark.parametrize("sequences", [63, 64, 127, 300, 3969, 3970, 5000])
@pytest.mark.parametrize("longest", [(3, 5), (200, 90)])
def test_many_sequences(sequences, longest):
    """More than a wave looks up at a time, once and twice over, empty ones among them."""
    gen = torch.Generator().manual_seed(sequences)
    queries = torch.randint(0, 4, (sequences,), generator=gen)
    keys = torch.randint(0, 6, (sequences,), generator=gen)
    queries[torch.rand(sequences, generator=gen) < 0.3] = 0
    queries[sequences // 2], keys[sequences // 2] = longest[0], longest[1]
    queries[-1], keys[0] = longest[0], longest[1]
    queries, keys = queries.tolist(), keys.tolist()
    q, k, v = inputs(gen, queries, keys, 1, 32, torch.bfloat16)
    check(q, k, v, starts_of(queries), starts_of(keys), 0.2)


def test_rows_far_apart():
    """Queries, keys and values whose last rows lie past 2^31 elements."""
    gen = torch.Generator().manual_seed(23)
    rows, step = 70000, 32768  # 2.3e9 elements
    base = torch.zeros(rows, step, dtype=torch.bfloat16, device=DEV)
    q, k, v = (base[:, a: a + 64].view(rows, 1, 64) for a in (0, 64, 128))
    at = [0, 5, rows - 300, rows - 40, rows]
    for x in (q, k, v):
        for a, b in ((0, 5), (rows - 300, rows)):
            x[a:b] = torch.randn(b - a, 1, 64, generator=gen).to(torch.bfloat16).to(DEV)
    out = run(q, k, v, at, at, 0.125)
    tail = [x[rows - 300:].contiguous() for x in (q, k, v)]
    found = cross(*tail, [0, 260, 300], [0, 260, 300], 0.125)
    limit = cross_tolerance(torch.bfloat16, 64, 260, *found)
    assert bool(((out[rows - 300:].double().cpu() - found[0]).abs() <= limit).all())
    found = cross(*(x[:5].contiguous() for x in (q, k, v)), [0, 5], [0, 5], 0.125)
    limit = cross_tolerance(torch.bfloat16, 64, 5, *found)
    assert bool(((out[:5].double().cpu() - found[0]).abs() <= limit).all())
    assert not out[5: rows - 300].any()
