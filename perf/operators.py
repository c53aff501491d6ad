"""Performance cases of the operators around a K/V cache held in 8 bits, and of scoring:

append  -- new keys and values quantised into the paged cache, one power-of-two scale per
           block of tokens and head
attend  -- decode attention over that cache, the beams of a request sharing its pages
score   -- log probabilities of given tokens, each row's entropy and its best alternatives

A cache holds e4m3 values; value * scales[block, head, 0 or 1] is the key or value they
stand for.  K pools are [blocks, heads, block, dim]; V pools keep a block's tokens in groups
of four, [block / 4][dim][4] inside the same shape.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # The step of a lone four-beam request: four new tokens, each in its own block.
        dict(name="append_single", kind="append", sequences=4, shortest=1, longest=1, prior=72,
             heads=12, dim=64, block=16, dtype="bf16"),
        # The step of the throughput batch, 64 requests x 4 beams.
        dict(name="append_step", kind="append", sequences=256, shortest=1, longest=1, prior=1000,
             heads=16, dim=64, block=16, dtype="bf16"),
        # The encoder K/V of 64 admitted prompts of mixed lengths, one layer.
        dict(name="append_prompts", kind="append", sequences=64, shortest=256, longest=1024,
             prior=0, heads=16, dim=64, block=16, dtype="bf16"),
        # Cross-attention of a lone four-beam request over an image's tokens and a short text.
        dict(name="attend_single", kind="attend", groups=1, beams=4, shortest=590, longest=590,
             idle=0, heads=12, dim=64, block=16, dtype="bf16"),
        # Greedy decoding under continuous batching: rows at every length, an odd count.
        dict(name="attend_greedy", kind="attend", groups=93, beams=1, shortest=6, longest=1000,
             idle=3, heads=16, dim=64, block=16, dtype="fp16"),
        # Cross-attention of the throughput batch, 64 requests x 4 beams.
        dict(name="attend_batch", kind="attend", groups=64, beams=4, shortest=256, longest=1024,
             idle=0, heads=16, dim=64, block=16, dtype="bf16"),
        # Two rows over very long contexts, wider heads: the work has to be split over tokens.
        dict(name="attend_long", kind="attend", groups=2, beams=1, shortest=17001, longest=39999,
             idle=0, heads=8, dim=128, block=32, dtype="bf16"),
        # The engine's default data type with beams.
        dict(name="attend_fp32", kind="attend", groups=16, beams=4, shortest=256, longest=1024,
             idle=0, heads=16, dim=64, block=16, dtype="fp32"),
        # A lone four-beam request's candidates with eight alternatives each.
        dict(name="score_single", kind="score", rows=4, vocab=51289, keep=8, dtype="bf16"),
        # One step of the throughput batch, the chosen tokens alone.
        dict(name="score_batch", kind="score", rows=256, vocab=50265, keep=0, dtype="bf16"),
        # The engine's default data type, an odd number of rows, the most alternatives.
        dict(name="score_fp32", kind="score", rows=93, vocab=51289, keep=20, dtype="fp32"),
        # Four documents of 1024 tokens scored in one pass, five alternatives per token.
        dict(name="score_text", kind="score", rows=4096, vocab=50265, keep=5, dtype="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], evenly over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("append", "attend", "attend", "score"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind == "score":
        vocab = rng.choice((50265, 51289, _spread(rng, 1000, 200000)))
        most = (400 << 20) // (vocab * (4 if dtype == "fp32" else 2))
        return dict(kind=kind, rows=_spread(rng, 1, min(4096, most)), vocab=vocab,
                    keep=rng.choice((0, rng.randint(1, 8), rng.randint(1, 20))), dtype=dtype)
    heads = rng.choice((8, 12, 16))
    dim = rng.choice((64, 64, 128, rng.choice((32, 48, 80, 96, 112, 160, 256))))
    block = rng.choice((16, 16, 32))
    if kind == "append":
        if rng.random() < 0.5:  # a decode step
            return dict(kind=kind, sequences=_spread(rng, 1, 512), shortest=1, longest=1,
                        prior=_spread(rng, 1, 1000), heads=heads, dim=dim, block=block,
                        dtype=dtype)
        longest = _spread(rng, 2, 1024)  # prompts, or parts of them after earlier ones
        most = (40 << 20) // (longest * heads * dim)
        return dict(kind=kind, sequences=_spread(rng, 1, max(2, min(64, most))),
                    shortest=max(1, int(longest * rng.uniform(0.05, 1.0))), longest=longest,
                    prior=rng.choice((0, _spread(rng, 1, 500))), heads=heads, dim=dim,
                    block=block, dtype=dtype)
    longest = _spread(rng, 8, 40000)
    most = (80 << 20) // (longest * heads * dim)
    beams = rng.choice((1, 1, 2, 3, 4, 5, 8))
    return dict(kind=kind, groups=_spread(rng, 1, max(2, min(512 // beams, most))), beams=beams,
                shortest=max(1, int(longest * rng.uniform(0.02, 1.0))), longest=longest,
                idle=rng.choice((0, 0, rng.randint(1, 5))), heads=heads, dim=dim, block=block,
                dtype=dtype)


# ---------------------------------------------------------------------------
# what the case alone decides
# ---------------------------------------------------------------------------
def _lengths(low, high, count):
    """``count`` lengths evenly over [low, high], in a fixed mixed order."""
    lens = [low + round((high - low) * (i + 0.5) / count) for i in range(count)]
    random.Random(count).shuffle(lens)
    return lens


def _append_plan(case):
    """Per sequence, how many tokens it has and how many are new."""
    n = case["sequences"]
    new = _lengths(case["shortest"], case["longest"], n)
    prior = [round(case["prior"] * (i + 0.5) / n) for i in range(n)]
    return prior, new


def _attend_lengths(case):
    return _lengths(case["shortest"], case["longest"], case["groups"]) + [0] * case["idle"]


def _size(case):
    return DTYPES[case["dtype"]].itemsize


def work(case):
    if case["kind"] == "score":
        cells = case["rows"] * case["vocab"]
        # the logits and tokens read; log probability, entropy and alternatives written;
        # per value a difference, an exponential, two sums and a product
        return dict(bytes=cells * _size(case) + case["rows"] * (16 + 12 * case["keep"]),
                    flops=5 * cells)
    heads, dim, block = case["heads"], case["dim"], case["block"]
    if case["kind"] == "append":
        prior, new = _append_plan(case)
        tokens = sum(new)
        blocks = sum((p + n - 1) // block - p // block + 1 for p, n in zip(prior, new))
        # keys and values read and stored, slots read, scales read and written
        return dict(bytes=2 * tokens * heads * dim * (_size(case) + 1) + 8 * tokens
                    + 16 * blocks * heads, flops=4 * tokens * heads * dim)
    lens = _attend_lengths(case)
    rows, blocks = len(lens) * case["beams"], sum(-(-n // block) for n in lens)
    # each group's K and V once, their scales and ids, the queries and outputs
    return dict(bytes=2 * sum(lens) * heads * dim + 8 * blocks * heads + 4 * blocks
                + 2 * rows * heads * dim * _size(case),
                flops=4 * case["beams"] * sum(lens) * heads * dim)


# ---------------------------------------------------------------------------
# what the seed decides
# ---------------------------------------------------------------------------
def _e4m3(gen, shape, std):
    """Cache contents: e4m3 values as a scale that fits them leaves behind."""
    return torch.randn(shape, generator=gen, device="cuda").mul_(std).clamp_(-448, 448).to(E4M3)


def _scales(gen, blocks, heads, low, high):
    e = torch.randint(low, high + 1, (blocks, heads, 2), generator=gen, device="cuda")
    return ((e + 127) << 23).int().view(torch.float32)  # 2^e


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case=case)
    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        # the LM head's logits: rows padded to a multiple of eight values, the tokens that
        # generation never emits at -inf
        wide = torch.empty(rows, -(-vocab // 8) * 8, dtype=dtype, device="cuda")
        wide.normal_(0.0, 2.5, generator=gen)
        logits = wide[:, :vocab]
        logits[:, torch.tensor([0, 3, vocab - 1], device="cuda")] = -math.inf
        tokens = torch.randint(4, vocab - 1, (rows,), generator=gen, device="cuda")
        tokens[::2] = logits[::2].argmax(dim=1)  # half of them the model's own choice
        return dict(state, logits=logits, tokens=tokens)
    heads, dim, block = case["heads"], case["dim"], case["block"]
    placing = random.Random(seed)
    if case["kind"] == "append":
        prior, new = _append_plan(case)
        spans = [(p // block, (p + n - 1) // block + 1) for p, n in zip(prior, new)]
        pool = sum(b - a for a, b in spans) + 8
        ids = torch.tensor(placing.sample(range(pool), pool - 8))
        count = torch.tensor(new)
        first = torch.tensor([p % block for p in prior])  # offset in the span's first block
        held = torch.tensor([b - a for a, b in spans])
        seq = torch.repeat_interleave(torch.arange(len(new)), count)
        at = first[seq] + torch.arange(int(count.sum())) - (count.cumsum(0) - count)[seq]
        slots = ids[(held.cumsum(0) - held)[seq] + at // block] * block + at % block
        tokens = slots.numel()
        # keys and values are the last thirds of a fused projection's rows
        qkv = torch.empty(tokens, 3, heads, dim, dtype=dtype, device="cuda")
        qkv.normal_(0.0, 1.0, generator=gen)
        return dict(state, key=qkv[:, 1], value=qkv[:, 2], slots=slots.cuda(),
                    k_cache=_e4m3(gen, (pool, heads, block, dim), 100.0),
                    v_cache=_e4m3(gen, (pool, heads, block, dim), 100.0),
                    scales=_scales(gen, pool, heads, -9, -6))
    lens = _attend_lengths(case)
    beams, width = case["beams"], max(-(-max(lens) // block), 1)
    counts = [-(-n // block) for n in lens]
    pool = sum(counts) + 8
    ids = placing.sample(range(pool), pool - 8)
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    starts = torch.tensor([0] + counts).cumsum(0)
    filled = torch.arange(width)[None] < torch.tensor(counts)[:, None]
    table[filled] = torch.tensor(ids, dtype=torch.int32)[: int(starts[-1])]
    lengths = torch.tensor(lens, dtype=torch.int32)
    rows = len(lens) * beams
    query = torch.empty(rows, heads, dim, dtype=dtype, device="cuda")
    query.normal_(0.0, 1.0, generator=gen)
    return dict(state, query=query, scale=dim**-0.5,
                table=table.repeat_interleave(beams, 0).cuda(),
                lengths=lengths.repeat_interleave(beams).cuda(),
                starts=(torch.arange(len(lens) + 1, dtype=torch.int32) * beams).cuda(),
                order=torch.argsort(lengths, descending=True, stable=True).int().cuda(),
                k_cache=_e4m3(gen, (pool, heads, block, dim), 100.0),
                v_cache=_e4m3(gen, (pool, heads, block, dim), 100.0),
                scales=_scales(gen, pool, heads, -8, -6))


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _OWN[kind](state)
    return _PLAIN[kind](state)


def _own_append(s):
    from vflorence_amd import hip_attn

    hip_attn.reshape_and_cache_8bit(s["key"], s["value"], s["k_cache"], s["v_cache"],
                                    s["scales"], s["slots"])
    return dict(k=s["k_cache"], v=s["v_cache"], scales=s["scales"])


def _own_attend(s):
    from vflorence_amd import hip_attn

    meta, case, q = s.get("metadata"), s["case"], s["query"]
    if meta is None:  # made once per batch, as the engine does
        meta = s["metadata"] = hip_attn.get_scheduler_metadata(
            num_reqs=q.shape[0], num_heads=case["heads"], num_kv_heads=case["heads"],
            head_dim=case["dim"], dtype=q.dtype, block_size=case["block"],
            group_start=s["starts"] if case["beams"] > 1 else None, group_order=s["order"],
            max_group_size=case["beams"])
    out = torch.empty_like(q)
    hip_attn.attention_with_kv_cache_8bit(q, s["k_cache"], s["v_cache"], s["scales"], out,
                                          s["lengths"], scale=s["scale"], block_table=s["table"],
                                          scheduler_metadata=meta)
    return out


def _own_score(s):
    from vflorence_amd import decoder_ops

    logprobs, entropy, top, ids = decoder_ops.token_logprobs(s["logits"], s["tokens"],
                                                             s["case"]["keep"])
    if not s["case"]["keep"]:
        return dict(logprobs=logprobs, entropy=entropy)
    return dict(logprobs=logprobs, entropy=entropy, top=top, ids=ids)


def _grouped(v):
    """[..., block, dim] of a V pool's storage, tokens by four -> tokens in order."""
    block, dim = v.shape[-2:]
    return v.unflatten(-2, (block // 4, 4)).reshape(*v.shape[:-2], block // 4, dim, 4) \
        .transpose(-1, -2).reshape(v.shape)


def _regrouped(v):
    """The other way: tokens in order -> a V pool's storage."""
    block, dim = v.shape[-2:]
    return v.reshape(*v.shape[:-2], block // 4, 4, dim).transpose(-1, -2).reshape(v.shape)


def _plain_append(s):
    kc, vc, scales, slots = s["k_cache"], s["v_cache"], s["scales"], s["slots"]
    block = kc.shape[2]
    used, at = torch.unique(slots // block, return_inverse=True)
    off = slots % block
    x = torch.stack([s["key"], s["value"]], dim=2).float()  # [tokens, heads, 2, dim]
    largest = x.abs().amax(dim=-1)  # [tokens, heads, 2]
    amax = torch.zeros(used.numel(), *largest.shape[1:], device=x.device)
    amax.scatter_reduce_(0, at[:, None, None].expand_as(largest), largest, "amax")
    fresh = torch.zeros(used.numel(), dtype=torch.bool, device=x.device)
    fresh[at[off == 0]] = True
    # the smallest power of two that brings the largest value to 448 = 0.875 * 2^9 or less
    mantissa, exponent = torch.frexp(amax)
    exponent = (exponent - 9 + (mantissa > 0.875)).masked_fill(amax == 0, -100).clamp(min=-100)
    need = ((exponent + 127) << 23).view(torch.float32)
    old = scales[used].masked_fill(fresh[:, None, None], 0.0)
    new = torch.maximum(old, need)
    held = torch.stack([kc.view(torch.uint8)[used].view(E4M3).float(),
                        _grouped(vc.view(torch.uint8)[used].view(E4M3).float())], dim=2)
    held = torch.where(fresh[:, None, None, None, None], 0.0, held * (old / new)[..., None, None])
    held[at, :, :, off] = x / new[at][..., None]
    q = held.to(E4M3).view(torch.uint8)
    kc.view(torch.uint8)[used] = q[:, :, 0]
    vc.view(torch.uint8)[used] = _regrouped(q[:, :, 1])
    scales[used] = new
    return dict(k=kc, v=vc, scales=scales)


def _plain_attend(s):
    case, q, block = s["case"], s["query"], s["case"]["block"]
    beams, heads, dim = case["beams"], case["heads"], case["dim"]
    table, lens = s["table"][::beams].long(), s["lengths"][::beams]
    groups, width = table.shape
    pages = [c.view(torch.uint8)[table].view(E4M3).float() for c in (s["k_cache"], s["v_cache"])]
    pages[1] = _grouped(pages[1])
    scales = s["scales"][table]  # [groups, width, heads, 2]
    k, v = ((p * scales[..., i, None, None]).transpose(1, 2).flatten(2, 3)
            for i, p in enumerate(pages))  # [groups, heads, width * block, dim]
    seen = torch.arange(width * block, device=q.device)[None] < lens[:, None]
    x = q.float().view(groups, beams, heads, dim).transpose(1, 2)
    w = torch.matmul(x, k.transpose(-1, -2).contiguous()) * s["scale"]
    w = w.masked_fill(~seen[:, None, None], -math.inf)
    top = w.amax(dim=-1, keepdim=True)
    w = torch.exp(w - top.masked_fill(top == -math.inf, 0.0))
    v = v.masked_fill(~seen[:, None, :, None], 0.0)
    total = w.sum(dim=-1, keepdim=True)
    out = torch.matmul(w, v) / total.masked_fill(total == 0, 1.0)
    return out.transpose(1, 2).reshape(q.shape).to(q.dtype)


def _plain_score(s):
    keep = s["case"]["keep"]
    x = s["logits"].float()
    top = x.amax(dim=1, keepdim=True)
    t = x - top
    e = torch.exp(t)
    total = e.sum(dim=1)
    log_total = total.log()
    logprobs = t.gather(1, s["tokens"][:, None])[:, 0] - log_total
    entropy = log_total - (t * e).masked_fill(e == 0, 0.0).sum(dim=1) / total
    if not keep:
        return dict(logprobs=logprobs, entropy=entropy)
    # one whole number per value that orders by value, then by lower index
    bits = x.view(torch.int32)
    rank = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    places = torch.arange(x.shape[1], device=x.device)
    best = torch.topk((rank << 32) + (x.shape[1] - 1 - places), keep, dim=1).values
    ids = x.shape[1] - 1 - (best & 0xFFFFFFFF)
    return dict(logprobs=logprobs, entropy=entropy,
                top=t.gather(1, ids) - log_total[:, None], ids=ids)


_OWN = dict(append=_own_append, attend=_own_attend, score=_own_score)
_PLAIN = dict(append=_plain_append, attend=_plain_attend, score=_plain_score)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _nearest_e4m3(x):
    """The e4m3 value next to x, ties to the even one: steps of 2^(exponent - 3), 2^-9 at
    least."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0**-6)))
    e = e - (torch.exp2(e) > x.abs().clamp(min=2.0**-6)).double()
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _v_places(block, dim):
    """Where token t's value d lies in a V pool's [block, dim] storage."""
    t, d = torch.arange(block)[:, None], torch.arange(dim)[None]
    return (((t // 4) * dim + d) * 4 + t % 4).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    return dict(append=_exact_append, attend=_exact_attend, score=_exact_score)[case["kind"]](s)


def _exact_append(s):
    slots = s["slots"].tolist()
    pools, block, dim = [s["k_cache"], s["v_cache"]], s["k_cache"].shape[2], s["k_cache"].shape[3]
    scales = s["scales"].double()
    held = [p.float().double().flatten(2) for p in pools]
    places = [torch.arange(block * dim, device="cuda").view(block, dim), _v_places(block, dim)]
    blocks = sorted({n // block for n in slots})
    begun = {n // block for n in slots if n % block == 0}
    touched = torch.tensor(blocks, device="cuda")
    begun = torch.tensor(sorted(begun), dtype=torch.long, device="cuda")
    where = s["slots"] // block
    for i, x in enumerate((s["key"].double(), s["value"].double())):
        largest = torch.zeros(scales.shape[:2], dtype=torch.float64, device="cuda")
        largest.scatter_reduce_(0, where[:, None].expand(-1, x.shape[1]), x.abs().amax(-1),
                                "amax")
        need = torch.exp2(torch.ceil(torch.log2((largest / 448).clamp(min=2.0**-100))))
        was = scales[..., i].clone()
        was[begun] = 0.0
        held[i][begun] = 0.0
        now = torch.maximum(was, need)
        held[i][touched] = _nearest_e4m3(held[i][touched] * (was / now)[touched][..., None])
        for t in range(block):  # a block's slot is written once: no two tokens meet
            mine = (s["slots"] % block == t).nonzero()[:, 0]
            if mine.numel():
                b = where[mine]
                row = held[i][b]
                row[:, :, places[i][t]] = _nearest_e4m3(x[mine] / now[b][..., None])
                held[i][b] = row
        scales[touched, :, i] = now[touched]
    return dict(k=held[0].view(pools[0].shape), v=held[1].view(pools[1].shape), scales=scales)


def _exact_attend(s):
    case, block, dim = s["case"], s["case"]["block"], s["case"]["dim"]
    beams, order = case["beams"], _v_places(block, dim).flatten()
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    for g, n in enumerate(s["lengths"].tolist()[::beams]):
        if n == 0:
            continue
        rows = slice(g * beams, (g + 1) * beams)
        pages = s["table"][g * beams, : -(-n // block)].long()
        scales = s["scales"].double()[pages]
        k = s["k_cache"].view(torch.uint8)[pages].view(E4M3).double() * scales[..., 0, None, None]
        v = s["v_cache"].view(torch.uint8)[pages].view(E4M3).double().flatten(2)[..., order]
        v = v.view(k.shape) * scales[..., 1, None, None]
        k, v = (a.transpose(0, 1).reshape(case["heads"], -1, dim)[:, :n] for a in (k, v))
        q = s["query"][rows].double().transpose(0, 1)
        weights = torch.softmax(q @ k.transpose(1, 2).contiguous() * s["scale"], dim=-1)
        out[rows] = (weights @ v.contiguous()).transpose(0, 1)
    return out


def _exact_score(s):
    keep = s["case"]["keep"]
    found = []
    for x, token in zip(s["logits"].split(256), s["tokens"].split(256)):
        logp = torch.log_softmax(x.double(), dim=1)
        p = logp.exp()
        row = [logp.gather(1, token[:, None])[:, 0],
               -torch.where(p > 0, p * logp, 0.0).sum(dim=1)]
        if keep:  # equal values keep the order of their indices
            ids = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :keep]
            row += [logp.gather(1, ids), ids]
        found.append(row)
    names = ("logprobs", "entropy", "top", "ids")
    return {name: torch.cat(part) for name, part in zip(names, zip(*found))}
