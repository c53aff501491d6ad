"""Token scoring on the GPU against log_softmax in 64 bits: figures within derived bounds,
alternatives exactly, over vocabularies of one value to rows longer than a workgroup holds."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def check(logits, tokens, k, got):
    """`got` against the definition.  With t = x - max and e = exp(t): t is rounded once
    (2^-24 |t|) and scaled by log2 e (as much again), and the exponential is good to 2^-22,
    so e is off by (|t| 2^-23 + 2^-22) of itself; S adds at most 256 terms in a chain and 20
    partial sums.  W / S carries the same, weighted by |t|."""
    logprobs, entropy, top, ids = got
    x = logits.double()
    t = x - x.amax(1, keepdim=True)
    e = t.exp()
    S = e.sum(1)
    p = e / S[:, None]
    size = torch.where(p > 0, t.abs(), 0.0)
    chain = (min(256, -(-x.shape[1] // 256)) + 20) * 2.0**-24
    off_s = (p * (size * 2.0**-23 + 2.0**-22)).sum(1) + chain
    w = (p * size).sum(1)
    off_w = (p * size * (size * 2.0**-23 + 2.0**-22)).sum(1) + w * (chain + off_s + 2.0**-23)
    logp = t - S.log()[:, None]

    def near(have, want, tol):
        assert have.dtype == torch.float32
        # (a logprob past fp32's range is -inf in fp32)
        same = (have == want.float()) | ((have.double() - want).abs() <= tol)
        assert same.all(), ((have.double() - want).abs() / tol).nan_to_num(0).max()

    tol = off_s + 2.0**-23 * (1 + S.log())
    wide = tokens if tokens.dim() == 2 else tokens[:, None]
    want = logp.gather(1, wide)
    near(logprobs.view(want.shape), want,
         tol[:, None] + 2.0**-23 * want.abs().nan_to_num(0, posinf=0))
    assert logprobs.shape == tokens.shape
    near(entropy, S.log() + w, off_s + off_w + 2.0**-23 * (1 + S.log() + w))
    if k == 0:
        assert top is None and ids is None
        return
    order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
    assert ids.dtype == torch.int64 and torch.equal(ids, order)
    best = logp.gather(1, order)
    near(top, best, tol[:, None] + 2.0**-23 * best.abs().nan_to_num(0, posinf=0))


def score(logits, tokens, k):
    from vflorence_amd import decoder_ops

    return decoder_ops.token_logprobs(logits, tokens, k)


def case(rows, vocab, dtype, seed=0, std=2.5, pad=0):
    gen = torch.Generator().manual_seed(seed + rows + vocab)
    logits = (torch.randn(rows, vocab + pad, generator=gen) * std).to(dtype).to(DEV)
    tokens = torch.randint(0, vocab, (rows,), generator=gen).to(DEV)
    return logits[:, :vocab], tokens


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 3, 7, 8, 9, 63, 64, 65, 255, 1000, 4097, 12289, 33000,
                                   50265, 51289, 57344, 57345, 65536, 130001, 256000])
def test_vocabularies(dtype, vocab):
    for rows, k in ((3, min(20, vocab)), (2, 0), (1, min(5, vocab))):
        logits, tokens = case(rows, vocab, dtype)
        check(logits, tokens, k, score(logits, tokens, k))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 9, 64, 257, 700])
@pytest.mark.parametrize("vocab", [5000, 50265])
def test_row_counts(dtype, rows, vocab):
    for k in (0, 1, 8, 20):
        logits, tokens = case(rows, vocab, dtype, seed=k)
        check(logits, tokens, k, score(logits, tokens, k))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [50, 5001, 50265, 130001])
@pytest.mark.parametrize("std", [0.0, 1e-3, 0.3, 40.0])
def test_flat_peaked_and_tied_rows(dtype, vocab, std):
    """Equal values keep the order of their ids; one-hot rows; values far below the best."""
    logits, tokens = case(4, vocab, dtype, std=std)
    logits[1] = logits[1].mul(2).round()  # many ties
    logits[2, vocab // 3] = 60000.0  # every other weight is 0
    check(logits, tokens, 20, score(logits, tokens, 20))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [31, 5001, 50265, 130001])
def test_masked_values(dtype, vocab):
    """-inf and the type's lowest value in masked places; fewer values left than k."""
    logits, tokens = case(5, vocab, dtype)
    logits[0, ::2] = -math.inf
    logits[1, 3:] = -math.inf
    logits[2, : vocab - 1] = -math.inf
    logits[3, 2:] = torch.finfo(dtype).min
    logits[4, tokens[4]] = -math.inf
    got = score(logits, tokens, 20)
    check(logits, tokens, 20, got)
    assert got[0][4] == -math.inf


@pytest.mark.parametrize("vocab", [31, 5001, 50265, 130001])
@pytest.mark.parametrize("k", [0, 6])
def test_rows_without_a_distribution(vocab, k):
    logits, tokens = case(6, vocab, torch.float32)
    logits[1, vocab - 1] = math.nan
    logits[2, 4] = math.inf
    logits[3] = -math.inf
    logits[4, vocab // 2] = -math.nan
    logprobs, entropy, top, ids = score(logits, tokens, k)
    lost = torch.tensor([False, True, True, True, True, False], device=DEV)
    assert torch.equal(logprobs.isnan(), lost) and torch.equal(entropy.isnan(), lost)
    if k:
        assert torch.equal(top.isnan(), lost[:, None].expand(6, k))
        assert torch.equal(ids == -1, lost[:, None].expand(6, k))
    keep = ~lost
    check(logits[keep], tokens[keep], k, [t if t is None else t[keep]
                                          for t in (logprobs, entropy, top, ids)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [31, 5001, 50265, 130001])
@pytest.mark.parametrize("left", [0, 1, 3])
def test_rows_of_nan(dtype, vocab, left):
    """All NaN but for fewer values than k: every place of the alternatives is written."""
    k = 6
    logits, tokens = case(3, vocab, dtype)
    score(logits, tokens, k)  # (whose memory the next call's results may take)
    logits[1] = math.nan
    logits[1, vocab - left :] = 1.0
    logprobs, entropy, top, ids = score(logits, tokens, k)
    assert logprobs[1].isnan().all() and entropy[1].isnan()
    assert top[1].isnan().all() and (ids[1] == -1).all()
    keep = [0, 2]
    check(logits[keep], tokens[keep], k, [t[keep] for t in (logprobs, entropy, top, ids)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [9, 50265, 130001])
def test_given_tokens(dtype, vocab):
    """Several tokens a row, the first and last ones, the same one twice, ones outside."""
    logits, _ = case(3, vocab, dtype)
    tokens = torch.tensor([[0, vocab - 1, vocab // 2, vocab // 2]] * 3, device=DEV)
    check(logits, tokens, 2, score(logits, tokens, 2))
    outside = torch.tensor([[-1, 0], [vocab, 1], [-100, 1 << 40]], device=DEV)
    logprobs = score(logits, outside, 0)[0]
    assert logprobs.isnan().tolist() == [[True, False], [True, False], [True, True]]
    many = torch.arange(vocab, device=DEV).repeat(3, 1)[:, :3000]
    check(logits, many, 0, score(logits, many, 0))
    none = torch.empty(3, 0, dtype=torch.int64, device=DEV)
    assert score(logits, none, 1)[0].shape == (3, 0)
    strided = torch.stack([tokens, tokens], dim=2)[:, :, 0]
    check(logits, strided, 0, score(logits, strided, 0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [100, 50265, 130001])
@pytest.mark.parametrize("offset,pad", [(0, 7), (1, 0), (3, 2), (5, 8)])
def test_rows_at_any_alignment(dtype, vocab, offset, pad):
    gen = torch.Generator().manual_seed(offset)
    flat = (torch.randn(offset + 3 * (vocab + pad), generator=gen) * 2).to(dtype).to(DEV)
    logits = flat.as_strided((3, vocab), (vocab + pad, 1), offset)
    tokens = torch.randint(0, vocab, (3,), generator=gen).to(DEV)
    check(logits, tokens, 20, score(logits, tokens, 20))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [31, 5001, 50265, 130001])
@pytest.mark.parametrize("level", [2e38, -2e38, -3.3e38])
def test_rows_at_the_types_limits(dtype, vocab, level):
    """Maxima whose product with log2 e overflows: the weight lies on the equal values alone.
    A row masked throughout with one low value is uniform."""
    logits, tokens = case(4, vocab, dtype)
    logits[0] = level
    logits[1] = torch.where(logits[1] > 0, level, torch.finfo(dtype).min)
    logits[2] = -math.inf
    logits[2, vocab // 2:] = level
    logits[3, tokens[3]] = level
    got = score(logits, tokens, 5)
    check(logits, tokens, 5, got)
    assert abs(float(got[1][0]) - math.log(vocab)) < 1e-5


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [3000, 50265, 130001])
def test_rows_below_zero(dtype, vocab):
    """Log probabilities themselves, -0.0 and 0.0 among the best, and the same bits again."""
    logits, tokens = case(5, vocab, dtype)
    logits.copy_(torch.log_softmax(logits.float(), 1))
    logits[3:] = logits[3:].clamp(max=-2.0)
    logits[2, [5, 900, 77]] = torch.tensor([-0.0, 0.0, 0.0], dtype=dtype, device=DEV)
    logits[4, 100:130:2], logits[4, 101:130:2] = 0.0, -0.0
    for k in (2, 3, 9):
        check(logits, tokens, k, score(logits, tokens, k))
    got = score(logits, tokens, 20)
    check(logits, tokens, 20, got)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(got, score(logits, tokens, 20)))


@pytest.mark.parametrize("vocab", [1003, 50265, 130001])
def test_broadcast_rows(vocab):
    """One row repeated by a stride of 0, and a single row whose stride says nothing."""
    logits, _ = case(1, vocab, torch.bfloat16)
    tokens = torch.arange(5, device=DEV)
    wide = logits.expand(5, -1)
    check(wide, tokens, 4, score(wide, tokens, 4))
    one = logits.as_strided((1, vocab), (3, 1))
    check(one, tokens[:1], 4, score(one, tokens[:1], 4))


def test_best_values_side_by_side():
    """All alternatives inside one thread's share of the row, ascending, and at its ends."""
    for vocab in (3000, 50265, 130001):
        logits, tokens = case(3, vocab, torch.float32)
        logits[0, 512: 532] = torch.arange(20.0, device=DEV) + 50
        logits[1, -20:] = torch.arange(20.0, device=DEV) + 50
        logits[2, :1500] = 50.0
        check(logits, tokens, 20, score(logits, tokens, 20))


def test_graph_stream_and_gradient():
    logits, tokens = case(5, 50265, torch.bfloat16)
    want = [t.clone() for t in score(logits, tokens, 8)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = score(logits, tokens, 8)
    for turn in range(3):
        graph.replay()
        other = score(*case(7, 51289, torch.bfloat16, seed=turn), 4)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)) and len(other) == 4
        logits.copy_(logits.flip(1))
        graph.replay()
        check(logits, tokens, 8, held)
        logits.copy_(logits.flip(1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = score(logits, tokens, 8)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    leaf = logits.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        score(leaf, tokens, 0)
    with torch.no_grad():
        score(leaf, tokens, 0)
    assert score(logits[:0], tokens[:0], 3)[2].shape == (0, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [31, 5001, 50265, 130001])
@pytest.mark.parametrize("level", [65535.5, 65600.0, 1e6, 3e7, 1e9, 3e9, 5e9, 1e10, 1e12, 1e20,
                                   1e30, 9e37])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_rows_of_any_magnitude(dtype, vocab, level, sign):
    """Maxima whose product with log2 e no longer holds units: uniform rows, neighbouring
    values, low values among and before ordinary ones, one value far above the others."""
    logits, tokens = case(8, vocab, dtype)
    noise = logits.float().clone()
    level = float(torch.tensor(sign * level).to(dtype))
    half = torch.arange(vocab, device=DEV) < vocab // 2
    logits[0] = level
    logits[1] = (level + noise[1]).to(dtype)  # steps of the type about the level
    logits[2, half] = -math.inf
    logits[2, ~half] = level
    logits[3, tokens[3]] = level
    logits[4] = (noise[4] * (level / 4)).to(dtype)
    logits[5] = torch.where(half, -abs(level), noise[5]).to(dtype)
    logits[6] = torch.where(noise[6] > 0, -abs(level), noise[6]).to(dtype)
    logits[7] = -abs(level)
    logits[7, tokens[7]] = 1.0
    for k in (5, 0):
        got = score(logits, tokens, k)
        check(logits, tokens, k, got)
    assert abs(float(got[1][0]) - math.log(vocab)) < 1e-5


@pytest.mark.parametrize("vocab", [31, 5001, 50265, 130001])
@pytest.mark.parametrize("level", [1e10, -1e10])
def test_large_rows_without_a_distribution(vocab, level):
    logits, tokens = case(4, vocab, torch.float32)
    logits[:] = level
    logits[1, vocab - 1] = math.nan
    logits[2, 4] = math.inf
    logprobs, entropy, top, ids = score(logits, tokens, 6)
    lost = torch.tensor([False, True, True, False], device=DEV)
    assert torch.equal(logprobs.isnan(), lost) and torch.equal(entropy.isnan(), lost)
    assert torch.equal(top.isnan(), lost[:, None].expand(4, 6))
    assert torch.equal(ids == -1, lost[:, None].expand(4, 6))
    keep = ~lost
    check(logits[keep], tokens[keep], 6, [t[keep] for t in (logprobs, entropy, top, ids)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [31, 5001, 50265, 130001])
@pytest.mark.parametrize("gap", [3.0, 8.0, 12.0, 15.0])
def test_confident_rows(dtype, vocab, gap):
    """One token with nearly all of the weight, whose log probability is close to 0; two others
    have the rest, w <= 2 e^-3 < 0.1 of it, and a thread may see any of the low ones first.  A
    weight's exponent is rounded about its thread's reference (which lags by 16 in log2 at most)
    and about the maximum, 31 * 2^-23 of the weight at most, and the exponential is good to 2^-22;
    the largest term is 1.  So 1 + w is off by 0.1 (2^-22 + 31 * 2^-23) and three roundings of
    2^-24 (the division by the largest term, two sums), its log by 2^-23 of itself more."""
    gen = torch.Generator().manual_seed(int(gap) + vocab)
    logits = torch.full((6, vocab), -200.0)
    tokens = torch.randint(0, vocab, (6,), generator=gen)
    for r in range(6):
        others = torch.randperm(vocab, generator=gen)[:2]
        logits[r, others] = 4.0 * r - gap - torch.rand(2, generator=gen)
        logits[r, tokens[r]] = 4.0 * r
    logits, tokens = logits.to(dtype).to(DEV), tokens.to(DEV)
    got = score(logits, tokens, 1)
    want = torch.log_softmax(logits.double(), 1).gather(1, tokens[:, None])
    bound = 0.1 * (2.0**-22 + 31 * 2.0**-23) + 3 * 2.0**-24 + 0.1 * 2.0**-23
    for have in (got[0], got[2][:, 0]):
        off = (have.double() - want[:, 0]).abs().max()
        print(f"error / bound {float(off / bound):.3f}", flush=True)
        assert off <= bound
