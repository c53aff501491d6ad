"""The 8-bit cache's operators and token scoring refuse bad calls on the host, before
anything is launched; their helpers work on the CPU."""

import pytest
import torch

from tests.cache_8bit_oracle import Cache, nearest_e4m3, needed_scale

E4M3 = torch.float8_e4m3fn
A = 16 * 1000  # a 16-byte aligned stand-in address (never dereferenced)


def test_values_and_layout_helpers():
    from vflorence_amd import hip_attn

    k, v, scales = hip_attn.kv_cache_8bit(3, 2, 16, 32, "cpu")
    assert k.dtype == v.dtype == E4M3 and k.shape == v.shape == (3, 2, 16, 32)
    assert scales.dtype == torch.float32 and scales.shape == (3, 2, 2)
    logical = torch.randn(3, 2, 16, 32).clamp(-4, 4).to(E4M3)
    stored = hip_attn.v_cache_from_logical(logical)
    # token t of dim d lies at ((t / 4) * D + d) * 4 + t % 4 of its block and head
    assert stored.view(torch.uint8).flatten(2)[1, 1, (2 * 32 + 7) * 4 + 3] \
        == logical.view(torch.uint8)[1, 1, 11, 7]
    scales = torch.rand(3, 2, 2)
    kv, vv = hip_attn.kv_cache_8bit_values(logical, stored, scales)
    assert torch.equal(kv, logical.float() * scales[:, :, 0, None, None])
    assert torch.equal(vv, logical.float() * scales[:, :, 1, None, None])
    with pytest.raises(ValueError):
        hip_attn.kv_cache_8bit(3, 2, 24, 64, "cpu")
    with pytest.raises(ValueError):
        hip_attn.kv_cache_8bit(3, 2, 16, 72, "cpu")


def test_oracle_rounds_as_the_type():
    every = torch.arange(256, dtype=torch.uint8).view(E4M3).float().double()
    finite = every[every.isfinite()]
    assert torch.equal(nearest_e4m3(finite), finite)
    x = torch.cat([torch.randn(4000, dtype=torch.float64) * s for s in (1e-3, 0.02, 1, 100)])
    x = x.clamp(-448, 448).float().double()
    assert torch.equal(nearest_e4m3(x), x.float().to(E4M3).float().double())
    for value, scale in ((448.0, 1.0), (448.5, 2.0), (0.0, 2.0**-100), (3.5, 2.0**-7),
                         (1.0, 2.0**-8), (2.0**-120, 2.0**-100)):
        assert needed_scale(torch.tensor([value, -value / 3], dtype=torch.float64)) == scale


def _append_args(dtype=torch.bfloat16):
    from vflorence_amd import hip_attn

    k, v, s = hip_attn.kv_cache_8bit(4, 2, 16, 64, "cpu")
    x = torch.zeros(3, 2, 64, dtype=dtype)
    return dict(key=x, value=x.clone(), k_cache=k, v_cache=v, kv_scales=s,
                slot_mapping=torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize("name,make", [
    ("key", lambda a: a["key"][:, :, :32]),
    ("key", lambda a: a["key"][0]),
    ("key", lambda a: a["key"].to(torch.float16)),
    ("key", lambda a: a["key"].to(torch.float64)),
    ("value", lambda a: a["value"].transpose(1, 2).contiguous().transpose(1, 2)),
    ("value", lambda a: a["value"][:2]),
    ("k_cache", lambda a: a["k_cache"].view(torch.uint8)),
    ("k_cache", lambda a: torch.zeros(4, 2, 16, 64)),
    ("v_cache", lambda a: a["v_cache"][:3]),
    ("v_cache", lambda a: torch.zeros(8, 2, 16, 64, dtype=torch.uint8).view(E4M3)[::2]),
    ("kv_scales", lambda a: a["kv_scales"].double()),
    ("kv_scales", lambda a: a["kv_scales"][:, :1]),
    ("kv_scales", lambda a: torch.zeros(4, 2, 4)[..., ::2]),
    ("slot_mapping", lambda a: a["slot_mapping"].int()),
    ("slot_mapping", lambda a: a["slot_mapping"][:2]),
])
def test_append_refuses(name, make):
    from vflorence_amd import hip_attn

    args = _append_args()
    args[name] = make(args)
    with pytest.raises(ValueError):
        hip_attn.reshape_and_cache_8bit(**args)


def _attend_args():
    from vflorence_amd import hip_attn

    k, v, s = hip_attn.kv_cache_8bit(4, 2, 16, 64, "cpu")
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    return dict(query=q, k_cache=k, v_cache=v, kv_scales=s, out=torch.empty_like(q),
                seq_lens=torch.zeros(3, dtype=torch.int32), scale=0.125,
                block_table=torch.zeros(3, 2, dtype=torch.int32))


@pytest.mark.parametrize("name,make", [
    ("query", lambda a: a["query"][:, :1]),
    ("query", lambda a: a["query"][0]),
    ("query", lambda a: a["query"].double()),
    ("query", lambda a: a["query"].transpose(1, 2).contiguous().transpose(1, 2)),
    ("out", lambda a: a["out"].float()),
    ("out", lambda a: a["out"][:2]),
    ("out", lambda a: torch.zeros(3, 2, 128, dtype=torch.bfloat16)[..., ::2]),
    ("k_cache", lambda a: a["k_cache"].view(torch.int8)),
    ("kv_scales", lambda a: a["kv_scales"][..., 0]),
    ("seq_lens", lambda a: a["seq_lens"].long()),
    ("seq_lens", lambda a: a["seq_lens"][:2]),
    ("block_table", lambda a: a["block_table"].long()),
    ("block_table", lambda a: a["block_table"][:2]),
    ("block_table", lambda a: a["block_table"][0]),
])
def test_attention_refuses(name, make):
    from vflorence_amd import hip_attn

    args = _attend_args()
    args[name] = make(args)
    with pytest.raises(ValueError):
        hip_attn.attention_with_kv_cache_8bit(**args)


def test_cpu_tensors_have_no_path():
    from vflorence_amd import decoder_ops, hip_attn

    with pytest.raises(RuntimeError, match="no CPU path"):
        hip_attn.reshape_and_cache_8bit(**_append_args())
    with pytest.raises(RuntimeError, match="no CPU path"):
        hip_attn.attention_with_kv_cache_8bit(**_attend_args())
    with pytest.raises(RuntimeError, match="no CPU path"):
        decoder_ops.token_logprobs(torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("logits,tokens,k", [
    (torch.zeros(2, 3, 9), torch.zeros(2, dtype=torch.int64), 0),
    (torch.zeros(9, 2).t(), torch.zeros(2, dtype=torch.int64), 0),
    (torch.zeros(2, 9, dtype=torch.float64), torch.zeros(2, dtype=torch.int64), 0),
    (torch.zeros(2, 9), torch.zeros(2, dtype=torch.int32), 0),
    (torch.zeros(2, 9), torch.zeros(3, dtype=torch.int64), 0),
    (torch.zeros(2, 9), torch.zeros(2, 1, 1, dtype=torch.int64), 0),
    (torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64), 10),
    (torch.zeros(2, 90), torch.zeros(2, dtype=torch.int64), 21),
    (torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64), -1),
])
def test_token_logprobs_refuses(logits, tokens, k):
    from vflorence_amd import decoder_ops

    with pytest.raises(ValueError):
        decoder_ops.token_logprobs(logits, tokens, k)


def test_c_entries_check_before_launch():
    from vflorence_amd._lib import lib

    def append(key=A, kc=A, vc=A, sc=A, slots=A, tokens=4, heads=2, dim=64, bs=16, nb=10, dt=1):
        return lib.vfl_reshape_and_cache_8bit(key, A, 128, 64, 128, 64, kc, vc, sc, slots, tokens,
                                              heads, dim, bs, nb, dt, None)

    assert append(tokens=0) == 0 and append(nb=0) == 0  # nothing to do, nothing read
    assert append(dt=3) == -1 and b"dtype" in lib.vfl_last_error()
    assert append(dim=72) == -2 and append(bs=24) == -2 and append(bs=8) == -2
    assert append(tokens=-1) == -1 and append(tokens=1 << 31) == -1
    assert append(tokens=1 << 30, heads=64) == -1 and append(nb=1 << 31) == -1
    assert append(tokens=1 << 29, heads=3, dim=512) == -1  # more threads than a launch takes
    assert append(heads=0) == -1 and append(heads=65536) == -1 and append(nb=-1) == -1
    for bad in (dict(key=None), dict(kc=None), dict(vc=None), dict(sc=None), dict(slots=None)):
        assert append(**bad) == -1 and b"null" in lib.vfl_last_error()
    for bad in (dict(kc=A + 8), dict(vc=A + 4), dict(sc=A + 2), dict(slots=A + 4),
                dict(key=A + 1)):
        assert append(**bad) == -1 and b"misaligned" in lib.vfl_last_error()

    def attend(q=A, kc=A, vc=A, sc=A, out=A, lens=A, bt=A, stride=8, width=8, starts=None, rows=4,
               groups=4, heads=2, dim=64, bs=16, nb=10, dt=1, ws=None, scale=0.125):
        return lib.vfl_attention_with_kv_cache_8bit(q, 128, 64, kc, vc, sc, out, lens, bt, stride,
                                                    width, starts, None, rows, groups, heads, dim,
                                                    bs, nb, scale, dt, ws, None)

    assert attend(rows=0, groups=0) == 0 and attend(groups=0, starts=A) == 0
    assert attend(dt=3) == -1 and attend(dim=72) == -2 and attend(bs=48) == -2
    assert attend(rows=-1) == -1 and attend(groups=5) == -1 and attend(groups=3) == -1
    assert attend(width=-1) == -1 and attend(stride=7) == -1
    assert attend(width=1 << 28, stride=1 << 28) == -1  # more tokens than an int counts
    assert attend(rows=1 << 30, groups=1 << 30) == -1  # more threads than a launch takes
    assert attend(scale=float("nan")) == -1 and attend(scale=float("inf")) == -1
    for bad in (dict(q=None), dict(kc=None), dict(vc=None), dict(sc=None), dict(out=None),
                dict(lens=None), dict(bt=None)):
        assert attend(**bad) == -1 and b"null" in lib.vfl_last_error()
    for bad in (dict(kc=A + 8), dict(vc=A + 8), dict(sc=A + 4), dict(q=A + 1), dict(out=A + 1),
                dict(ws=A + 4)):
        assert attend(**bad) == -1 and b"misaligned" in lib.vfl_last_error()
    # few rows over a long table need a workspace, many or short ones none
    assert attend(width=4096, stride=4096) == -1 and b"workspace" in lib.vfl_last_error()
    assert lib.vfl_attention_8bit_workspace(4, 4, 2, 64, 16, 4096) > 0
    assert lib.vfl_attention_8bit_workspace(4, 4, 2, 64, 16, 64) == 0
    assert lib.vfl_attention_8bit_workspace(4096, 4096, 16, 64, 16, 4096) == 0
    assert lib.vfl_attention_8bit_workspace(0, 0, 2, 64, 16, 64) == 0

    def score(x=A, stride=100, rows=4, vocab=100, dt=1, tokens=A, n=1, k=0, lp=A, ent=A, top=A,
              ids=A, ws=None):
        return lib.vfl_token_logprobs(x, stride, rows, vocab, dt, tokens, n, k, lp, ent, top, ids,
                                      ws, None)

    assert score(rows=0) == 0
    assert score(dt=5) == -1 and score(vocab=0) == -1 and score(stride=99) == -1
    assert score(k=-1) == -1 and score(k=21) == -1 and score(vocab=5, k=6) == -1
    assert score(rows=-1) == -1 and score(n=-1) == -1 and score(rows=1 << 22) == -1
    assert score(x=None, stride=0) == -1  # (a stride of 0 is one row repeated)
    assert score(x=None) == -1 and score(ent=None) == -1 and score(tokens=None) == -1
    assert score(lp=None) == -1 and score(k=2, top=None) == -1 and score(k=2, ids=None) == -1
    assert score(x=A + 1) == -1
    assert score(vocab=(1 << 20) + 1, stride=1 << 21) == -1
    assert score(vocab=200000, stride=200000) == -1 and b"null" in lib.vfl_last_error()
    assert score(vocab=200000, stride=200000, ws=A + 8) == -1
    assert lib.vfl_token_logprobs_workspace(50265, 0, 20) == 0
    assert lib.vfl_token_logprobs_workspace(57344, 1, 20) == 0
    assert lib.vfl_token_logprobs_workspace(200000, 1, 20) == 4 * (16 + 8 * 20)


def test_oracle_append_rescales_a_growing_block():
    from vflorence_amd import hip_attn

    cache = Cache.of(*hip_attn.kv_cache_8bit(2, 1, 16, 32, "cpu"))
    one = torch.ones(1, 1, 32)
    cache.append(one, one, torch.tensor([16]))
    assert cache.scales[1, 0, 0] == 2.0**-8 and float(cache.values()[0][1, 0, 0, 0]) == 1.0
    cache.append(one * 1000, one, torch.tensor([17]))
    assert cache.scales[1, 0, 0] == 4.0 and float(cache.values()[0][1, 0, 0, 0]) == 1.0
    assert float(cache.values()[0][1, 0, 1, 0]) == 1024.0  # 250 lies between 240 and 256
