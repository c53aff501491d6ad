"""The 4-bit cache's operators and packed cross-attention refuse bad calls on the host, before
anything is launched; their helpers work on the CPU."""

import math

import pytest
import torch

from tests.cache_4bit_oracle import SIZES, nearest_e2m1, needed_scale, quantised

A = 16 * 1000  # a 16-byte aligned stand-in address (never dereferenced)


def place(heads, bs, dim, h, t, d, value):
    """(byte, high half, scale byte) of token t's dim d in a block, as the format says."""
    groups, parts = -(-dim // 32), bs // 16
    tile = ((h * parts + t // 16) * groups + d // 32) * 256
    half = heads * parts * groups * 256
    scale = (2 * half + (h * parts + t // 16) * 32 * groups + t % 16 // 4 * 8 * groups
             + (4 * groups if value else 0) + d // 32 * 4 + t % 4)
    if value:
        return half + tile + d % 16 * 16 + t % 16, d % 32 >= 16, scale
    return tile + t % 16 * 16 + d % 32 // 2, d % 2 == 1, scale


@pytest.mark.parametrize("heads,bs,dim", [(2, 16, 64), (1, 32, 48), (3, 16, 96), (1, 32, 512)])
def test_values_follow_the_format(heads, bs, dim):
    from vflorence_amd import hip_attn

    gen = torch.Generator().manual_seed(dim)
    cache = hip_attn.kv_cache_4bit(3, heads, bs, dim, "cpu")
    groups = -(-dim // 32)
    assert cache.dtype == torch.uint8 and cache.shape == (3, heads, bs, 34 * groups)
    assert not cache.any()
    cache.copy_(torch.randint(0, 256, cache.shape, generator=gen))
    scales = cache.view(3, -1)[:, heads * bs * groups * 32:]
    scales.copy_(torch.randint(27, 253, scales.shape, generator=gen))
    scales[1, 5] = 255
    got = hip_attn.kv_cache_4bit_values(cache, dim)
    stands = list(SIZES) + [-x for x in SIZES]
    flat = cache.view(3, -1).tolist()
    for value, x in enumerate(got):
        assert x.shape == (3, heads, bs, dim) and x.dtype == torch.float32
        x = x.tolist()
        for b in range(3):
            for h in range(heads):
                for t in range(0, bs, 3):
                    for d in range(0, dim, 5):
                        byte, high, scale = place(heads, bs, dim, h, t, d, value)
                        code = flat[b][byte] >> 4 if high else flat[b][byte] & 15
                        if flat[b][scale] == 255:
                            assert math.isnan(x[b][h][t][d])
                        else:
                            assert x[b][h][t][d] == stands[code] * 2.0 ** (flat[b][scale] - 127)
    for bad in ((3, 2, 24, 64), (3, 2, 16, 72)):
        with pytest.raises(ValueError):
            hip_attn.kv_cache_4bit(*bad, "cpu")
    for cache, dim in ((cache[..., :-1], dim), (cache.int(), dim), (cache, 40), (cache[0], dim)):
        with pytest.raises(ValueError):
            hip_attn.kv_cache_4bit_values(cache, dim)


def test_oracle_rounds_as_the_type():
    every = torch.tensor(list(SIZES) + [-x for x in SIZES], dtype=torch.float64)
    x = torch.cat([torch.linspace(-7, 7, 2801, dtype=torch.float64), every])
    order = (x[:, None] - every[None, :8].abs() * torch.sign(x)[:, None]).abs()
    least = order.min(dim=1)
    assert torch.equal((nearest_e2m1(x) - x).abs(), least.values)
    for tie, even in ((0.25, 0.0), (0.75, 1.0), (1.25, 1.0), (1.75, 2.0), (2.5, 2.0), (3.5, 4.0),
                      (5.0, 4.0), (7.0, 6.0), (100.0, 6.0)):
        both = nearest_e2m1(torch.tensor([tie, -tie], dtype=torch.float64))
        assert both.tolist() == [even, -even]
    for value, scale in ((6.0, 1.0), (6.01, 2.0), (0.0, 2.0**-100), (3.0, 0.5), (4.0, 1.0),
                         (2.0**-120, 2.0**-100), (3.4e38, 2.0**125)):
        group = torch.tensor([value, -value / 3] + [0.0] * 30, dtype=torch.float64)
        assert needed_scale(group) == scale
        assert torch.equal(quantised(group), nearest_e2m1(group / scale) * scale)


def _rows(dtype=torch.bfloat16, dim=64):
    from vflorence_amd import hip_attn

    x = torch.zeros(3, 2, dim, dtype=dtype)
    return dict(key=x, value=x.clone(), cache=hip_attn.kv_cache_4bit(4, 2, 16, dim, "cpu"),
                slot_mapping=torch.zeros(3, dtype=torch.int64))


ROWS = [
    ("key", lambda a: a["key"][:, :, :32]),
    ("key", lambda a: a["key"][:, :1]),
    ("key", lambda a: a["key"][0]),
    ("key", lambda a: a["key"].to(torch.float16)),
    ("key", lambda a: a["key"].to(torch.float64)),
    ("value", lambda a: a["value"].transpose(1, 2).contiguous().transpose(1, 2)),
    ("value", lambda a: a["value"][:2]),
    ("cache", lambda a: a["cache"].view(torch.int8)),
    ("cache", lambda a: a["cache"][:, :1]),
    ("cache", lambda a: a["cache"][..., :34]),
    ("cache", lambda a: torch.zeros(4, 2, 24, 68, dtype=torch.uint8)),
    ("slot_mapping", lambda a: a["slot_mapping"].int()),
    ("slot_mapping", lambda a: a["slot_mapping"][:2]),
]


@pytest.mark.parametrize("name,make", ROWS)
@pytest.mark.parametrize("call", ["reshape_and_cache_4bit", "gather_cache_4bit"])
def test_rows_refused(call, name, make):
    from vflorence_amd import hip_attn

    args = _rows()
    args[name] = make(args)
    with pytest.raises(ValueError):
        getattr(hip_attn, call)(**args)


def _attend_args():
    from vflorence_amd import hip_attn

    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    return dict(query=q, cache=hip_attn.kv_cache_4bit(4, 2, 16, 64, "cpu"),
                out=torch.empty_like(q), seq_lens=torch.zeros(3, dtype=torch.int32), scale=0.125,
                block_table=torch.zeros(3, 2, dtype=torch.int32))


@pytest.mark.parametrize("name,make", [
    ("query", lambda a: a["query"][:, :1]),
    ("query", lambda a: a["query"][0]),
    ("query", lambda a: a["query"].double()),
    ("query", lambda a: a["query"].transpose(1, 2).contiguous().transpose(1, 2)),
    ("out", lambda a: a["out"].float()),
    ("out", lambda a: a["out"][:2]),
    ("out", lambda a: torch.zeros(3, 2, 128, dtype=torch.bfloat16)[..., ::2]),
    ("cache", lambda a: a["cache"].view(torch.int8)),
    ("cache", lambda a: a["cache"][..., :34]),
    ("seq_lens", lambda a: a["seq_lens"].long()),
    ("seq_lens", lambda a: a["seq_lens"][:2]),
    ("block_table", lambda a: a["block_table"].long()),
    ("block_table", lambda a: a["block_table"][:2]),
    ("block_table", lambda a: a["block_table"][0]),
])
def test_attention_refused(name, make):
    from vflorence_amd import hip_attn

    args = _attend_args()
    args[name] = make(args)
    with pytest.raises(ValueError):
        hip_attn.attention_with_kv_cache_4bit(**args)


def _cross_args():
    q, k = torch.zeros(5, 2, 64, dtype=torch.float16), torch.zeros(7, 2, 64, dtype=torch.float16)
    return dict(query=q, key=k, value=k.clone(), out=torch.empty_like(q),
                query_start_loc=torch.tensor([0, 2, 5], dtype=torch.int32),
                key_start_loc=torch.tensor([0, 3, 7], dtype=torch.int32), scale=0.125,
                max_query_len=3, max_key_len=4)


@pytest.mark.parametrize("name,make", [
    ("query", lambda a: a["query"][:, :1]),
    ("query", lambda a: a["query"][0]),
    ("query", lambda a: a["query"].bfloat16()),
    ("key", lambda a: a["key"][..., :32]),
    ("key", lambda a: a["key"][:6]),
    ("key", lambda a: a["key"].transpose(1, 2).contiguous().transpose(1, 2)),
    ("value", lambda a: a["value"].float()),
    ("out", lambda a: a["out"][:4]),
    ("out", lambda a: a["out"].float()),
    ("out", lambda a: torch.zeros(5, 2, 128, dtype=torch.float16)[..., ::2]),
    ("query_start_loc", lambda a: a["query_start_loc"].long()),
    ("query_start_loc", lambda a: a["query_start_loc"][:2]),
    ("key_start_loc", lambda a: a["key_start_loc"][:, None]),
    ("max_query_len", lambda a: -1),
    ("max_key_len", lambda a: -1),
])
def test_cross_refused(name, make):
    from vflorence_amd import hip_attn

    args = _cross_args()
    args[name] = make(args)
    with pytest.raises(ValueError):
        hip_attn.packed_cross_attention(**args)


def test_cross_head_sizes():
    from vflorence_amd import hip_attn

    for dim in (512, 72):
        args = _cross_args()
        for name in ("query", "key", "value", "out"):
            args[name] = args[name].new_zeros(args[name].shape[0], 2, dim)
        with pytest.raises(ValueError):
            hip_attn.packed_cross_attention(**args)
    with pytest.raises(TypeError):
        hip_attn.packed_cross_attention(**dict(_cross_args(), max_query_len=2.5))


def test_cpu_tensors_have_no_path():
    from vflorence_amd import hip_attn

    for call, args in (("reshape_and_cache_4bit", _rows()), ("gather_cache_4bit", _rows()),
                       ("attention_with_kv_cache_4bit", _attend_args()),
                       ("packed_cross_attention", _cross_args())):
        with pytest.raises(RuntimeError, match="no CPU path"):
            getattr(hip_attn, call)(**args)


def _message():
    from vflorence_amd._lib import lib

    return lib.vfl_last_error().decode()


def test_c_entries_refuse():
    from vflorence_amd._lib import VFL_BFLOAT16, VFL_FLOAT32, lib

    def store(call=lib.vfl_reshape_and_cache_4bit, key=A, cache=A, slots=A, tokens=4, heads=2,
              dim=64, block=16, blocks=8, dtype=VFL_BFLOAT16):
        if call is lib.vfl_gather_cache_4bit:
            return call(cache, slots, key, A, 128, 64, 128, 64, tokens, heads, dim, block, blocks,
                        dtype, None)
        return call(key, A, 128, 64, 128, 64, cache, slots, tokens, heads, dim, block, blocks,
                    dtype, None)

    for call in (lib.vfl_reshape_and_cache_4bit, lib.vfl_gather_cache_4bit):
        for bad in (dict(key=None), dict(cache=None), dict(slots=None), dict(cache=A + 8),
                    dict(slots=A + 4), dict(key=A + 1), dict(tokens=-1), dict(heads=0),
                    dict(dim=40), dict(block=24), dict(blocks=-1), dict(dtype=7),
                    dict(tokens=1 << 31), dict(tokens=1 << 30, heads=4096)):
            assert store(call, **bad) != 0 and _message(), bad
        assert store(call, tokens=0, key=None) == 0

    def attend(q=A, cache=A, out=A, lens=A, table=A, stride=4, width=4, rows=3, groups=3, most=1,
               heads=2, dim=64, block=16, blocks=8, scale=0.125, dtype=VFL_BFLOAT16, work=None,
               start=None):
        return lib.vfl_attention_with_kv_cache_4bit(
            q, 128, 64, cache, out, lens, table, stride, width, start, None, rows, groups, most,
            heads, dim, block, blocks, scale, dtype, work, None)

    for bad in (dict(q=None), dict(cache=None), dict(out=None), dict(lens=None),
                dict(table=None), dict(stride=3), dict(width=1 << 30, stride=1 << 30),
                dict(rows=-1), dict(groups=2), dict(groups=4), dict(most=0), dict(most=9),
                dict(heads=0), dict(dim=72), dict(block=8), dict(scale=float("inf")),
                dict(scale=float("nan")), dict(dtype=3), dict(cache=A + 4), dict(work=A + 8),
                dict(q=A + 1), dict(rows=1 << 30, groups=1 << 30, heads=65535),
                dict(rows=1, groups=1, heads=1, width=4096, stride=4096)):  # null workspace
        assert attend(**bad) != 0 and _message(), bad
    assert attend(rows=0, groups=0) == 0
    assert lib.vfl_attention_4bit_workspace(1, 1, 1, 64, 16, 4096) > 0
    assert lib.vfl_attention_4bit_workspace(256, 64, 16, 64, 16, 64) == 0
    # rows of no group take no more than a bounded workspace: four parts of 4096 rows x 16 heads of
    # 128 would be 4 * 2^16 * (128 * 4 + 8) = 136.3 MB, more than 2^27
    for rows in (1, 500, 2000, 4096, 1 << 20, 1 << 62):
        need = lib.vfl_attention_4bit_workspace(rows, 1, 16, 128, 16, 2500)
        assert (need > 0) == (rows <= 2000) and need <= 1 << 27

    def cross(q=A, k=A, v=A, out=A, starts=A, queries=5, keys=7, sequences=2, heads=2, dim=64,
              longest=(3, 4), scale=0.125, dtype=VFL_FLOAT32, work=None):
        return lib.vfl_packed_cross_attention(
            q, 128, 64, k, 128, 64, v, 128, 64, out, starts, A, queries, keys, sequences, heads,
            dim, *longest, scale, dtype, work, None)

    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(starts=None),
                dict(queries=-1), dict(keys=-1), dict(sequences=-1), dict(heads=0),
                dict(heads=65536), dict(dim=512), dict(dim=72), dict(longest=(-1, 4)),
                dict(longest=(3, -1)), dict(scale=float("nan")), dict(dtype=5), dict(q=A + 2),
                dict(work=A + 4), dict(queries=1 << 32), dict(sequences=1 << 30),
                dict(longest=(3, 100000))):  # null workspace
        assert cross(**bad) != 0 and _message(), bad
    assert cross(queries=0) == 0 and cross(sequences=0) == 0
    assert lib.vfl_packed_cross_attention_workspace(5, 2, 2, 64, 3, 100000, VFL_FLOAT32) > 0
    assert lib.vfl_packed_cross_attention_workspace(5, 2, 2, 64, 3, 4, VFL_FLOAT32) == 0
    assert cross(queries=(1 << 31) - 1) != 0 and cross(keys=(1 << 31) - 1) != 0
    # rows of no sequence take no more than a bounded workspace: two parts of 2^15 rows x 8 heads
    # would be 2 * 2^18 * (64 * 4 + 8) = 138.4 MB, more than 2^27
    for rows in (9, 1000, 1 << 15, 1 << 20, 1 << 31, 1 << 62):
        need = lib.vfl_packed_cross_attention_workspace(rows, 1, 8, 64, 9, 40000, VFL_BFLOAT16)
        assert (need > 0) == (rows < 1 << 15) and need <= 1 << 27


def test_entry_callables():
    """The extension module's callables convert as the entries' types ask, and reach the same
    library: its message is the one that the other binding reads."""
    from vflorence_amd._lib import VFL_BFLOAT16, calls, lib

    args = [A, A, 128, 64, 128, 64, A, A, 0, 2, 64, 16, 8, VFL_BFLOAT16, None]
    call = calls.vfl_reshape_and_cache_4bit
    assert call(*args) == 0
    assert call(*args[:10], 40, *args[11:]) == lib.vfl_reshape_and_cache_4bit(
        *args[:10], 40, *args[11:]) != 0
    lib.vfl_reshape_and_cache_4bit(*args)  # clears the message
    assert call(*args[:13], 9, None) != 0 and "dtype code 9" in _message()
    for bad, error in ((args[:-1], TypeError), (args + [0], TypeError),
                       (["x", *args[1:]], TypeError), ([-1, *args[1:]], OverflowError),
                       ([*args[:9], 1 << 31, *args[10:]], OverflowError),
                       ([*args[:2], 1 << 63, *args[3:]], OverflowError),
                       ([*args[:2], 1.5, *args[3:]], TypeError)):
        with pytest.raises(error):
            call(*bad)
    with pytest.raises(TypeError):
        calls.vfl_packed_cross_attention(*[A] * 19, "scale", 1, None, None)


def test_entries_without_the_extension_module(tmp_path):
    """A package that holds the library alone loads, and calls the same entries through it."""
    import os
    import shutil
    import subprocess
    import sys

    import vflorence_amd
    from vflorence_amd import _lib

    assert _lib._load_calls(str(tmp_path / "_calls.so")) is _lib.lib
    (tmp_path / "_calls.so").write_text("no shared object")
    assert _lib._load_calls(str(tmp_path / "_calls.so")) is _lib.lib
    here = os.path.dirname(vflorence_amd.__file__)
    shutil.copytree(here, tmp_path / "vflorence_amd",
                    ignore=lambda _, names: [n for n in names
                                             if n.startswith("_calls") or n in ("_build", "csrc")])
    code = ("from vflorence_amd import _lib, hip_attn\n"
            f"assert _lib.__file__.startswith({str(tmp_path)!r}), _lib.__file__\n"
            "assert hip_attn.calls is _lib.lib\n"
            f"args = [{A}, {A}, 128, 64, 128, 64, {A}, {A}, 0, 2, 64, 16, 8, 1, None]\n"
            "assert hip_attn.calls.vfl_reshape_and_cache_4bit(*args) == 0\n"
            "args[13] = 9\n"
            "assert hip_attn.calls.vfl_reshape_and_cache_4bit(*args) != 0\n")
    run = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, capture_output=True, text=True,
                         env=dict(os.environ, PYTHONPATH=str(tmp_path)))
    assert run.returncode == 0, run.stderr
