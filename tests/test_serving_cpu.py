"""What the serving calls refuse (nothing is launched: the tensors are on the CPU), the rotary tables, and the exported symbols."""
import ctypes
import math
import re
from fractions import Fraction
from pathlib import Path

import pytest
import torch

import risaattention_b200 as risa

ROOT = Path(__file__).resolve().parents[1]
BF16 = torch.bfloat16


def test_library_exports_every_declared_symbol():
    declared = set(re.findall(r"\b(risa_b200_\w+)\s*\(", (ROOT / "include" / "risa_b200_cache.h").read_text()))
    declared -= {"risa_b200_last_error", "risa_b200_device_status"}
    assert len(declared) >= 7
    lib = ctypes.CDLL(str(ROOT / "risaattention_b200" / "librisa_b200.so"))
    for name in sorted(declared):
        assert hasattr(lib, name), name


def test_frequencies():
    assert risa.rotary_frequencies(8, base=10000.0) == [10000.0 ** (-i / 4) for i in range(4)]
    assert risa.rotary_frequencies(8, scaling="linear", factor=4.0) == [f / 4 for f in risa.rotary_frequencies(8)]
    based, plain = risa.rotary_frequencies(8, scaling="base", factor=4.0), risa.rotary_frequencies(8)
    assert based[0] == plain[0] and based[-1] == pytest.approx(plain[-1] / 4, rel=1e-12)
    parts = risa.rotary_frequencies(64, scaling="parts", factor=4.0, original_length=4096, slow_turns=1.0, fast_turns=32.0)
    plain = risa.rotary_frequencies(64)
    for f, p in zip(parts, plain):
        turns = 4096 * p / (2 * math.pi)
        assert f == p if turns >= 32 else f == p / 4 if turns <= 1 else p / 4 < f < p


def test_table_holds_turns():
    table = risa.rotary_table(16, device="cpu")
    assert table.rotary_dim == 16 and table.turns.dtype == torch.int64
    for unit, f in zip(table.turns.tolist(), risa.rotary_frequencies(16)):
        # the double f / 2 pi is off by 2^-52 of itself
        assert abs(Fraction(unit % 2 ** 64, 2 ** 64) - Fraction(f / (2 * math.pi))) <= Fraction(1, 2 ** 60)


@pytest.mark.parametrize("arguments,error", [
    (dict(rotary_dim=7), ValueError), (dict(rotary_dim=0), ValueError), (dict(rotary_dim=8, base=1.0), ValueError), (dict(rotary_dim=8, scaling="other"), ValueError),
    (dict(rotary_dim=8, factor=0.0), ValueError), (dict(rotary_dim=8, factor=math.nan), ValueError), (dict(rotary_dim=8, scaling="parts"), ValueError),
    (dict(rotary_dim=8, scaling="parts", original_length=9, slow_turns=2.0, fast_turns=2.0), ValueError), (dict(rotary_dim=8, magnitude=math.inf), ValueError)])
def test_table_refusals(arguments, error):
    with pytest.raises(error):
        risa.rotary_table(**arguments, device="cpu")


def x(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_rotation_refusals():
    table = risa.rotary_table(8, device="cpu")
    rotate = risa.rotate_positions
    with pytest.raises(TypeError, match="RotaryTable"):
        rotate(x(2, 3, 8), ints(2), table.turns)
    for args, error in [((x(2, 8), ints(2)), ValueError), ((x(2, 3, 8), ints(3)), ValueError), ((x(2, 3, 8), ints(1, 2)), ValueError),
                        ((x(2, 3, 5, 8), ints(3, 5)), ValueError), ((x(0, 3, 8), ints(0)), ValueError), ((x(2, 3, 6), ints(2)), ValueError),
                        ((x(2, 3, 8, dtype=torch.float64), ints(2)), TypeError), ((x(2, 3, 8), ints(2).float()), TypeError),
                        ((x(2, 3, 16)[..., ::2], ints(2)), ValueError)]:
        with pytest.raises(error):
            rotate(*args, table)
    with pytest.raises(ValueError, match="out"):
        rotate(x(2, 3, 8), ints(2), table, out=x(2, 3, 9))
    with pytest.raises(TypeError, match="out"):
        rotate(x(2, 3, 8), ints(2), table, out=x(2, 3, 8, dtype=torch.float16))
    with pytest.raises(ValueError, match="expanded"):
        rotate(x(2, 3, 8), ints(2), table, out=x(2, 1, 8).expand(2, 3, 8))
    with pytest.raises(ValueError, match="gradient"):
        rotate(x(2, 3, 8, dtype=torch.float32).requires_grad_(), ints(2), table, out=x(2, 3, 8, dtype=torch.float32))
    with pytest.raises(ValueError, match="CUDA device"):
        rotate(x(2, 3, 8), ints(2), table)


def test_cache_refusals():
    make = risa.KeyValueCache
    for args, error in [((x(2, 1, 16, 64), x(2, 1, 16, 128)), ValueError), ((x(2, 16, 64), x(2, 16, 64)), ValueError), ((x(2, 1, 24, 64),) * 2, ValueError),
                        ((x(2, 1, 16, 80),) * 2, ValueError), ((x(0, 1, 16, 64),) * 2, ValueError), ((x(2, 1, 16, 64, dtype=torch.float32),) * 2, TypeError),
                        ((x(2, 1, 16, 64), x(2, 1, 16, 64, dtype=torch.float16)), TypeError), ((x(2, 16, 1, 64).transpose(1, 2),) * 2, None),
                        ((x(2, 16, 3, 64).transpose(1, 2),) * 2, ValueError), ((x(2, 1, 16, 64, dtype=torch.int8),) * 2, ValueError),
                        ((x(2, 1, 16, 64),) * 2 + (x(2, 1, 16, dtype=torch.float32),) * 2, ValueError),
                        ((x(2, 1, 16, 64, dtype=torch.int8),) * 2 + (x(2, 1, 16),) * 2, TypeError),
                        ((x(2, 1, 16, 64, dtype=torch.int8),) * 2 + (x(2, 1, 15, dtype=torch.float32),) * 2, ValueError)]:
        if error is None:
            make(*args)
            continue
        with pytest.raises(error):
            make(*args)
    cache = risa.allocate_key_value_cache(3, 2, 32, 64, dtype=torch.int8, device="cpu")
    assert cache.quantized and cache.page_size == 32 and cache.key_scales.shape == (3, 2, 32)


@pytest.fixture
def cache():
    return risa.allocate_key_value_cache(4, 2, 16, 64, device="cpu")


def refuses(error, call, *args, match=None, **kwargs):
    with pytest.raises(error, match=match):
        call(*args, **kwargs)


def test_step_refusals(cache):
    attend = risa.paged_attention
    q = x(3, 4, 64)
    good = (ints(3, 2), ints(3))
    refuses(ValueError, attend, q, cache, ints(3), ints(3), match="page_table")
    refuses(ValueError, attend, q, cache, ints(3, 0), ints(3), match="page_table")
    refuses(ValueError, attend, q, cache, ints(3, 2), ints(2), match="lengths")
    refuses(ValueError, attend, q, cache, ints(2, 2), ints(2), match="one token")
    refuses(ValueError, attend, q, cache, *good, query_offsets=ints(3), match="query_offsets")
    refuses(TypeError, attend, q, cache, ints(3, 2).long(), ints(3), match="int32")
    refuses(TypeError, attend, q, cache, ints(3, 2), ints(3).long(), match="int32")
    refuses(ValueError, attend, q, cache, ints(3, 4)[:, ::2], ints(3), match="contiguous")
    refuses(ValueError, attend, x(0, 4, 64), cache, *good, query_offsets=ints(4), match="tokens")
    refuses(ValueError, attend, q, cache, *good, match="CUDA device")


def test_attention_refusals(cache):
    attend = risa.paged_attention
    step = (ints(3, 2), ints(3))
    refuses(TypeError, attend, x(3, 4, 64), cache.keys, *step, match="KeyValueCache")
    refuses(ValueError, attend, x(3, 64), cache, *step, match="q must have shape")
    refuses(ValueError, attend, x(3, 4, 128), cache, *step, match="q must have shape")
    refuses(ValueError, attend, x(3, 3, 64), cache, *step, match="divisible")
    refuses(TypeError, attend, x(3, 4, 64, dtype=torch.float32), cache, *step, match="float16 or bfloat16")
    refuses(TypeError, attend, x(3, 4, 64, dtype=torch.float16), cache, *step, match="dtype of the cache")
    refuses(ValueError, attend, x(3, 4, 64), cache, *step, window=0, match="window")
    refuses(ValueError, attend, x(3, 4, 64), cache, *step, window=4, is_causal=False, match="causal")
    refuses(ValueError, attend, x(3, 4, 64), cache, *step, out=x(3, 4, 32), match="out")
    refuses(TypeError, attend, x(3, 4, 64), cache, *step, out=x(3, 4, 64, dtype=torch.float16), match="out")
    refuses(ValueError, attend, x(3, 4, 64), cache, *step, out=x(3, 4, 65)[..., 1:], match="out")
    refuses(ValueError, attend, x(3, 4, 64), cache, *step, out=x(1, 4, 64).expand(3, 4, 64), match="expanded")


def test_outputs_that_overlap_their_input(cache):
    memory, table = x(5, 4, 64), risa.rotary_table(64, device="cpu")
    for out in (memory[1:4], memory[:3].view(4, 3, 64).transpose(0, 1)):
        refuses(ValueError, risa.rotate_positions, memory[:3], ints(3), table, out=out, match="another view")
        refuses(ValueError, risa.paged_attention, memory[:3], cache, ints(3, 2), ints(3), out=out, match="another view")
    for out in (memory[:3], x(3, 4, 64)):
        refuses(ValueError, risa.rotate_positions, memory[:3], ints(3), table, out=out, match="CUDA device")
        refuses(ValueError, risa.paged_attention, memory[:3], cache, ints(3, 2), ints(3), out=out, match="CUDA device")


def test_more_query_rows_than_31_bits(cache):
    q, step = x(1, 1, 64).expand(2 ** 17, 2 ** 15, 64), (ints(1, 2), ints(1))
    refuses(ValueError, risa.paged_attention, q, cache, *step, query_offsets=ints(2), match="too many rows")
    lse = x(1, 1, dtype=torch.float32).expand(2 ** 17, 2 ** 15)
    refuses(ValueError, risa.cached_key_weights, q, lse, cache, *step, query_offsets=ints(2), match="too many rows")


def test_append_refusals(cache):
    append = risa.append_to_cache
    k, step = x(3, 2, 64), (ints(3, 2), ints(3))
    table = risa.rotary_table(64, device="cpu")
    refuses(ValueError, append, cache, x(3, 4, 64), x(3, 4, 64), *step, match="k and v")
    refuses(ValueError, append, cache, k, x(3, 2, 32), *step, match="k and v")
    refuses(TypeError, append, cache, k.half(), k.half(), *step, match="dtype of the cache")
    refuses(TypeError, append, cache, k, k.half(), *step, match="same dtype")
    refuses(ValueError, append, cache, k, k, *step, q=x(3, 4, 64), match="rotary")
    refuses(ValueError, append, cache, k, k, *step, q=x(2, 4, 64), rotary=table, match="q must have shape")
    refuses(ValueError, append, cache, k, k, *step, positions=ints(3), match="rotary")
    refuses(ValueError, append, cache, k, k, *step, rotary=table, positions=ints(2), match="positions")
    refuses(TypeError, append, cache, k, k, *step, rotary=table, positions=ints(3).float(), match="positions")
    refuses(ValueError, append, cache, k, k, *step, rotary=risa.rotary_table(24, device="cpu"), match="multiple of 16")
    refuses(ValueError, append, cache, k, k, *step, rotary=risa.rotary_table(128, device="cpu"), match="rotary_dim")
    refuses(TypeError, append, cache, k, k, *step, rotary=table.turns, match="RotaryTable")
    refuses(ValueError, append, cache, k, k, *step, rotary=table, match="CUDA device")


def test_weight_and_eviction_refusals(cache):
    weigh, evict = risa.cached_key_weights, risa.evict_from_cache
    q, lse, step = x(3, 4, 64), x(3, 4, dtype=torch.float32), (ints(3, 2), ints(3))
    refuses(ValueError, weigh, q, lse[:2], cache, *step, match="lse")
    refuses(TypeError, weigh, q, lse.half(), cache, *step, match="lse")
    refuses(ValueError, weigh, q, lse, cache, *step, previous=x(3, 2, 16, dtype=torch.float32), match="previous")
    refuses(TypeError, weigh, q, lse, cache, *step, previous=x(3, 2, 32), match="previous")
    refuses(ValueError, weigh, q, lse, cache, *step, match="CUDA device")
    weights, target = x(3, 2, 32, dtype=torch.float32), ints(3, 1)
    refuses(ValueError, evict, cache, *step, weights[..., :16], target, budget=8, match="weights")
    refuses(TypeError, evict, cache, *step, weights.half(), target, budget=8, match="weights")
    refuses(ValueError, evict, cache, *step, weights, ints(2, 1), budget=8, match="target_table")
    refuses(TypeError, evict, cache, *step, weights, target.long(), budget=8, match="int32")
    refuses(ValueError, evict, cache, *step, weights, target, budget=0, match="budget")
    refuses(ValueError, evict, cache, *step, weights, target, budget=8, recent=9, match="recent")
    refuses(ValueError, evict, cache, *step, weights, target, budget=8, recent=-1, match="recent")
    refuses(ValueError, evict, cache, *step, weights, target, budget=17, match="hold the budget")
    refuses(ValueError, evict, cache, *step, weights, step[0], budget=8, match="other pages")
    refuses(ValueError, evict, cache, *step, weights, target, budget=8, match="CUDA device")


def test_rotation_refuses_forward_mode():
    """A dual tensor need not require a gradient; its tangent must not be lost on the way."""
    table = risa.rotary_table(8, device="cpu")
    for grad in (False, True):
        with torch.autograd.forward_ad.dual_level():
            dual = torch.autograd.forward_ad.make_dual(x(2, 3, 8, dtype=torch.float32).requires_grad_(grad), torch.ones(2, 3, 8))
            refuses(ValueError, risa.rotate_positions, dual, ints(2), table, match="forward-mode")
            with torch.no_grad():
                refuses(ValueError, risa.rotate_positions, dual, ints(2), table, match="forward-mode")
    # the same tensor without a tangent goes on to the next check
    refuses(ValueError, risa.rotate_positions, x(2, 3, 8), ints(2), table, match="CUDA device")


def test_tables_that_lead_past_31_bits():
    """Kernels count a sequence's keys in 32 bits, and step past the last one."""
    cache = risa.allocate_key_value_cache(1, 1, 128, 64, device="cpu")
    wide, most = ints(1, 2 ** 24 - 3), 2 ** 24 - 65  # pages of 128 keys: 2^31 - 384 keys, and as many as there may be
    q, lse, few = x(1, 1, 64), x(1, 1, dtype=torch.float32), ints(1, 1)
    weights = x(1, 1, 1, dtype=torch.float32)
    for call, args in ((risa.paged_attention, (q, cache)), (risa.cached_key_weights, (q, lse, cache)), (risa.append_to_cache, (cache, q, q))):
        refuses(ValueError, call, *args, wide, ints(1), match="2\\^31 - 8192")
        refuses(ValueError, call, *args, wide[:, :most], ints(1), match="CUDA device")
    refuses(ValueError, risa.evict_from_cache, cache, wide, ints(1), weights, few, budget=8, match="2\\^31 - 8192")
    refuses(ValueError, risa.evict_from_cache, cache, few, ints(1), x(1, 1, 128, dtype=torch.float32), wide, budget=8, match="2\\^31 - 8192")
    refuses(ValueError, risa.evict_from_cache, cache, few, ints(1), x(1, 1, 128, dtype=torch.float32), wide[:, :most], budget=8, match="CUDA device")


def test_c_entries_check_heads_and_scale():
    """What the module's own checks let through or never produce; nothing is read: the addresses are aligned numbers."""
    lib = ctypes.CDLL(str(ROOT / "risaattention_b200" / "librisa_b200.so"))
    lib.risa_b200_last_error.restype = ctypes.c_char_p

    class Cache(ctypes.Structure):
        _fields_ = [(n, ctypes.c_void_p) for n in ("keys", "values", "key_scales", "value_scales")] + [(n, ctypes.c_int) for n in ("pages", "kv_heads", "page_size", "head_dim", "dtype_code")]

    class Step(ctypes.Structure):
        _fields_ = [(n, ctypes.c_void_p) for n in ("page_table", "lengths", "query_offsets")] + [(n, ctypes.c_int) for n in ("batch", "table_width", "tokens")]

    class Rotary(ctypes.Structure):
        _fields_ = [("turns", ctypes.c_void_p), ("rotary_dim", ctypes.c_int), ("magnitude", ctypes.c_float), ("interleaved", ctypes.c_int)]

    at, strides = ctypes.c_void_p(4096), (ctypes.c_int64 * 2)(512, 128)
    cache, step, rotary = Cache(4096, 4096, None, None, 8, 2, 16, 128, 2), Step(4096, 4096, None, 1, 8, 1), Rotary(4096, 128, 1.0, 0)
    invalid = int(re.search(r"RISA_B200_INVALID (\d+)", (ROOT / "include" / "risa_b200.h").read_text())[1])
    for heads in (0, -4):
        assert lib.risa_b200_cache_append(ctypes.byref(cache), ctypes.byref(step), at, strides, at, strides, at, strides, at, strides, heads, 2, ctypes.byref(rotary), None, 0, None) == invalid
        assert b"heads" in lib.risa_b200_last_error()
    for scale in (3e38, math.inf, math.nan):  # 3e38 is finite, and in units of log 2 it is not
        assert lib.risa_b200_paged_attention(ctypes.byref(cache), ctypes.byref(step), at, strides, 4, 2, at, strides, at, ctypes.c_float(scale), 1, 0, 3, at, ctypes.c_size_t(1 << 30), None) == invalid
        assert b"scale" in lib.risa_b200_last_error()
        assert lib.risa_b200_key_weights(ctypes.byref(cache), ctypes.byref(step), at, strides, 4, 2, at, ctypes.c_float(scale), 1, 0, None, at, at, ctypes.c_size_t(1 << 30), None) == invalid
