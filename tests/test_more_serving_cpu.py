"""What the serving calls refuse of positions with several axes (nothing is launched: the tensors are on the CPU), and the tables."""
import pytest
import torch

import risaattention_b200 as risa

BF16 = torch.bfloat16


def x(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def refuses(error, call, *args, match=None, **kwargs):
    with pytest.raises(error, match=match):
        call(*args, **kwargs)


# ---- positions of several axes ---------------------------------------------------------------------------
def test_sections():
    table = risa.rotary_table(16, sections=(2, 3, 3), device="cpu")
    assert table.axes.tolist() == [0, 0, 1, 1, 1, 2, 2, 2] and table.axis_count == 3 and table.axes.dtype == torch.uint8
    assert torch.equal(table.turns, risa.rotary_table(16, device="cpu").turns)
    dealt = risa.rotary_table(16, sections=(2, 3, 3), dealt=True, device="cpu")
    assert dealt.axes.tolist() == [0, 1, 2, 0, 1, 2, 1, 2]
    fresh = risa.rotary_table(16, sections=[2, 3, 3], restart=True, device="cpu")
    own = [risa.rotary_table(2 * n, device="cpu").turns.tolist() for n in (2, 3, 3)]
    assert fresh.turns.tolist() == own[0] + own[1] + own[2]
    both = risa.rotary_table(16, sections=(2, 3, 3), dealt=True, restart=True, scaling="linear", factor=2.0, device="cpu")
    own = [risa.rotary_table(2 * n, scaling="linear", factor=2.0, device="cpu").turns.tolist() for n in (2, 3, 3)]
    assert both.turns.tolist() == [own[0][0], own[1][0], own[2][0], own[0][1], own[1][1], own[2][1], own[1][2], own[2][2]]


@pytest.mark.parametrize("arguments", [dict(sections=(2, 3, 2)), dict(sections=()), dict(sections=(8, 0)), dict(sections=(1,) * 8 + (0,)), dict(sections=(9, -1)),
                                       dict(sections=(4.0, 4.0)), dict(dealt=True), dict(restart=True)])
def test_section_refusals(arguments):
    refuses(ValueError, risa.rotary_table, 16, **arguments, device="cpu")
    refuses(ValueError, risa.rotary_table, 18, sections=(1,) * 9, device="cpu")


def test_axes_refusals():
    table = risa.rotary_table(8, sections=(1, 3), device="cpu")
    rotate = risa.rotate_positions
    for shape, positions in [((2, 3, 8), ints(3)), ((2, 3, 8), ints(1, 2)), ((2, 3, 8), ints(3, 2)), ((2, 3, 8), ints(2, 1, 2)), ((2, 3, 5, 8), ints(2, 3, 5)),
                             ((2, 3, 5, 8), ints(2, 2, 4)), ((3, 3, 5, 8), ints(3, 5))]:
        refuses(ValueError, rotate, x(*shape), positions, table, match="positions")
    for shape, positions in [((2, 3, 8), ints(2)), ((2, 3, 8), ints(2, 2)), ((4, 3, 5, 8), ints(2, 4, 5)), ((4, 3, 5, 8), ints(2, 5)), ((4, 3, 5, 8), ints(5))]:
        refuses(ValueError, rotate, x(*shape), positions, table, match="CUDA device")
    refuses(ValueError, rotate, x(2, 3, 8), ints(2, 2), risa.rotary_table(8, device="cpu"), match="positions")
    refuses(TypeError, rotate, x(2, 3, 8), ints(2, 2), risa.RotaryTable(table.turns, 1.0, table.axes.int(), 2), match="uint8")
    refuses(ValueError, rotate, x(2, 3, 8), ints(2, 2), risa.RotaryTable(table.turns, 1.0, table.axes[:3], 2), match="each pair")
    for count in (0, 9, -1):
        refuses(ValueError, rotate, x(2, 3, 8), ints(2, 2), risa.RotaryTable(table.turns, 1.0, table.axes, count), match="1 to 8")
    cache, k, step = risa.allocate_key_value_cache(4, 2, 16, 64, device="cpu"), x(3, 2, 64), (ints(3, 2), ints(3))
    table = risa.rotary_table(64, sections=(16, 8, 8), device="cpu")
    append = risa.append_to_cache
    refuses(ValueError, append, cache, k, k, *step, rotary=table, positions=ints(2, 3), match="row for each")
    refuses(ValueError, append, cache, k, k, *step, rotary=table, positions=ints(3, 2), match="positions")
    refuses(ValueError, append, cache, k, k, *step, rotary=risa.rotary_table(64, device="cpu"), positions=ints(3, 3), match="positions")
    refuses(ValueError, append, cache, k, k, *step, rotary=table, positions=ints(3, 6)[:, ::2], match="contiguous")
    for positions in (None, ints(3), ints(3, 3)):
        refuses(ValueError, append, cache, k, k, *step, rotary=table, positions=positions, match="CUDA device")


# ---- first keys that stay visible ----------------------------------------------------------------------------
def test_sinks_refusals():
    cache = risa.allocate_key_value_cache(4, 2, 16, 64, device="cpu")
    q, lse, step = x(3, 4, 64), x(3, 4, dtype=torch.float32), (ints(3, 2), ints(3))
    for call, args in ((risa.paged_attention, (q, cache)), (risa.cached_key_weights, (q, lse, cache))):
        refuses(ValueError, call, *args, *step, sinks=4, match="window")
        refuses(ValueError, call, *args, *step, window=8, sinks=-1, match="negative")
        refuses(ValueError, call, *args, *step, window=8, sinks=2 ** 31, match="sinks")
        refuses(ValueError, call, *args, *step, window=8, sinks=4, is_causal=False, match="causal")
        refuses(ValueError, call, *args, *step, window=8, sinks=4, match="CUDA device")


# ---- a cache in 4 bits ---------------------------------------------------------------------------------------
U8 = torch.uint8


def test_four_bit_caches():
    cache = risa.allocate_key_value_cache(3, 2, 32, 128, dtype=U8, device="cpu")
    assert cache.quantized and cache.page_size == 32 and cache.head_dim == 128
    assert cache.keys.shape == (3, 2, 32, 64) and cache.key_scales.shape == (3, 2, 32 * 9) and cache.value_scales.dtype == U8
    make, rows, scales = risa.KeyValueCache, x(2, 1, 16, 32, dtype=U8), x(2, 1, 16 * 5, dtype=U8)
    make(rows, rows, scales, scales)
    for args, error in [((rows, rows), ValueError), ((rows, rows, scales[..., :64], scales), ValueError), ((rows, rows, scales, x(2, 1, 80, dtype=torch.int8)), TypeError),
                        ((rows, rows, scales, x(2, 80, 1, dtype=U8).transpose(1, 2)), None), ((rows, rows, scales, x(2, 80, 2, dtype=U8).transpose(1, 2)[:, :1]), ValueError),
                        ((x(2, 1, 16, 64, dtype=U8),) * 2 + (scales, scales), ValueError), ((x(2, 1, 16, 16, dtype=U8),) * 2 + (scales, scales), ValueError),
                        ((rows, rows.to(torch.int8), scales, scales), TypeError), ((x(2, 1, 16, 64, dtype=torch.int8),) * 2 + (scales, scales), TypeError)]:
        if error is None:
            make(*args)
            continue
        refuses(error, make, *args)


def test_four_bit_refusals():
    cache, step = risa.allocate_key_value_cache(4, 2, 16, 64, dtype=U8, device="cpu"), (ints(3, 2), ints(3))
    refuses(ValueError, risa.paged_attention, x(3, 4, 32), cache, *step, match="q must have shape")
    refuses(TypeError, risa.paged_attention, x(3, 4, 64, dtype=torch.float32), cache, *step, match="float16 or bfloat16")
    refuses(ValueError, risa.append_to_cache, cache, x(3, 2, 32), x(3, 2, 32), *step, match="k and v")
    refuses(ValueError, risa.paged_attention, x(3, 4, 64), cache, *step, match="CUDA device")
    refuses(ValueError, risa.append_to_cache, cache, x(3, 2, 64), x(3, 2, 64), *step, match="CUDA device")
    read = risa.read_from_cache
    refuses(ValueError, read, cache, *step, match="say which")
    refuses(TypeError, read, cache, *step, dtype=torch.float32, match="float16 or bfloat16")
    refuses(ValueError, read, cache, *step, query_offsets=ints(4), dtype=BF16, match="number of tokens")
    refuses(ValueError, read, cache, *step, tokens=5, dtype=BF16, match="one token")
    refuses(ValueError, read, cache, *step, query_offsets=ints(4), tokens=0, dtype=BF16, match="tokens")
    refuses(ValueError, read, cache, *step, dtype=BF16, match="CUDA device")
    refuses(TypeError, read, cache.keys, *step, dtype=BF16, match="KeyValueCache")
    plain = risa.allocate_key_value_cache(4, 2, 16, 64, device="cpu")
    refuses(TypeError, read, plain, *step, dtype=torch.float16, match="dtype of the cache")
    refuses(ValueError, read, plain, *step, match="CUDA device")


# ---- pages -----------------------------------------------------------------------------------------------------
def test_page_refusals():
    cache, table, lengths, references = risa.allocate_key_value_cache(4, 2, 16, 64, device="cpu"), ints(3, 2), ints(3), ints(4)
    other = risa.allocate_key_value_cache(2, 2, 16, 64, device="cpu")
    calls = [(risa.fork_sequences, (ints(5),)), (risa.resize_sequences, (ints(3),)), (risa.compact_cache, (other,))]
    for call, rest in calls:
        refuses(TypeError, call, cache.keys, references, table, lengths, *rest, match="KeyValueCache")
        refuses(ValueError, call, cache, ints(5), table, lengths, *rest, match="references")
        refuses(TypeError, call, cache, references.long(), table, lengths, *rest, match="references")
        refuses(ValueError, call, cache, ints(8)[::2], table, lengths, *rest, match="references")
        refuses(ValueError, call, cache, references, ints(3), lengths, *rest, match="page_table")
        refuses(ValueError, call, cache, references, table, ints(2), *rest, match="lengths")
        refuses(TypeError, call, cache, references, table.long(), lengths, *rest, match="int32")
        refuses(ValueError, call, cache, references, table, lengths, *rest, match="CUDA device")
    step = (cache, references, table, lengths)
    refuses(ValueError, risa.fork_sequences, *step, ints(0), match="parents")
    refuses(ValueError, risa.fork_sequences, *step, ints(2, 1), match="parents")
    refuses(TypeError, risa.fork_sequences, *step, ints(2).long(), match="int32")
    refuses(ValueError, risa.resize_sequences, *step, ints(4), match="new_lengths")
    refuses(TypeError, risa.resize_sequences, *step, ints(3).long(), match="int32")
    refuses(TypeError, risa.compact_cache, *step, other.keys, match="KeyValueCache")
    for make, error in ((dict(dtype=torch.float16), TypeError), (dict(dtype=torch.int8), TypeError)):
        refuses(error, risa.compact_cache, *step, risa.allocate_key_value_cache(4, 2, 16, 64, device="cpu", **make), match="dtype")
    for shape in ((4, 1, 16, 64), (4, 2, 32, 64), (4, 2, 16, 128)):
        refuses(ValueError, risa.compact_cache, *step, risa.allocate_key_value_cache(*shape, device="cpu"), match="same kind")
    refuses(ValueError, risa.compact_cache, *step, cache, match="another pool")
    refuses(ValueError, risa.compact_cache, *step, risa.KeyValueCache(cache.keys[1:], other.values.repeat(2, 1, 1, 1)[1:]), match="another pool")
    refuses(ValueError, risa.compact_cache, *step, risa.KeyValueCache(other.keys, cache.keys[:2]), match="another pool")
