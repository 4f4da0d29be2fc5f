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
