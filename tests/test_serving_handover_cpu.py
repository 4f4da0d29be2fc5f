"""The hand-over of half sums between the warps of weigh_tc.cu, in every interleaving (a model on the CPU).

Scores of tile t are there once every warp of both halves has freed those of tile t - 2.  With blocks of one tile a giving
warp frees tile b, writes its sum into slot b and arrives; a taking warp frees tile b, waits for slot b's barrier and reads."""
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parents[1] / "risaattention_b200" / "csrc" / "weigh_tc.cu").read_text()
SLOTS = 4


def faults(warps, blocks, barriers):
    """What goes wrong with `barriers` barriers (phases told apart by parity) over SLOTS slots: "stuck", "wrong sum"."""
    start = ((0,) * warps, (0,) * warps, ((0, 0),) * barriers, ((-1,) * warps,) * SLOTS)
    put = lambda t, i, x: t[:i] + (x,) + t[i + 1:]  # noqa: E731
    seen, todo, found = {start}, [start], set()
    while todo:
        give, take, bars, slots = todo.pop()
        moves = []
        ready = lambda b: b < 2 or all(p > 2 * (b - 2) for p in give + take)  # noqa: E731
        for i in range(warps):
            b, freed = divmod(give[i], 2)
            if b < blocks and not freed and ready(b):
                moves.append((put(give, i, give[i] + 1), take, bars, slots))
            if b < blocks and freed:
                phase, count = bars[b % barriers]
                bar = (phase, count + 1) if count + 1 < warps else (phase + 1, 0)
                moves.append((put(give, i, give[i] + 1), take, put(bars, b % barriers, bar), put(slots, b % SLOTS, put(slots[b % SLOTS], i, b))))
            b, freed = divmod(take[i], 2)
            if b < blocks and not freed and ready(b):
                moves.append((give, put(take, i, take[i] + 1), bars, slots))
            if b < blocks and freed and bars[b % barriers][0] % 2 != b // barriers % 2:
                if slots[b % SLOTS][i] != b:
                    found.add("wrong sum")
                moves.append((give, put(take, i, take[i] + 1), bars, slots))
        if not moves and min(give + take) < 2 * blocks:
            found.add("stuck")
        todo += [m for m in moves if m not in seen]
        seen.update(moves)
    return found


@pytest.mark.parametrize("warps,blocks", [(1, 13), (2, 9), (3, 5)])
def test_a_barrier_for_every_slot(warps, blocks):
    assert faults(warps, blocks, SLOTS) == set()


def test_one_barrier_is_too_few():
    assert faults(1, 5, 1) == {"stuck"} and faults(2, 5, 1) == {"stuck", "wrong sum"}


def test_the_kernel_is_the_model():
    slots = re.search(r"constexpr int kHalves = (\d+);", SOURCE)
    assert slots and int(slots[1]) == SLOTS
    assert "half_full[2][kHalves]" in SOURCE and "float half[kHalves][2][128]" in SOURCE
    assert "notes->half[block % kHalves][g][lane]" in SOURCE
    assert "bars->half_full[g][block % kHalves]), parity = block / kHalves & 1" in SOURCE
