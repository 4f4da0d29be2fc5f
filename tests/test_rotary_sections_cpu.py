"""Sections of a rotary table from anything that gives its numbers once."""
import pytest
import torch

import risaattention_b200 as risa


@pytest.mark.parametrize("options", [{}, {"dealt": True}, {"restart": True}, {"dealt": True, "restart": True}])
def test_sections_are_read_once(options):
    want = risa.rotary_table(16, sections=(2, 3, 3), device="cpu", **options)
    for sections in (iter((2, 3, 3)), (n for n in (2, 3, 3)), map(int, "233")):
        got = risa.rotary_table(16, sections=sections, device="cpu", **options)
        assert torch.equal(got.turns, want.turns) and torch.equal(got.axes, want.axes) and got.axis_count == 3
