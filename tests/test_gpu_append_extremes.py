"""Rotated keys at both ends of 32 bits on their way into a cache in 4 bits: the codes are those of the exactly rotated rows."""
import four_bits_util as F
import pytest
import serving_util as U
import torch

import risaattention_b200 as risa

pytestmark = pytest.mark.gpu


def check(k, *, interleaved=False, turned=None, magnitude=1.0):
    n, heads, d = k.shape
    pages = -(-n // 16)
    cache = risa.allocate_key_value_cache(pages, heads, 16, d, dtype=torch.uint8)
    table, length = torch.arange(pages, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda")
    rotary = risa.rotary_table(turned or d, magnitude=magnitude)
    risa.append_to_cache(cache, k, k, table, length, query_offsets=torch.tensor([0, n], dtype=torch.int32, device="cuda"), rotary=rotary, interleaved=interleaved)
    place = torch.arange(n, device="cuda")
    frequencies = [u % 2 ** 64 / 2 ** 64 * 2 * torch.pi for u in rotary.turns.tolist()]
    x = U.turned(k, place[:, None].expand(n, heads), frequencies, float(torch.tensor(magnitude)), interleaved)
    codes, groups, exponents = F.quantized(x)
    e, s = F.scales_of(cache.key_scales, 16)
    at = (place // 16, slice(None), place % 16)
    assert torch.equal(e[at], exponents) and torch.equal(s[at], groups) and torch.equal(F.unpacked(cache.keys)[at], codes)
    return x


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,turned", [(64, 64), (128, 64), (256, 256)])
def test_rows_that_pass_the_largest_float(d, turned, interleaved):
    """Both channels of a pair near bf16's maximum come to sqrt(2) times that, which 32 bits do not hold and the scales do; beside rows that are not
    finite, and such that lie near a border."""
    g = torch.Generator("cuda").manual_seed(d)
    k = torch.randn(400, 5, d, device="cuda", generator=g)
    k[:, 1] = k[:, 1].sign() * torch.finfo(torch.bfloat16).max
    k[::2, 2], k[1::2, 3] = k[::2, 2].sign() * 3e38, k[1::2, 3].sign() * 2.2e38
    k[::5, 4, 3] = torch.nan
    k[1::5, 4, d - 1] = torch.inf
    x = check(k.bfloat16(), interleaved=interleaved, turned=turned)
    assert bool((x[:, 1].abs().amax(-1) > torch.finfo(torch.float32).max).float().mean() > 0.9)


def test_rows_that_the_scales_do_not_hold():
    """Past 2^119 times 7 * 448 (by a magnitude of the table) a row becomes one that is not finite."""
    k = torch.full((20, 2, 64), 3e38, device="cuda")
    k[:, 1] = 1.0
    cache = risa.allocate_key_value_cache(2, 2, 16, 64, dtype=torch.uint8)
    table, length = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), torch.tensor([20], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 20], dtype=torch.int32, device="cuda")
    risa.append_to_cache(cache, k.bfloat16(), k.bfloat16(), table, length, query_offsets=offsets, rotary=risa.rotary_table(64, magnitude=1e6))
    keys, values = risa.read_from_cache(cache, table, length, query_offsets=offsets, tokens=20, dtype=torch.bfloat16)
    assert bool(keys[:, 0].isnan().all()) and bool(keys[:, 1].isfinite().all()) and bool(values.isfinite().all())


@pytest.mark.parametrize("exponent", [-126, -130, -132, -133])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rows_below_the_smallest_normal_float(exponent, interleaved):
    g = torch.Generator("cuda").manual_seed(-exponent)
    check((torch.randn(60000, 8, 64, device="cuda", generator=g) * 2.0 ** (exponent / 2) * 2.0 ** (exponent / 2)).bfloat16(), interleaved=interleaved)
