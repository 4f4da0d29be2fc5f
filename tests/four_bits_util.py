"""A cache in 4 bits written out in 64 bits: packing, unpacking and what a row becomes, for the tests."""
from __future__ import annotations

import serving_util as U
import torch

import risaattention_b200 as risa


def packed(codes):
    """int codes [..., channels] -> uint8 [..., channels / 2]."""
    u = (codes.long() + 8).unflatten(-1, (-1, 4, 2))
    words = sum(u[..., i, j] << (16 * j + 4 * i) for i in range(4) for j in range(2))
    return torch.stack([(words >> (8 * b)) & 255 for b in range(4)], -1).flatten(-2).to(torch.uint8)


def unpacked(data):
    """uint8 [..., channels / 2] -> int64 codes [..., channels]."""
    b = data.long().unflatten(-1, (-1, 4))
    words = sum(b[..., i] << (8 * i) for i in range(4))
    return torch.stack([((words >> (16 * j + 4 * i)) & 15) - 8 for i in range(4) for j in range(2)], -1).flatten(-2)


def scales_of(data, page):
    """(exponents int64 [..., page], group scales float64 [..., page, groups])."""
    groups = data[..., page:].unflatten(-1, (page, -1)).contiguous().view(torch.float8_e4m3fn).float().double()
    return data[..., :page].long(), groups


def power(exponents):
    return torch.where(exponents > 0, torch.where(exponents == 255, torch.inf, torch.exp2(exponents.double() - 127)), 0.0)


def values_of(codes, groups, exponents):
    return (codes.double().unflatten(-1, (-1, 16)) * groups[..., None]).flatten(-2) * power(exponents)[..., None]


def pool_values(cache, what):
    """float64 [pages, kv_heads, page, head_dim]"""
    exponents, groups = scales_of(getattr(cache, what[:-1] + "_scales"), cache.page_size)
    return values_of(unpacked(getattr(cache, what)), groups, exponents)


def cached(batch, s, what="keys"):
    """``serving_util.cached`` for any cache."""
    if batch.cache.keys.dtype != torch.uint8:
        return plain_cached(batch, s, what)
    n, page = int(batch.lengths[s]), batch.cache.page_size
    ids = batch.table[s, :-(-n // page)].long()
    return pool_values(batch.cache, what)[ids].transpose(0, 1).flatten(1, 2)[:, :n]


plain_cached = U.cached


def quantized(x):
    """Codes, group scales and exponents of rows x (64 bits)."""
    most = x.abs().amax(-1)
    exponent = torch.ceil(torch.log2(most.clamp_min(1e-300) / 3136.0)).long()
    exponent += (torch.exp2(exponent.double()) * 3136 < most).long()
    exponent -= (torch.exp2(exponent.double() - 1) * 3136 >= most).long()
    exponent = exponent.clamp_min(-126)
    token = torch.exp2(exponent.double())[..., None]
    grouped = x.unflatten(-1, (-1, 16))
    ratio = grouped.abs().amax(-1) / 7 / token
    step = torch.exp2(torch.floor(torch.log2(ratio.clamp_min(2.0 ** -6))) - 3)
    groups = (ratio / step).round() * step
    size = groups[..., None] * token[..., None]
    codes = torch.where(size > 0, grouped / size, 0.0).round().clamp(-7, 7).flatten(-2)
    bad, zero = ~most.isfinite(), most == 0
    exponent = torch.where(bad, 255, torch.where(zero, 0, exponent + 127))
    gone = (bad | zero)[..., None]
    return torch.where(gone, 0.0, codes).long(), torch.where(gone, 0.0, groups), exponent


def batch_of(lengths, chunks, *, q_heads, kv_heads, head_dim, page, dtype=torch.bfloat16, seed=0, spread=3, **more):
    """``serving_util.batch_of`` with the cache in 4 bits; what no sequence uses holds ones in every bit."""
    b = U.batch_of(lengths, chunks, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype, seed=seed, **more)
    g = torch.Generator("cuda").manual_seed(seed)
    used = ~b.cache.keys[..., 0].isnan()  # [pages, heads, page]
    tensors = [[], []]
    for _ in range(2):
        codes = torch.randint(-7, 8, b.cache.keys.shape, device="cuda", generator=g)
        groups = (448 * torch.rand(*used.shape, head_dim // 16, device="cuda", generator=g) ** 2).to(torch.float8_e4m3fn).view(torch.uint8)
        exponents = torch.randint(127 - 10 - spread, 127 - 9, used.shape, device="cuda", generator=g).to(torch.uint8)
        rows = packed(codes)
        rows[~used], groups[~used], exponents[~used] = 255, 255, 255
        tensors[0].append(rows)
        tensors[1].append(torch.cat((exponents, groups.flatten(-2)), -1))
    b.cache = risa.KeyValueCache(*tensors[0], *tensors[1])
    return b


def assert_attention(batch, out, lse, **options):
    """``serving_util.assert_attention`` for 4-bit caches: codes enter exactly, and a probability (times its key's scale) is rounded to
    fp16 or, where bf16 queries are many, to bf16: half a step of the queries' type covers both."""
    want, want_lse, spread, size = U.attention(batch, **options)
    half = torch.finfo(out.dtype).eps / 2
    score = size * out.shape[-1] * 2.0 ** -23 + 2.0 ** -20 * (1 + size)
    assert torch.equal(torch.isneginf(lse.double()), torch.isneginf(want_lse))
    visible = ~torch.isneginf(want_lse)
    assert bool(((lse.double() - want_lse).abs()[visible] <= (score + 2.0 ** -22 * (1 + want_lse.abs()))[visible]).all())
    bound = half * want.abs() + spread * (half + 2.1 * score[..., None]) + torch.finfo(out.dtype).tiny
    error = (out.double() - want).abs()
    assert bool((error <= bound).all()), f"{float((error / bound.clamp_min(1e-300)).max()):.2f} of the bound"
    assert not bool(out[~visible].any())
