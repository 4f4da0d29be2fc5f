"""Steps of small batches and the serving operators written out in 64 bits, token by token, for the tests."""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

import risaattention_b200 as risa


@dataclass
class Batch:
    cache: risa.KeyValueCache
    table: torch.Tensor
    lengths: torch.Tensor
    offsets: torch.Tensor
    chunks: list
    q: torch.Tensor
    seed: int


def batch_of(lengths, chunks, *, q_heads, kv_heads, head_dim, page, dtype=torch.bfloat16, quantized=False, spare=3, extra_rows=0,
             stale=float("nan"), seed=0, width=None):
    """A cache whose pages lie in random order, with ``stale`` in every place that no sequence uses, and the
    queries of a step.  Table entries behind a sequence are -1."""
    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=g)
    shape = (pages, kv_heads, page, head_dim)
    width = width or max(max(counts), 1)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    used = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for s, (n, c) in enumerate(zip(lengths, counts)):
        ids = order[at:at + c]
        at += c
        table[s, :c] = ids.int()
        for i in range(n):
            used[ids[i // page], i % page] = True
    if quantized:
        keys, values = (torch.randint(-127, 128, shape, generator=g, dtype=torch.int8) for _ in range(2))
        scales = [(torch.rand(shape[:3], generator=g) + 0.5) / 73 for _ in range(2)]
        for x in scales:
            x[~used[:, None, :].expand(shape[:3])] = stale
        cache = risa.KeyValueCache(keys.cuda(), values.cuda(), *(x.cuda() for x in scales))
    else:
        keys, values = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
        for x in (keys, values):
            x[~used[:, None, :, None].expand(shape)] = stale
        cache = risa.KeyValueCache(keys.cuda(), values.cuda())
    offsets = torch.tensor([0] + list(chunks)).cumsum(0).int()
    q = torch.randn(int(offsets[-1]) + extra_rows, q_heads, head_dim, generator=g).to(dtype)
    return Batch(cache, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), offsets.cuda(), list(chunks), q.cuda(), seed)


def cached(batch, s, what="keys"):
    """[kv_heads, tokens, head_dim] of sequence s in 64 bits."""
    pool = getattr(batch.cache, what)
    n, page = int(batch.lengths[s]), batch.cache.page_size
    ids = batch.table[s, :-(-n // page)].long()
    rows = pool[ids].double()
    if batch.cache.quantized:
        rows = rows * getattr(batch.cache, what[:-1] + "_scales")[ids].double()[..., None]
    return rows.transpose(0, 1).flatten(1, 2)[:, :n]


def seen(n, count, causal, window, device):
    """bool [count, n]"""
    place = torch.arange(n - count, n, device=device)[:, None]
    key = torch.arange(n, device=device)
    if not causal:
        return torch.ones(count, n, dtype=torch.bool, device=device)
    return (key <= place) & ((key > place - window) if window else True)


def attention(batch, *, scale=None, causal=True, window=None):
    """(out, lse, probabilities @ |values|, largest |scale q||k|) of every row, in 64 bits."""
    q = batch.q.double()
    tokens, q_heads, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((tokens, q_heads), -torch.inf, dtype=torch.float64, device=q.device)
    size = torch.zeros(tokens, q_heads, dtype=torch.float64, device=q.device)
    first = 0
    for s, count in enumerate(batch.chunks):
        k, v = cached(batch, s), cached(batch, s, "values")
        group = q_heads // k.shape[0]
        n = k.shape[1]
        mask = seen(n, count, causal, window, q.device)
        rows = mask.any(-1)
        for h in range(q_heads):
            qs = q[first:first + count, h]
            x = (qs @ k[h // group].T * scale).masked_fill(~mask, -torch.inf)
            part = x.logsumexp(-1) if n else torch.full((count,), -torch.inf, dtype=torch.float64, device=q.device)
            p = (x - part[:, None]).exp()
            p = torch.where(rows[:, None], p, 0.0)
            out[first:first + count, h], spread[first:first + count, h] = p @ v[h // group], p @ v[h // group].abs()
            lse[first:first + count, h] = part
            if n:
                size[first:first + count, h] = (qs.abs() @ k[h // group].abs().T * abs(scale)).amax(-1)
        first += count
    return out, lse, spread, size


def assert_attention(batch, out, lse, **options):
    """Errors counted: scores are sums of head_dim products in 32 bits whose terms add up to ``size`` at most
    (2^-23 of it for each addition, and 2^-20 for the exponent's own scaling and exponential), which moves a probability
    by that relative amount, twice with the denominator; a probability is rounded once (half a step of its type; over a
    cache of codes that is fp16); the output is rounded once.  Codes themselves are exact."""
    want, want_lse, spread, size = attention(batch, **options)
    half = torch.finfo(out.dtype).eps / 2
    part = torch.finfo(torch.float16).eps / 2 if batch.cache.quantized else half
    score = size * out.shape[-1] * 2.0 ** -23 + 2.0 ** -20 * (1 + size)
    assert torch.equal(torch.isneginf(lse.double()), torch.isneginf(want_lse))
    visible = ~torch.isneginf(want_lse)
    assert ((lse.double() - want_lse).abs()[visible] <= (score + 2.0 ** -22 * (1 + want_lse.abs()))[visible]).all()
    bound = half * want.abs() + spread * (part + 2.1 * score[..., None]) + torch.finfo(out.dtype).tiny
    error = (out.double() - want).abs()
    assert (error <= bound).all(), f"{float((error / bound.clamp_min(1e-300)).max()):.2f} of the bound"
    assert (out[~visible] == 0).all()


def weights(batch, lse, *, scale=None, causal=True, window=None):
    """float64 [batch, kv_heads, slots] for the given lse, and the largest |scale q||k| that enters."""
    q = batch.q.double()
    d = q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    kv_heads = batch.cache.keys.shape[1]
    group = q.shape[1] // kv_heads
    out = torch.zeros(len(batch.chunks), kv_heads, batch.table.shape[1] * batch.cache.page_size, dtype=torch.float64, device=q.device)
    first, size = 0, 0.0
    for s, count in enumerate(batch.chunks):
        k = cached(batch, s)
        n = k.shape[1]
        mask = seen(n, count, causal, window, q.device)
        for h in range(q.shape[1]):
            qs = q[first:first + count, h]
            x = qs @ k[h // group].T * scale
            w = (x - lse[first:first + count, h].double()[:, None]).exp()
            out[s, h // group, :n] += torch.where(mask, w, 0.0).sum(0)
            if n and count:
                size = max(size, float((qs.abs() @ k[h // group].abs().T).max()) * abs(scale))
        first += count
    return out, size


def turned(x, positions, frequencies, magnitude, interleaved, sign=1):
    """x [..., channels] rotated by positions of shape x.shape[:-1], in 64 bits."""
    x = x.double().clone()
    f = torch.tensor(frequencies, dtype=torch.float64, device=x.device)
    r = 2 * len(frequencies)
    # frequencies and positions are exact enough in 64 bits up to 2^31 positions (2^-53 of 2^31 radians)
    angle = positions.double()[..., None] * f * sign
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., first].clone(), x[..., second].clone()
    x[..., first] = magnitude * (a * angle.cos() - b * angle.sin())
    x[..., second] = magnitude * (b * angle.cos() + a * angle.sin())
    return x


def evicted(weights, length, budget, recent):
    """Places that one key head keeps."""
    count = min(length, budget)
    recent = min(recent, count)
    key = lambda i: (-math.inf if math.isnan(weights[i]) else -weights[i], not math.isnan(weights[i]), i)  # noqa: E731
    others = sorted(range(length - recent), key=key)[:count - recent]
    return sorted(others) + list(range(length - recent, length))
