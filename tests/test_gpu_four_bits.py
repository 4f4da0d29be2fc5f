"""A cache in 4 bits: what append writes, reading it back, attention and key weights over it, eviction from it, against 64 bits."""
import four_bits_util as F
import pytest
import serving_util as U
import torch
from test_gpu_serving import BF16, F16

import risaattention_b200 as risa
from risaattention_b200 import _backend

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def prepared(monkeypatch):
    monkeypatch.setattr(U, "cached", F.cached)
    yield
    torch.cuda.synchronize()
    _backend._C.device_status()


def with_sinks(monkeypatch, sinks):
    plain = U.seen

    def seen(n, count, causal, window, device):
        mask = plain(n, count, causal, window, device)
        if window:
            mask |= plain(n, count, causal, None, device) & (torch.arange(n, device=device) < sinks)
        return mask
    monkeypatch.setattr(U, "seen", seen)


CASES = [
    # lengths, chunks, (q_heads, kv_heads), head_dim, page, options
    ([1], [1], (4, 1), 128, 16, {}),
    ([0, 16, 17, 300, 15], [1, 1, 1, 1, 1], (8, 2), 128, 16, {}),
    ([1000, 63], [1, 1], (8, 8), 64, 32, {}),
    ([700, 129], [1, 1], (16, 2), 256, 64, {}),
    ([2500], [1], (16, 1), 128, 128, {"scale": -0.07}),             # 16 rows, parts of a long sequence, a negative scale
    ([90, 33, 5], [4, 3, 5], (4, 2), 64, 16, {}),                    # some tokens each
    ([40, 500], [4, 1], (8, 2), 256, 16, {"is_causal": False}),
    ([260], [260], (2, 1), 128, 16, {}),                             # tensor cores
    ([1000, 40, 77], [100, 1, 40], (4, 2), 128, 64, {}),
    ([515], [70], (4, 4), 64, 32, {"is_causal": False}),
    ([300, 290], [130, 33], (2, 2), 256, 128, {"scale": 0.0}),
    ([900, 20], [1, 1], (8, 2), 128, 32, {"window": 100, "sinks": 5}),
    ([900, 700], [50, 3], (8, 2), 128, 16, {"window": 77, "sinks": 20}),
    ([640], [90], (2, 2), 64, 64, {"window": 200}),
    ([3], [5], (2, 1), 128, 16, {}),                                 # more new tokens than the sequence has
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_attention(case, dtype, monkeypatch):
    lengths, chunks, (q_heads, kv_heads), head_dim, page, options = case
    b = F.batch_of(lengths, chunks, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype)
    options = dict(options)
    if "sinks" in options:
        with_sinks(monkeypatch, options["sinks"])
    offsets = None if set(chunks) == {1} else b.offsets
    out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=offsets, return_lse=True, **options)
    plain = {("causal" if k == "is_causal" else k): v for k, v in options.items() if k != "sinks"}
    F.assert_attention(b, out, lse, **plain)
    # the weights that keys receive, for the rows' own denominators
    previous = torch.rand(len(lengths), kv_heads, b.table.shape[1] * page, device="cuda")
    got = risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=offsets, previous=previous, **options)
    want, size = U.weights(b, torch.where(lse.isneginf(), torch.inf, lse), **plain)
    rows = max(chunks) * (q_heads // kv_heads)
    score = size * head_dim * 2.0 ** -23 + 2.0 ** -20 * (1 + size)
    bound = want * (2 * score + rows * 2.0 ** -23 + 2.0 ** -22) + 2.0 ** -23 * (want + previous.double()) + 1e-30
    assert bool(((got.double() - previous.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("chunk,dtype", [(1, BF16), (40, BF16), (40, F16)])
def test_scales_of_every_size(chunk, dtype):
    """Tokens whose scales differ by 2^40, scales of zero, groups of zero: small values are lost beside large ones, nothing else."""
    b = F.batch_of([300, 64], [chunk, chunk], q_heads=4, kv_heads=2, head_dim=128, page=16, spread=0, dtype=dtype)
    for scales, rest in ((b.cache.key_scales, 0), (b.cache.value_scales, 1)):
        exponents = scales[..., :16]
        used = exponents != 255
        exponents[..., 3::7] = 0
        if rest:
            exponents[..., 5::7] -= 40
        exponents[~used] = 255
        scales[..., 16 + 8 * 2:16 + 8 * 3][used.any(-1)] = 0  # all groups of the third token of a page
    out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    F.assert_attention(b, out, lse)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_row_that_is_not_finite_is_nan_for_those_who_see_it(dtype):
    for chunk in (1, 40):
        b = F.batch_of([200, 150], [chunk, chunk], q_heads=2, kv_heads=1, head_dim=128, page=16, dtype=dtype)
        want = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets)
        b.cache.value_scales[int(b.table[0, 3]), 0, 5] = 255
        out = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets)
        assert bool(out[:chunk].isnan().any(-1).all()) and torch.equal(out[chunk:], want[chunk:])


APPENDS = [
    # lengths, chunks, (q_heads, kv_heads), head_dim, page, rotary
    ([40, 17, 90, 8], [40, 1, 33, 0], (4, 2), 128, 16, dict(rotary_dim=128)),
    ([33, 128, 1], [1, 1, 1], (8, 1), 64, 32, dict(rotary_dim=32)),
    ([300], [300], (3, 3), 256, 128, dict(rotary_dim=256, sections=(32, 48, 48))),
    ([16, 70], [16, 65], (4, 4), 128, 64, None),
    ([1000, 500], [999, 400], (8, 8), 128, 16, dict(rotary_dim=96, magnitude=1.3)),
    ([3, 20], [7, 2], (2, 2), 64, 16, None),   # more tokens than the sequence has
    ([60, 9], [50, 9], (40, 40), 128, 16, dict(rotary_dim=128)),   # more heads than a block of threads takes at once
    ([40], [33], (80, 20), 64, 32, dict(rotary_dim=64)),
    ([40], [33], (9, 9), 256, 16, dict(rotary_dim=128, sections=(24, 40), dealt=True)),
]


def places_of(lengths, chunks):
    return torch.cat([torch.arange(n - c, n) for n, c in zip(lengths, chunks)]).cuda(), [s for s, c in enumerate(chunks) for _ in range(c)]


@pytest.mark.parametrize("case", APPENDS)
@pytest.mark.parametrize("dtype,interleaved", [(BF16, False), (F16, True)])
def test_append(case, dtype, interleaved):
    lengths, chunks, (q_heads, kv_heads), d, page, rotary = case
    b = F.batch_of(lengths, chunks, q_heads=q_heads, kv_heads=kv_heads, head_dim=d, page=page, dtype=dtype, extra_rows=2)
    g = torch.Generator("cuda").manual_seed(7)
    n = sum(chunks)
    k, v = (torch.randn(n + 2, kv_heads, d, device="cuda", generator=g) * torch.exp(2 * torch.randn(n + 2, kv_heads, 1, device="cuda", generator=g)) for _ in range(2))
    v[::3, :, ::5] = v[::3, :, 1:2] / 2  # ties between codes
    k[::4, :, 16:32] *= 1e-4             # groups far below the others
    k[1], v[2] = 0, 0
    k, v = k.to(dtype), v.to(dtype)
    before = [x.clone() for x in b.cache.tensors]
    options, want_k = {}, k.double()
    place, owner = places_of(lengths, chunks)
    if rotary is not None:
        table = risa.rotary_table(**rotary)  # of several axes: without positions all of them have the place
        frequencies = [u % 2 ** 64 / 2 ** 64 * 2 * torch.pi for u in table.turns.tolist()]
        options = dict(q=b.q, rotary=table, interleaved=interleaved)
        positions = torch.cat((place, place.new_zeros(2)))
        want_k = U.turned(k, positions[:, None].expand(n + 2, kv_heads), frequencies, float(torch.tensor(table.magnitude)), interleaved)
    out = risa.append_to_cache(b.cache, k, v, b.table, b.lengths, query_offsets=b.offsets, **options)
    assert (out is None) == (rotary is None)
    written = torch.zeros(before[0].shape[:3], dtype=torch.bool, device="cuda")
    for i, (p, s) in enumerate(zip(place.tolist(), owner)):
        if p >= 0:
            written[int(b.table[s, p // page]), :, p % page] = True
    for what, rows in (("keys", want_k), ("values", v.double())):
        codes, groups, exponents = F.quantized(rows)
        e, s = F.scales_of(getattr(b.cache, what[:-1] + "_scales"), page)
        got = F.unpacked(getattr(b.cache, what))
        there = place >= 0
        ids = torch.tensor([int(b.table[o, p // page]) if p >= 0 else 0 for p, o in zip(place.tolist(), owner)], device="cuda")[there]
        at = (ids, slice(None), place[there] % page)
        assert torch.equal(e[at], exponents[:n][there]) and torch.equal(s[at], groups[:n][there]) and torch.equal(got[at], codes[:n][there])
    # what no token of the step owns stays as it was
    after = b.cache.tensors
    for i in range(2):
        assert torch.equal(after[i][~written], before[i][~written])
        a, c = after[2 + i], before[2 + i]
        assert torch.equal(a[..., :page][~written], c[..., :page][~written])
        assert torch.equal(a[..., page:].unflatten(-1, (page, -1))[~written], c[..., page:].unflatten(-1, (page, -1))[~written])
    # and it reads back as it was stored
    keys, values = risa.read_from_cache(b.cache, b.table, b.lengths, query_offsets=b.offsets, tokens=n + 2, dtype=dtype)
    for got, what in ((keys, "keys"), (values, "values")):
        pool = F.pool_values(b.cache, what)
        for i, (p, s) in enumerate(zip(place.tolist(), owner)):
            want = pool[int(b.table[s, p // page]), :, p % page].float().to(dtype) if p >= 0 else torch.zeros_like(got[i])
            assert torch.equal(got[i], want)
        assert not bool(got[n:].any())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_append_of_extreme_rows(dtype):
    top = torch.finfo(dtype).max
    tiny = torch.finfo(dtype).smallest_normal
    rows = torch.zeros(12, 1, 64)
    rows[0] = top
    rows[1, :, 5] = -top
    rows[2] = tiny
    rows[3, :, 63] = tiny / 16
    rows[4, :, ::2] = torch.inf
    rows[5, :, 9] = torch.nan
    rows[6] = torch.arange(-32, 32)          # whole numbers: ties at every half
    rows[7] = 3136.0 / 1024
    rows[8] = torch.linspace(-1, 1, 64) * 3136.0 / 1024
    rows[9, :, 0], rows[9, :, 16:] = 1.0, 2.0 ** -14
    rows[10] = torch.tensor([7.0, 3.5, -3.5, 0.5, -0.5, 2.5, 1.5, -6.5] * 8)
    rows = rows.to(dtype).cuda()
    cache = risa.allocate_key_value_cache(1, 1, 16, 64, dtype=torch.uint8)
    step = (torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.tensor([12], dtype=torch.int32, device="cuda"))
    offsets = torch.tensor([0, 12], dtype=torch.int32, device="cuda")
    risa.append_to_cache(cache, rows, rows.flip(0), *step, query_offsets=offsets)
    for what, want in (("keys", rows), ("values", rows.flip(0))):
        codes, groups, exponents = F.quantized(want.double())
        e, s = F.scales_of(getattr(cache, what[:-1] + "_scales"), 16)
        assert torch.equal(e[0, 0, :12], exponents[:, 0]) and torch.equal(s[0, 0, :12], groups[:, 0]) and torch.equal(F.unpacked(getattr(cache, what))[0, 0, :12], codes[:, 0])
    keys, _ = risa.read_from_cache(cache, *step, query_offsets=offsets, tokens=12, dtype=BF16)
    assert bool(keys[4:6].isnan().all()) and bool(keys[[0, 1, 2, 3, 6, 7, 8, 9, 10, 11]].isfinite().all())


def test_rows_beside_ones_that_are_not_finite():
    """Rotated keys of which every other head is not finite: the others are those of the formula, also where they are decided in 64
    bits (many rows, so that some of them are)."""
    n, d = 600, 128
    cache = risa.allocate_key_value_cache(38, 4, 16, d, dtype=torch.uint8)
    table, length = torch.arange(38, dtype=torch.int32, device="cuda")[None], torch.tensor([n], dtype=torch.int32, device="cuda")
    k = torch.randn(n, 4, d, device="cuda").bfloat16()
    k[::2, 1, 5], k[1::2, 1, 100], k[:, 3, 64] = torch.nan, torch.inf, -torch.inf
    rotary = risa.rotary_table(d)
    risa.append_to_cache(cache, k, k, table, length, query_offsets=torch.tensor([0, n], dtype=torch.int32, device="cuda"), rotary=rotary)
    place = torch.arange(n, device="cuda")
    frequencies = [u % 2 ** 64 / 2 ** 64 * 2 * torch.pi for u in rotary.turns.tolist()]
    codes, groups, exponents = F.quantized(U.turned(k, place[:, None].expand(n, 4), frequencies, 1.0, False))
    e, s = F.scales_of(cache.key_scales, 16)
    got = F.unpacked(cache.keys)
    at = (place // 16, slice(None), place % 16)
    assert torch.equal(e[at], exponents) and torch.equal(s[at], groups) and torch.equal(got[at], codes)
    assert bool((exponents[:, 1::2] == 255).all()) and bool((exponents[:, ::2] < 255).all())


@pytest.mark.parametrize("kind", [BF16, F16, torch.int8])
def test_reading_other_caches(kind):
    quantized = kind == torch.int8
    b = U.batch_of([40, 0, 130], [3, 0, 130], q_heads=2, kv_heads=3, head_dim=64, page=32, dtype=BF16 if quantized else kind, quantized=quantized, extra_rows=1)
    dtype = F16 if quantized else None
    keys, values = risa.read_from_cache(b.cache, b.table, b.lengths, query_offsets=b.offsets, tokens=134, dtype=dtype)
    for got, what in ((keys, "keys"), (values, "values")):
        want = torch.cat((U.cached(b, 0, what)[:, 37:], U.cached(b, 2, what)), 1).transpose(0, 1)
        assert got.dtype == (dtype or kind) and bool(((got[:133].double() - want).abs() <= 2.0 ** -11 * want.abs()).all()) and not bool(got[133].any())
    one = risa.read_from_cache(b.cache, b.table, b.lengths, dtype=dtype)
    assert torch.equal(one[0][0], keys[2]) and not bool(one[0][1].any()) and torch.equal(one[1][2], values[132])


@pytest.mark.parametrize("head_dim,page", [(64, 16), (128, 32), (256, 16)])
def test_eviction(head_dim, page):
    b = F.batch_of([200, 5, 64], [1, 1, 1], q_heads=2, kv_heads=2, head_dim=head_dim, page=page, spare=12)
    g = torch.Generator("cuda").manual_seed(3)
    weights = torch.rand(3, 2, b.table.shape[1] * page, device="cuda", generator=g)
    taken = {int(i) for row, n in zip(b.table.tolist(), b.lengths.tolist()) for i in row[:-(-n // page)]}
    free = [i for i in range(b.cache.keys.shape[0]) if i not in taken]
    each = -(-48 // page)
    target = torch.tensor(free[:3 * each], dtype=torch.int32, device="cuda").view(3, each)
    before = [torch.stack([F.cached(b, s, w)[h] for h in range(2)]) for w in ("keys", "values") for s in range(3)]
    kept, lengths, _ = risa.evict_from_cache(b.cache, b.table, b.lengths, weights, target, budget=48, recent=7)
    assert lengths.tolist() == [48, 5, 48]
    b.table, b.lengths = target, lengths
    for w, what in enumerate(("keys", "values")):
        for s in range(3):
            now = F.cached(b, s, what)
            for h in range(2):
                chosen = U.evicted(weights[s, h].tolist(), [200, 5, 64][s], 48, 7)
                assert kept[s, h, :len(chosen)].tolist() == chosen
                assert torch.equal(now[h], before[3 * w + s][h][chosen])


@pytest.mark.parametrize("chunk", [2, 33])
def test_the_largest_rows(chunk):
    """Keys of up to 2^117 against queries as small, and such values: sums of 100 of them in 32 bits end at 2^124.  (Values of 2^126
    themselves would overflow any such sum.)"""
    b = F.batch_of([100], [chunk], q_heads=1, kv_heads=1, head_dim=128, page=16)
    x = torch.randn(100, 1, 128, device="cuda").clamp(-3, 3) * 2.0 ** 115
    risa.append_to_cache(b.cache, x.bfloat16(), x.flip(0).bfloat16(), b.table, b.lengths, query_offsets=torch.tensor([0, 100], dtype=torch.int32, device="cuda"))
    b.q *= 2.0 ** -115
    out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    F.assert_attention(b, out, lse)


def test_a_conversation(monkeypatch):
    """Prompts taken in, tokens drawn, keys weighed and the conversation shortened, twice, with a window at the end."""
    d, page = 128, 16
    cache = risa.allocate_key_value_cache(64, 2, page, d, dtype=torch.uint8)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1)).int().view(2, 20).cuda()
    g = torch.Generator("cuda").manual_seed(2)
    rotary = risa.rotary_table(d, sections=(16, 24, 24))
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    weights = None
    for chunks in ([100, 37], [1, 1], [1, 1], [40, 1]):
        n = sum(chunks)
        lengths = lengths + torch.tensor(chunks, dtype=torch.int32, device="cuda")
        offsets = torch.tensor([0, chunks[0], n], dtype=torch.int32, device="cuda")
        q, k, v = (torch.randn(n, h, d, device="cuda", generator=g).bfloat16() for h in (4, 2, 2))
        positions = torch.randint(0, 4000, (3, n), device="cuda", generator=g)
        q = risa.append_to_cache(cache, k, v, table, lengths, query_offsets=offsets, q=q, rotary=rotary, positions=positions)
        out, lse = risa.paged_attention(q, cache, table, lengths, query_offsets=offsets, return_lse=True)
        b = U.Batch(cache, table, lengths, offsets, chunks, q, 0)
        F.assert_attention(b, out, lse)
        weights = risa.cached_key_weights(q, lse, cache, table, lengths, query_offsets=offsets, previous=weights)
    target = torch.arange(40, 48, dtype=torch.int32, device="cuda").view(2, 4)
    _, lengths, _ = risa.evict_from_cache(cache, table, lengths, weights, target, budget=60, recent=10)
    q = torch.randn(2, 4, d, device="cuda", generator=g).bfloat16()
    out, lse = risa.paged_attention(q, cache, target, lengths, window=20, sinks=3, return_lse=True)
    with_sinks(monkeypatch, 3)
    F.assert_attention(U.Batch(cache, target, lengths, torch.tensor([0, 1, 2]), [1, 1], q, 0), out, lse, window=20)


def test_pools_past_32_bits():
    """Pages that lie 4 GB into a pool give what they give at its front, in every call."""
    d, page, heads, lengths, chunks = 256, 128, 8, [500, 131], [40, 1]
    b = F.batch_of(lengths, chunks, q_heads=16, kv_heads=heads, head_dim=d, page=page, dtype=F16)
    few, far = b.cache.keys.shape[0], 34000
    big = risa.allocate_key_value_cache(far + 2 * few, heads, page, d, dtype=torch.uint8)
    assert big.keys[far:].data_ptr() - big.keys.data_ptr() > 2 ** 32
    for to, source in zip(big.tensors, b.cache.tensors):
        to[far:far + few] = source
    table = torch.where(b.table >= 0, b.table + far, -1)
    k, v = (torch.randn(41, heads, d, device="cuda").half() for _ in range(2))
    got = []
    for cache, rows in ((b.cache, b.table), (big, table)):
        step = (cache, rows, b.lengths)
        risa.append_to_cache(cache, k, v, *step[1:], query_offsets=b.offsets)
        out, lse = risa.paged_attention(b.q, *step, query_offsets=b.offsets, window=300, sinks=9, return_lse=True)
        weights = risa.cached_key_weights(b.q, lse, *step, query_offsets=b.offsets)
        got.append((out, lse, weights, *risa.read_from_cache(*step, query_offsets=b.offsets, tokens=41, dtype=F16)))
    assert all(torch.equal(x, y) for x, y in zip(*got))
    # a page that is shared is copied, and all pages in use move to another pool
    references = torch.ones(far + 2 * few, dtype=torch.int32, device="cuda")
    references[far + few:] = 0
    children, sizes = risa.fork_sequences(big, references, table, b.lengths, torch.tensor([1, 0], dtype=torch.int32, device="cuda"))
    sizes = risa.resize_sequences(big, references, children, sizes, sizes + 1) - 1
    assert bool((children == far + few).any()) and bool((children == far + few + 1).any())
    references[:far] = 0
    target = risa.allocate_key_value_cache(2 * few, heads, page, d, dtype=torch.uint8)
    moved, _, used = risa.compact_cache(big, references, children, sizes, target)
    offsets = torch.tensor([0, 131, 631], dtype=torch.int32, device="cuda")
    want = risa.read_from_cache(b.cache, b.table.flip(0), b.lengths.flip(0), query_offsets=offsets, tokens=631, dtype=F16)
    for cache, rows in ((big, children), (target, moved)):
        now = risa.read_from_cache(cache, rows, sizes, query_offsets=offsets, tokens=631, dtype=F16)
        assert torch.equal(now[0], want[0]) and torch.equal(now[1], want[1])
    assert int(used) == few + 2
    # and eviction copies to its end
    goal = torch.arange(far + few, far + few + 2, dtype=torch.int32, device="cuda").view(2, 1)
    kept, left, _ = risa.evict_from_cache(big, table, b.lengths, got[1][2], goal, budget=100, recent=20)
    now = risa.read_from_cache(big, goal, left, query_offsets=torch.tensor([0, 100, 200], dtype=torch.int32, device="cuda"), tokens=200, dtype=F16)
    whole = risa.read_from_cache(b.cache, b.table, b.lengths, query_offsets=torch.tensor([0, 500, 631], dtype=torch.int32, device="cuda"), tokens=631, dtype=F16)
    for s, start in enumerate((0, 500)):
        for h in range(heads):
            assert torch.equal(now[0][100 * s:100 * s + 100, h], whole[0][start + kept[s, h].long(), h])


def test_pages_outside_the_pool():
    for chunk in (1, 40):
        b = F.batch_of([200], [chunk], q_heads=2, kv_heads=1, head_dim=128, page=16)
        b.table[0, 4] = -5
        calls = [lambda: risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets),
                 lambda: risa.cached_key_weights(b.q, torch.zeros(chunk, 2, device="cuda"), b.cache, b.table, b.lengths, query_offsets=b.offsets)]
        if chunk == 40:
            b.table[0, 11] = 10 ** 7
            x = torch.zeros(40, 1, 128, device="cuda", dtype=BF16)
            calls += [lambda: risa.append_to_cache(b.cache, x, x, b.table, b.lengths, query_offsets=b.offsets),
                      lambda: risa.read_from_cache(b.cache, b.table, b.lengths, query_offsets=b.offsets, tokens=40, dtype=BF16)]
        for call in calls:
            out = call()
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError, match="page outside the pool"):
                _backend._C.device_status()
            assert out is None or all(bool(x.isfinite().all()) for x in (out if isinstance(out, tuple) else (out,)))


def test_replayed_on_another_stream():
    b = F.batch_of([300, 200], [40, 1], q_heads=4, kv_heads=2, head_dim=64, page=16, dtype=F16)
    k, v = (torch.randn(41, 2, 64, device="cuda").half() for _ in range(2))

    def step():
        risa.append_to_cache(b.cache, k, v, b.table, b.lengths, query_offsets=b.offsets)
        return risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for lengths in ([300, 200], [111, 200], [40, 1]):
        b.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        k.normal_()
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.current_stream())
            graph.replay()
        torch.cuda.synchronize()
        F.assert_attention(b, out, lse)
