"""A window in front of which the first keys stay visible: attention over all kinds of cache and the weights that keys receive, against 64 bits."""
import pytest
import serving_util as U
import torch
from test_gpu_serving import BF16, F16

import risaattention_b200 as risa
from risaattention_b200 import _backend

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_status():
    yield
    torch.cuda.synchronize()
    _backend._C.device_status()


def seen_with(sinks):
    """``U.seen`` for a window with first keys."""
    plain = U.seen

    def seen(n, count, causal, window, device):
        mask = plain(n, count, causal, window, device)
        if window:
            mask |= plain(n, count, causal, None, device) & (torch.arange(n, device=device) < sinks)
        return mask
    return seen


CASES = [
    # lengths, chunks, (q_heads, kv_heads), head_dim, page, window, sinks
    ([1000], [1], (8, 2), 128, 16, 100, 4),              # one token, a few first keys
    ([1000, 3, 90, 0], [1, 1, 1, 1], (16, 4), 64, 32, 60, 17),   # shorter than the window, than the sinks, empty
    ([700, 650], [1, 1], (8, 1), 128, 128, 1, 1),        # the smallest of both
    ([300, 301], [1, 1], (4, 4), 256, 16, 32, 300),      # first keys beyond the window's first
    ([2000, 37], [5, 2], (8, 2), 128, 16, 64, 64),       # some tokens each
    ([600], [7], (2, 1), 64, 64, 16, 599),               # all but one are first keys
    ([1500], [40], (4, 1), 128, 16, 129, 5),             # tensor cores: tiles in front, one key into a tile
    ([3000, 400, 1], [200, 33, 1], (8, 2), 128, 64, 256, 130),
    ([900], [300], (4, 2), 64, 32, 33, 128),             # a tile of first keys
    ([1200, 70], [64, 64], (2, 2), 256, 128, 100, 65),
    ([777], [777], (4, 4), 128, 16, 50, 20),             # a prompt from its start
    ([2100], [40], (4, 4), 128, 16, 2000, 2 ** 31 - 1),  # everything
]


def step(case, dtype, quantized, seed=0):
    lengths, chunks, (q_heads, kv_heads), head_dim, page, window, sinks = case
    b = U.batch_of(lengths, chunks, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page=page, dtype=dtype, quantized=quantized, seed=seed)
    return b, dict(window=window, sinks=sinks)


def hide_unread(b, window, sinks):
    """Pages that no token sees are gone: their entries lead nowhere, and what is between visible keys of a page is NaN."""
    page = b.cache.page_size
    for s, (n, c) in enumerate(zip(b.lengths.tolist(), b.chunks)):
        mask = U.seen(n, c, True, window, "cuda")
        unseen = ~mask.any(0)
        for i in range(-(-n // page)):
            gone = unseen[i * page:(i + 1) * page]
            rows = (int(b.table[s, i]), slice(None), gone.nonzero()[:, 0])
            for x in (b.cache.key_scales, b.cache.value_scales) if b.cache.quantized else (b.cache.keys, b.cache.values):
                x[rows[0], :, rows[2]] = float("nan")
            if gone.all():
                b.table[s, i] = -1


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype,quantized", [(BF16, False), (F16, False), (BF16, True)])
def test_attention(case, dtype, quantized, monkeypatch):
    b, options = step(case, dtype, quantized)
    monkeypatch.setattr(U, "seen", seen_with(options["sinks"]))
    offsets = b.offsets if max(b.chunks) > 1 or min(b.chunks) == 0 else None
    want, want_lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=offsets, return_lse=True, **options)
    U.assert_attention(b, want, want_lse, window=options["window"])
    weights = risa.cached_key_weights(b.q, want_lse, b.cache, b.table, b.lengths, query_offsets=offsets, **options)
    # keys that nobody sees are never read, nor are the entries of pages that hold nothing else
    hide_unread(b, options["window"], options["sinks"])
    out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=offsets, return_lse=True, **options)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    again = risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=offsets, **options)
    assert torch.equal(again, weights)


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype,quantized", [(BF16, False), (F16, True)])
def test_key_weights(case, dtype, quantized, monkeypatch):
    b, options = step(case, dtype, quantized, seed=1)
    monkeypatch.setattr(U, "seen", seen_with(options["sinks"]))
    lse = U.attention(b, window=options["window"])[1].float()
    want, size = U.weights(b, lse, window=options["window"])
    previous = torch.rand(want.shape, device="cuda")
    got = risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=b.offsets, previous=previous, **options)
    rows = max(b.chunks) * (b.q.shape[1] // b.cache.keys.shape[1])
    # a weight is off by its score's rounding (as in U.assert_attention), 2^-23 of each of the sum's additions, and the last one's
    score = size * b.q.shape[2] * 2.0 ** -23 + 2.0 ** -20 * (1 + size)
    bound = want * (2 * score + rows * 2.0 ** -23 + 2.0 ** -22) + 2.0 ** -23 * (want + previous.double()) + 1e-30
    assert bool(((got.double() - previous.double() - want).abs() <= bound).all())


def test_the_window_alone_is_as_it_was():
    b, _ = step(CASES[7], BF16, False)
    options = dict(query_offsets=b.offsets, return_lse=True)
    want = risa.paged_attention(b.q, b.cache, b.table, b.lengths, window=256, **options)
    got = risa.paged_attention(b.q, b.cache, b.table, b.lengths, window=256, sinks=0, **options)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # first keys inside every row's window change nothing of what is visible
    whole = risa.paged_attention(b.q, b.cache, b.table, b.lengths, window=5000, sinks=70, **options)
    want = risa.paged_attention(b.q, b.cache, b.table, b.lengths, **options)
    assert torch.equal(whole[0], want[0]) and torch.equal(whole[1], want[1])


def test_pages_outside_the_pool_in_front_of_the_window():
    """Hidden and reported, in first keys as anywhere."""
    for chunk in (1, 40):
        b, options = step(([800], [chunk], (4, 2), 128, 16, 64, 32), BF16, False)
        b.table[0, 1] = 10 ** 6
        out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True, **options)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="page outside the pool"):
            _backend._C.device_status()
        want = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True, window=64, sinks=16)
        # the same keys, in steps that may differ: sums of 80 products in another order, and one rounding of the output
        assert float((lse - want[1]).abs().max()) < 1e-4 and float((out.double() - want[0].double()).abs().max()) <= 2.0 ** -7 * float(out.abs().max())


def test_replayed_with_other_lengths(monkeypatch):
    b, options = step(([900, 500], [40, 1], (4, 2), 64, 16, 100, 9), F16, False)
    monkeypatch.setattr(U, "seen", seen_with(9))
    call = lambda: risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True, **options)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call()
    for lengths in ([900, 500], [41, 1], [300, 499]):
        b.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        U.assert_attention(b, out, lse, window=100)
