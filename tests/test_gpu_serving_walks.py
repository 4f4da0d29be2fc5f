"""Serving calls in which a worker walks over many tiles, blocks and units, so that its rings go round several times."""
import pytest
import serving_util as U
import torch
from test_gpu_serving import BF16, F16, assert_weights

import risaattention_b200 as risa
from risaattention_b200 import _backend

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_status():
    yield
    torch.cuda.synchronize()
    _backend._C.device_status()


@pytest.mark.parametrize("head_dim,page,dtype,quantized,chunks", [(64, 16, BF16, False, [16, 32, 9]), (64, 32, F16, True, [16, 20, 11]),
                                                                  (128, 64, F16, False, [16, 32, 10]), (256, 32, BF16, True, [16, 12, 9])])
def test_key_weights_of_many_blocks_of_one_tile(head_dim, page, dtype, quantized, chunks):
    """Up to 128 query rows of a key head are one tile of each block of 256 keys: a worker has some ten of them, adds what was
    there before and hands half of every sum from one group of warps to the other."""
    b = U.batch_of([32768, 20001, 9000], chunks, q_heads=32, kv_heads=8, head_dim=head_dim, page=page, dtype=dtype, quantized=quantized, seed=head_dim)
    _, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    weigh = lambda **more: risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=b.offsets, **more)  # noqa: E731
    plain = weigh()
    assert_weights(b, plain, lse)
    previous = torch.rand(plain.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    first = weigh(previous=previous)
    assert_weights(b, first, lse, previous)
    for _ in range(20):
        assert torch.equal(weigh(previous=previous), first)
    assert torch.equal(weigh(), plain)


@pytest.mark.parametrize("head_dim", [64, 128])
def test_key_weights_of_many_short_sequences(head_dim):
    """Blocks of at most 128 keys: the second group of keys sits out and hands its turns on."""
    lengths = [40 + (29 * i) % 89 for i in range(200)]
    b = U.batch_of(lengths, [9 + i % 20 for i in range(200)], q_heads=32, kv_heads=8, head_dim=head_dim, page=16, seed=2)
    _, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    previous = torch.rand(200, 8, b.table.shape[1] * 16, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    first = risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=b.offsets, previous=previous)
    assert_weights(b, first, lse, previous)
    for _ in range(20):
        assert torch.equal(risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=b.offsets, previous=previous), first)


def attend(b, **options):
    return risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True, **options)


@pytest.mark.parametrize("head_dim,page,dtype,quantized", [(64, 64, F16, False), (128, 64, BF16, False), (128, 16, BF16, True), (256, 32, BF16, False), (64, 128, F16, True), (256, 64, F16, True)])
@pytest.mark.parametrize("options", [{}, {"window": 5000}])
def test_long_chunks(head_dim, page, dtype, quantized, options):
    """A worker goes through more than twenty tiles and starts in the middle of a unit; attention, then the weights it gave."""
    b = U.batch_of([13001], [1100], q_heads=16, kv_heads=4, head_dim=head_dim, page=page, dtype=dtype, quantized=quantized, seed=head_dim)
    out, lse = attend(b, **options)
    U.assert_attention(b, out, lse, **options)
    for _ in range(5):
        again = attend(b, **options)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    weigh = lambda: risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=b.offsets, **options)  # noqa: E731
    first = weigh()
    assert_weights(b, first, lse, **options)
    for _ in range(5):
        assert torch.equal(weigh(), first)


@pytest.mark.parametrize("head_dim,quantized", [(64, False), (128, True), (256, False)])
@pytest.mark.parametrize("q_heads", [32, 64])
def test_many_units_of_one_tile(head_dim, quantized, q_heads):
    """A worker goes through some ten units: their queries follow one another, and (32 heads) the second row group sits out."""
    lengths = [34 + (31 * i) % 80 for i in range(240)]
    b = U.batch_of(lengths, [9 + i % 23 for i in range(240)], q_heads=q_heads, kv_heads=8, head_dim=head_dim, page=16, quantized=quantized, extra_rows=3, seed=2)
    out, lse = attend(b)
    U.assert_attention(b, out, lse)
    for _ in range(20):
        again = attend(b)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("quantized", [False, True])
def test_long_single_tokens(quantized):
    """More steps per worker than page numbers are looked up at a time."""
    b = U.batch_of([32768, 30011, 1, 20000], [1, 3, 1, 2], q_heads=16, kv_heads=8, head_dim=128, page=16, quantized=quantized, seed=1)
    out, lse = attend(b)
    U.assert_attention(b, out, lse)
    first = risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=b.offsets)
    assert_weights(b, first, lse)
    for _ in range(5):
        again = attend(b)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
        assert torch.equal(risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=b.offsets), first)
