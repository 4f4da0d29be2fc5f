"""Chunks over cached codes: what rounding a probability undergoes goes by what its own row sees, whatever the scales."""
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


def attend(b, **options):
    return risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True, **options)


@pytest.mark.parametrize("head_dim,page,dtype", [(64, 16, BF16), (128, 16, F16), (128, 128, BF16), (256, 32, BF16)])
@pytest.mark.parametrize("chunk,window", [(50, None), (200, None), (60, 90)])
def test_chunks_over_value_scales_of_any_size(head_dim, page, dtype, chunk, window):
    """Scales of values that differ by 2^60 within a tile, zeros among them.  What is rounded is at most 2^8 in units of the
    row's largest probability times scale, so fp16 holds everything down to 2^-25 of that; 300 keys of less lose 2^-17 of it
    together, which is far below the half step of those that count."""
    b = U.batch_of([300], [chunk], q_heads=4, kv_heads=2, head_dim=head_dim, page=page, dtype=dtype, quantized=True, seed=4)
    g = torch.Generator("cuda").manual_seed(0)
    used = b.table[0].long()
    scales = torch.pow(2.0, torch.randint(-60, 1, b.cache.value_scales[used].shape, device="cuda", generator=g).float())
    scales[0, :, 3:9] = 0
    b.cache.value_scales[used] = scales
    out, lse = attend(b, window=window)
    U.assert_attention(b, out, lse, window=window)


def assert_attention(b, out, lse, **options):
    """U.assert_attention's bound, which takes probability times scale as rounded relative to itself, and what fp16 adds to it:
    half of its smallest step, 2^-25, for each key, in units of at most the row's largest probability times scale and times
    codes of up to 127.  (Where the code of a key of scale 2^40 is 0, that is all there is of the channel: the other keys are
    2^-40 of it.)"""
    want, _, spread, size = U.attention(b, **options)
    top, first, d = torch.zeros(b.q.shape[:2], dtype=torch.float64, device="cuda"), 0, b.q.shape[2]
    for s, count in enumerate(b.chunks):
        n, k = int(b.lengths[s]), U.cached(b, s)
        scales = b.cache.value_scales[b.table[s].clamp_min(0).long()].transpose(0, 1).flatten(1).double()[:, :n]
        mask = U.seen(n, count, True, options.get("window"), "cuda")
        for h in range(b.q.shape[1]):
            x = (b.q[first:first + count, h].double() @ k[h * k.shape[0] // b.q.shape[1]].T * d ** -0.5).masked_fill(~mask, -torch.inf)
            top[first:first + count, h] = (x.softmax(-1) * scales[h * k.shape[0] // b.q.shape[1]]).amax(-1) * n
        first += count
    half, part = torch.finfo(out.dtype).eps / 2, torch.finfo(F16).eps / 2
    score = size * d * 2.0 ** -23 + 2.0 ** -20 * (1 + size)
    bound = half * want.abs() + spread * (part + 2.1 * score[..., None]) + torch.finfo(out.dtype).tiny + 127 * 2.0 ** -25 * top[..., None]
    assert ((out.double() - want).abs() <= bound).all()


# 2^14 times an ordinary scale is as much as an output in fp16 holds
@pytest.mark.parametrize("head_dim,dtype,large", [(64, F16, 2.0 ** 14), (64, BF16, 2.0 ** 40), (128, BF16, 2.0 ** 14), (128, BF16, 2.0 ** 40), (256, BF16, 2.0 ** 40)])
def test_a_hidden_key_of_large_scale_leaves_the_rows_that_do_not_see_it(head_dim, dtype, large):
    """Under the causal rule and in front of a window: the same bits as if the key's values were ordinary."""
    b = U.batch_of([260, 200], [60, 40], q_heads=8, kv_heads=2, head_dim=head_dim, page=16, dtype=dtype, quantized=True, seed=7)
    want, want_lse = attend(b)
    ordinary = b.cache.value_scales.clone()
    b.cache.value_scales[b.table[0, 16].long(), :, 3] *= large  # key 259: the last token of the first sequence alone
    out, lse = attend(b)
    assert torch.equal(out[:59], want[:59]) and torch.equal(out[60:], want[60:])
    assert not torch.equal(out[59], want[59])
    assert_attention(b, out, lse)
    assert ((lse - want_lse).abs() <= 2.0 ** -20 * (1 + want_lse.abs())).all()
    b.cache.value_scales.copy_(ordinary)
    want, _ = attend(b, window=30)
    b.cache.value_scales[b.table[1, 8].long(), :, 5] *= large  # key 133 of the second: tokens at 160 and later do not see it
    out, lse = attend(b, window=30)
    assert torch.equal(out[:60], want[:60]) and torch.equal(out[63:], want[63:])
    assert_attention(b, out, lse, window=30)


def test_a_row_of_small_scales_behind_one_of_large_scales():
    """A window slides from keys of scale 2^20 to keys of scale 2^-20: every row in its own units."""
    b = U.batch_of([600], [300], q_heads=8, kv_heads=2, head_dim=128, page=16, quantized=True, seed=9)
    for i, page in enumerate(b.table[0].long().tolist()):
        b.cache.value_scales[page] = 2.0 ** (20 - i)
    out, lse = attend(b, window=40)
    U.assert_attention(b, out, lse, window=40)
    # values of keys that no row sees may be anything finite
    b.cache.value_scales[b.table[0, :16].long()] = 3e38
    again, _ = attend(b, window=40)
    assert torch.equal(again, out)
