"""Rotary positions, the paged cache, attention over it, key weights and eviction against plain 64-bit
implementations, at the sizes and masks where they can go wrong."""
import math

import pytest
import serving_util as U
import torch

import risaattention_b200 as risa
from risaattention_b200 import _backend

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def no_status():
    yield
    torch.cuda.synchronize()
    _backend._C.device_status()


# ---- rotation ---------------------------------------------------------------------------------------------
ROTATIONS = [
    # dtype, shape, rotary_dim, interleaved, options
    (BF16, (64, 32, 128), 128, False, {}),
    (F16, (1, 3, 64), 64, True, {}),
    (F32, (7, 5, 128), 64, False, {"magnitude": 1.25}),
    (BF16, (2, 4, 33, 256), 128, True, {"scaling": "linear", "factor": 8.0}),
    (F32, (3, 2, 17, 80), 20, False, {"scaling": "base", "factor": 4.0}),
    (F16, (2, 3, 5, 10), 6, True, {}),
    (BF16, (1, 16, 1000, 64), 64, False, {"scaling": "parts", "factor": 4.0, "original_length": 4096}),
    (F32, (1, 1, 2), 2, False, {}),
]


def rotation_bound(x, want, magnitude):
    """Cosine and sine: the angle in turns is rounded to 2^-24 of itself (at most 1/2 turn = pi radians) and sincospi
    gives two units in the last place; each output is two products and a sum, then one rounding to the type."""
    r = x.double().abs()
    pair = r.amax(-1, keepdim=True) * 2 * abs(magnitude)
    return torch.finfo(x.dtype).eps / 2 * want.abs() + pair * (math.pi * 2.0 ** -24 + 2.0 ** -22) + torch.finfo(x.dtype).tiny


@pytest.mark.parametrize("dtype,shape,rotary_dim,interleaved,options", ROTATIONS)
@pytest.mark.parametrize("positions64", [False, True])
def test_rotation(dtype, shape, rotary_dim, interleaved, options, positions64):
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randn(shape, device="cuda", generator=g).to(dtype)
    table = risa.rotary_table(rotary_dim, **options)
    frequencies = risa.rotary_frequencies(rotary_dim, **{k: v for k, v in options.items() if k != "magnitude"})
    tokens = shape[0] if len(shape) == 3 else shape[2]
    where = (tokens,) if len(shape) == 3 else (shape[0], tokens)
    positions = torch.randint(-5, 2 ** 31 - 1 if positions64 else 200000, where, device="cuda", generator=g)
    positions = positions if positions64 else positions.int()
    spread = positions[:, None] if len(shape) == 3 else positions[:, None, :]
    for transposed in (False, True):
        out = risa.rotate_positions(x, positions, table, interleaved=interleaved, transposed=transposed)
        # 2^-53 of 2^31 radians: the 64-bit oracle's own angle is off by 2.4e-7 there
        want = U.turned(x, spread.expand(x.shape[:-1]), frequencies, table.magnitude, interleaved, -1 if transposed else 1)
        slack = 4e-7 * 2 * x.double().abs().amax(-1, keepdim=True) * table.magnitude if positions64 else 0
        assert ((out.double() - want).abs() <= rotation_bound(x, want, table.magnitude) + slack).all()
        assert torch.equal(out[..., rotary_dim:], x[..., rotary_dim:])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rotation_of_views_in_place_and_out(dtype):
    g = torch.Generator("cuda").manual_seed(4)
    table = risa.rotary_table(64)
    base = torch.randn(2, 19, 6 * 128, device="cuda", generator=g).to(dtype)
    x = base.view(2, 19, 6, 128).transpose(1, 2)  # token-major storage
    positions = torch.arange(19, device="cuda", dtype=torch.int32)
    want = risa.rotate_positions(x.contiguous(), positions, table)
    assert torch.equal(risa.rotate_positions(x, positions, table), want)
    odd = torch.randn(2, 6, 19, 131, device="cuda", generator=g).to(dtype)[..., 1:129]  # rows that start anywhere
    odd.copy_(x)
    assert torch.equal(risa.rotate_positions(odd, positions, table), want)
    strided = positions.repeat_interleave(2)[::2]
    assert torch.equal(risa.rotate_positions(x, strided, table), want)
    out = torch.full_like(odd, 7)
    assert risa.rotate_positions(x, positions, table, out=out) is not None and torch.equal(out, want)
    risa.rotate_positions(x, positions, table, out=x)
    assert torch.equal(x, want)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_gradient(interleaved):
    g = torch.Generator("cuda").manual_seed(5)
    table = risa.rotary_table(16, magnitude=1.5)
    frequencies = risa.rotary_frequencies(16)
    positions = torch.randint(0, 9000, (2, 3), device="cuda", generator=g)
    x = torch.randn(2, 2, 3, 24, device="cuda", generator=g).requires_grad_()
    grad = torch.randn(x.shape, device="cuda", generator=g)
    got, = torch.autograd.grad(risa.rotate_positions(x, positions, table, interleaved=interleaved), x, grad)
    want = U.turned(grad, positions[:, None].expand(2, 2, 3), frequencies, 1.5, interleaved, -1)
    assert ((got.double() - want).abs() <= rotation_bound(grad, want, 1.5)).all()
    # differences: the map is linear, so they are exact but for the two values' rounding (2^-24 of about 8 each)
    direction = torch.randn(x.shape, device="cuda", generator=g)
    f = lambda y: (risa.rotate_positions(y, positions, table, interleaved=interleaved).double() * grad.double()).sum()  # noqa: E731
    with torch.no_grad():
        difference = f(x + direction) - f(x - direction)
    slope = 2 * (got.double() * direction.double()).sum()
    assert abs(float(difference - slope)) <= 2 * x.numel() * 8 * 4 * 2.0 ** -22
    # gradients that arrive as expanded views, and the gradient's own gradient
    risa.rotate_positions(x, positions, table, interleaved=interleaved).sum().backward()
    ones = U.turned(torch.ones_like(x), positions[:, None].expand(2, 2, 3), frequencies, 1.5, interleaved, -1)
    assert ((x.grad.double() - ones).abs() <= rotation_bound(torch.ones_like(x), ones, 1.5)).all()
    v = grad.clone().requires_grad_()
    first, = torch.autograd.grad(risa.rotate_positions(x, positions, table, interleaved=interleaved), x, v, create_graph=True)
    second, = torch.autograd.grad(first, v, direction)
    with torch.no_grad():
        assert torch.equal(second, risa.rotate_positions(direction, positions, table, interleaved=interleaved))


def test_rotation_gradient_on_another_stream_and_in_a_graph():
    table = risa.rotary_table(64)
    positions = torch.arange(40, device="cuda")
    x = torch.randn(40, 3, 64, device="cuda").requires_grad_()
    grad = torch.randn_like(x)
    want, = torch.autograd.grad(risa.rotate_positions(x, positions, table), x, grad)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, = torch.autograd.grad(risa.rotate_positions(x, positions, table), x, grad)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    leaf = x.detach().clone().requires_grad_()
    with torch.cuda.stream(side):
        torch.autograd.grad(risa.rotate_positions(leaf, positions, table), leaf, grad)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured, = torch.autograd.grad(risa.rotate_positions(leaf, positions, table), leaf, grad)
    grad.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, 2 * want)
    with pytest.raises(ValueError):
        risa.rotate_positions(x, positions[:3], table)


# ---- append -------------------------------------------------------------------------------------------------
APPENDS = [
    # lengths, chunks, heads, head_dim, page, rotary_dim
    ([5, 1, 40, 17], [5, 1, 3, 0], (4, 2), 64, 16, 64),
    ([33, 128, 1], [1, 1, 1], (8, 1), 128, 32, 64),
    ([200], [200], (3, 3), 256, 128, 256),
    ([16, 70], [16, 65], (4, 4), 128, 64, None),
]


@pytest.mark.parametrize("lengths,chunks,heads,head_dim,page,rotary_dim", APPENDS)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(lengths, chunks, heads, head_dim, page, rotary_dim, dtype, quantized, interleaved):
    b = U.batch_of(lengths, chunks, q_heads=heads[0], kv_heads=heads[1], head_dim=head_dim, page=page, dtype=dtype, quantized=quantized, stale=0.0)
    g = torch.Generator("cuda").manual_seed(9)
    tokens = sum(chunks)
    k, v = (torch.randn(tokens, heads[1], head_dim, device="cuda", generator=g).to(dtype) for _ in range(2))
    v[0, 0] = 0  # a row without a scale
    before = [None if x is None else x.clone() for x in b.cache.tensors]
    table = risa.rotary_table(rotary_dim) if rotary_dim else None
    q = risa.append_to_cache(b.cache, k, v, b.table, b.lengths, query_offsets=b.offsets, q=b.q if table else None, rotary=table, interleaved=interleaved)
    places = torch.cat([torch.arange(n - c, n) for n, c in zip(lengths, chunks)])
    owners = torch.cat([torch.full((c,), s) for s, c in enumerate(chunks)])
    want_k = k.double()
    if table:
        frequencies = risa.rotary_frequencies(rotary_dim)
        where = places.cuda()[:, None]
        want_k = U.turned(k, where.expand(tokens, heads[1]), frequencies, 1.0, interleaved)
        want_q = U.turned(b.q, where.expand(tokens, heads[0]), frequencies, 1.0, interleaved)
        assert ((q.double() - want_q).abs() <= rotation_bound(b.q, want_q, 1.0)).all()
    else:
        assert q is None
    page_of = b.table.cpu()[owners, places // page].long().cuda()
    slot = (places % page).cuda()
    for name, x, want in (("keys", k, want_k), ("values", v, v.double())):
        rows = getattr(b.cache, name)[page_of, :, slot].double()
        if not quantized:
            assert ((rows - want).abs() <= rotation_bound(x, want, 1.0)).all()
        else:
            scales = getattr(b.cache, name[:-1] + "_scales")[page_of, :, slot].double()
            step = want.abs().amax(-1) / 127
            assert ((scales - step).abs() <= 2.0 ** -20 * step).all()
            # half a step of the code, and the 32-bit arithmetic in front of it
            assert ((rows * scales[..., None] - want).abs() <= (0.5 + 1e-3) * step[..., None]).all()
            assert rows.abs().amax() <= 127
        # nothing else changed
        rest = torch.ones(b.cache.keys.shape[:3], dtype=torch.bool, device="cuda")
        rest[page_of, :, slot] = False
        assert torch.equal(getattr(b.cache, name)[rest], before[0 if name == "keys" else 1][rest])


def test_append_positions_views_and_rows_behind_the_last_sequence():
    b = U.batch_of([20, 9], [2, 3], q_heads=4, kv_heads=2, head_dim=64, page=16, stale=0.0, extra_rows=3)
    g = torch.Generator("cuda").manual_seed(2)
    qkv = torch.randn(8, 8, 64, device="cuda", generator=g).bfloat16()  # one projection's output: views with a larger token stride
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    table = risa.rotary_table(64)
    positions = torch.tensor([7, 100000, 3, 2, 1, 0, 0, 0], device="cuda")
    out = risa.append_to_cache(b.cache, k, v, b.table, b.lengths, query_offsets=b.offsets, q=q, rotary=table, positions=positions)
    assert torch.equal(out[:5], risa.rotate_positions(q, positions, table)[:5]) and (out[5:] == 0).all()
    place = torch.tensor([18, 19, 6, 7, 8])
    pages = b.table.cpu()[torch.tensor([0, 0, 1, 1, 1]), place // 16].long().cuda()
    assert torch.equal(b.cache.keys[pages, :, (place % 16).cuda()], risa.rotate_positions(k, positions, table)[:5])
    assert torch.equal(b.cache.values[pages, :, (place % 16).cuda()], v[:5])


def test_append_writes_nothing_for_short_sequences_and_bad_pages():
    b = U.batch_of([2, 20, 33], [4, 1, 1], q_heads=2, kv_heads=2, head_dim=64, page=16, stale=0.0)
    before = b.cache.keys.clone()
    k = torch.ones(6, 2, 64, device="cuda").bfloat16()
    b.table[1, 1] = b.cache.keys.shape[0]  # one behind the pool
    b.table[2, 2] = -1
    risa.append_to_cache(b.cache, k, k, b.table, b.lengths, query_offsets=b.offsets)
    with pytest.raises(RuntimeError, match="outside the pool"):
        _backend._C.device_status()
    changed = (b.cache.keys != before).any(-1).any(1).nonzero()
    assert changed.tolist() == [[int(b.table[0, 0]), 0], [int(b.table[0, 0]), 1]]


def test_append_of_infinities_reads_back_as_nan():
    cache = risa.allocate_key_value_cache(1, 1, 16, 64, dtype=torch.int8)
    k = torch.zeros(1, 1, 64, device="cuda", dtype=BF16)
    k[0, 0, 3], v = math.inf, k.clone()
    v[0, 0, 5] = math.nan
    risa.append_to_cache(cache, k, v, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda"))
    assert torch.isnan(cache.keys[0, 0, 0].float() * cache.key_scales[0, 0, 0]).all()
    assert torch.isnan(cache.values[0, 0, 0].float() * cache.value_scales[0, 0, 0]).all()


# ---- attention ------------------------------------------------------------------------------------------------
STEPS = {
    "one_key": ([1], [1]),
    "single_tokens": ([17, 16, 300, 15, 1, 129], [1] * 6),
    "longer": ([1000, 2049], [1, 1]),
    "chunks": ([40, 200, 33, 150], [40, 17, 1, 130]),
    "empty": ([0, 5, 64, 3], [2, 5, 0, 6]),  # no keys; all keys new; no tokens; more tokens than keys
    "long_chunk": ([700], [300]),
}


@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("heads", [(4, 2), (8, 1), (3, 3), (20, 1)])
@pytest.mark.parametrize("head_dim,page", [(64, 16), (128, 32), (128, 128), (256, 64)])
@pytest.mark.parametrize("dtype,quantized", [(BF16, False), (F16, False), (BF16, True), (F16, True)])
def test_attention(step, heads, head_dim, page, dtype, quantized):
    lengths, chunks = STEPS[step]
    b = U.batch_of(lengths, chunks, q_heads=heads[0], kv_heads=heads[1], head_dim=head_dim, page=page, dtype=dtype, quantized=quantized, seed=len(step))
    offsets = None if chunks == [1] * len(chunks) else b.offsets
    out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=offsets, return_lse=True)
    U.assert_attention(b, out, lse)


@pytest.mark.parametrize("step", ["single_tokens", "chunks", "empty", "long_chunk"])
@pytest.mark.parametrize("options", [{"is_causal": False}, {"window": 1}, {"window": 20}, {"window": 128, "scale": 0.3}, {"scale": -0.05}, {"scale": 0.0}])
@pytest.mark.parametrize("head_dim,quantized", [(64, False), (128, True), (128, False)])
def test_attention_masks_and_scales(step, options, head_dim, quantized):
    lengths, chunks = STEPS[step]
    b = U.batch_of(lengths, chunks, q_heads=8, kv_heads=2, head_dim=head_dim, page=16, quantized=quantized, seed=3)
    out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True, **options)
    U.assert_attention(b, out, lse, causal=options.get("is_causal", True), window=options.get("window"), scale=options.get("scale"))


def test_attention_window_reads_no_page_in_front_of_it():
    b = U.batch_of([300, 500], [1, 40], q_heads=4, kv_heads=2, head_dim=128, page=16, seed=1)
    want = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, window=32)
    for s, first in ((0, 300 - 32), (1, 460 - 31)):  # first key that the first token sees
        gone = b.table[s, :first // 16].long()
        b.cache.keys[gone], b.cache.values[gone] = math.nan, math.nan
        page = int(b.table[s, first // 16])
        b.cache.values[page, :, :first % 16] = math.nan
        b.table[s, :first // 16] = -1
    assert torch.equal(risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, window=32), want)


@pytest.mark.parametrize("chunks", [[1, 1], [1, 200]])
def test_attention_hides_pages_outside_the_pool(chunks):
    b = U.batch_of([400, 400], chunks, q_heads=4, kv_heads=1, head_dim=128, page=16, seed=8)
    want = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets)
    b.table[1, 3], b.table[1, 5] = -7, 2 ** 30
    out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    with pytest.raises(RuntimeError, match="sequence 1 .*outside the pool"):
        _backend._C.device_status()
    assert torch.equal(out[:1], want[:1])
    # as if those keys were not there
    keep = torch.ones(400, dtype=torch.bool, device="cuda")
    keep[48:64] = keep[80:96] = False
    b.table[1, 3] = b.table[1, 5] = 0
    k, v = U.cached(b, 1)[0], U.cached(b, 1, "values")[0]
    place = torch.arange(400 - chunks[1], 400, device="cuda")[:, None]
    for h in range(4):
        x = (b.q[1:, h].double() @ k.T * 128 ** -0.5).masked_fill(~(keep & (torch.arange(400, device="cuda") <= place)), -torch.inf)
        p = x.softmax(-1)
        # as in assert_attention: scores to 1e-4, one rounding of the probability, one of the output
        assert ((out[1:, h].double() - p @ v).abs() <= 2.0 ** -8 * (p @ v).abs() + (2.0 ** -8 + 1e-3) * (p @ v.abs())).all()


def test_attention_rows_behind_the_last_sequence_and_out():
    b = U.batch_of([50, 70], [1, 3], q_heads=4, kv_heads=2, head_dim=64, page=16, extra_rows=5)
    out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    assert (out[4:] == 0).all() and torch.isneginf(lse[4:]).all()
    given = torch.full((9, 6, 64), 3.0, device="cuda", dtype=BF16)[:, 1:5]
    same = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, out=given)
    assert same.data_ptr() == given.data_ptr() and torch.equal(given[:4], out[:4]) and (given[4:] == 3).all()


def test_rows_of_no_sequence_in_front_and_in_a_given_output():
    b = U.batch_of([50, 70], [1, 60], q_heads=4, kv_heads=2, head_dim=64, page=16, extra_rows=5)
    want, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    q = torch.cat([b.q[-3:], b.q])
    for given in (None, torch.full_like(q, 3)):
        out, got = risa.paged_attention(q, b.cache, b.table, b.lengths, query_offsets=b.offsets + 3, return_lse=True, out=given)
        rest = 0 if given is None else 3
        assert torch.equal(out[3:64], want[:61]) and (out[:3] == rest).all() and (out[64:] == rest).all()
        assert torch.equal(got[3:64], lse[:61]) and torch.isneginf(got[:3]).all() and torch.isneginf(got[64:]).all()


@pytest.mark.parametrize("head_dim", [64, 256])
@pytest.mark.parametrize("lengths,chunks", [([900], [1]), ([40, 5000, 800], [1, 1, 200]), ([3000], [700])])
def test_attention_into_its_queries(lengths, chunks, head_dim):
    b = U.batch_of(lengths, chunks, q_heads=8, kv_heads=2, head_dim=head_dim, page=32)
    want = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets)
    wide = torch.zeros(b.q.shape[0], 12, head_dim, device="cuda", dtype=BF16)
    wide[:, 2:10] = b.q
    for q in (b.q.clone(), wide[:, 2:10]):
        assert torch.equal(risa.paged_attention(q, b.cache, b.table, b.lengths, query_offsets=b.offsets, out=q), want) and torch.equal(q, want)
    assert (wide[:, :2] == 0).all() and (wide[:, 10:] == 0).all()


def test_attention_of_query_views():
    b = U.batch_of([50, 70], [7, 3], q_heads=4, kv_heads=2, head_dim=128, page=16)
    want = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets)
    wide = torch.zeros(10, 9, 136, device="cuda", dtype=BF16)
    wide[:, 2:6, :128] = b.q
    assert torch.equal(risa.paged_attention(wide[:, 2:6, :128], b.cache, b.table, b.lengths, query_offsets=b.offsets), want)
    heads_first = b.q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(risa.paged_attention(heads_first, b.cache, b.table, b.lengths, query_offsets=b.offsets), want)
    odd = torch.zeros(10, 4, 131, device="cuda", dtype=BF16)[..., 1:129]
    odd.copy_(b.q)
    assert torch.equal(risa.paged_attention(odd, b.cache, b.table, b.lengths, query_offsets=b.offsets), want)


def test_attention_of_many_sequences():
    lengths = [1 + (37 * i) % 90 for i in range(400)]
    b = U.batch_of(lengths, [1] * 400, q_heads=4, kv_heads=2, head_dim=64, page=16)
    out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, return_lse=True)
    U.assert_attention(b, out, lse)


@pytest.mark.parametrize("head_dim,page,quantized", [(256, 128, False), (256, 16, True), (256, 128, True), (64, 128, False), (128, 16, True)])
@pytest.mark.parametrize("window", [None, 50])
def test_chunks_of_other_shapes(head_dim, page, quantized, window):
    """Pages larger than a tile and smaller, a group of three heads, blocks of query rows that end anywhere."""
    b = U.batch_of([257, 64, 500, 129], [100, 64, 11, 43], q_heads=6, kv_heads=2, head_dim=head_dim, page=page, quantized=quantized, seed=head_dim)
    out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, window=window, return_lse=True)
    U.assert_attention(b, out, lse, window=window)
    assert_weights(b, risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=b.offsets, window=window), lse, window=window)


def test_many_sequences_of_chunks_and_single_tokens():
    lengths = [20 + (53 * i) % 150 for i in range(70)]
    chunks = [(1, 0, 9, 20, 3)[i % 5] for i in range(70)]
    b = U.batch_of(lengths, chunks, q_heads=8, kv_heads=2, head_dim=64, page=16)
    out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    U.assert_attention(b, out, lse)
    assert_weights(b, risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=b.offsets), lse)


def test_two_calls_at_once():
    batches = [U.batch_of([2000 + 300 * i, 90], [1 + 60 * i, 40], q_heads=8, kv_heads=2, head_dim=128, page=16, seed=i, quantized=i == 1) for i in range(2)]
    attend = lambda b: risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)  # noqa: E731
    want = [attend(b) for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for b, stream in zip(batches, streams):
            with torch.cuda.stream(stream):
                got.append(attend(b))
    torch.cuda.synchronize()
    for i, (out, lse) in enumerate(got):
        assert torch.equal(out, want[i % 2][0]) and torch.equal(lse, want[i % 2][1])


def test_attention_gives_the_same_bits_again_and_on_another_stream():
    b = U.batch_of([3000, 70, 900], [1, 60, 300], q_heads=8, kv_heads=2, head_dim=128, page=64)
    first = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        second = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    third = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    torch.cuda.synchronize()
    for x, y, z in zip(first, second, third):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_attention_in_a_graph_follows_lengths():
    b = U.batch_of([300, 200], [1, 4], q_heads=8, kv_heads=2, head_dim=128, page=16, extra_rows=100)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets)
    for lengths, offsets in (([300, 200], [0, 1, 5]), ([17, 1], [0, 1, 2]), ([299, 180], [0, 90, 105]), ([0, 30], [0, 0, 30])):
        b.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        b.offsets.copy_(torch.tensor(offsets, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets))


def test_attention_of_offsets_past_32_bits():
    """Pages whose first element lies more than 2^31 elements into the pool."""
    pages = 2 ** 31 // (2 * 128 * 128) + 40
    cache = risa.KeyValueCache(*(torch.empty(pages, 2, 128, 128, device="cuda", dtype=BF16) for _ in range(2)))
    g = torch.Generator("cuda").manual_seed(1)
    table = torch.tensor([[pages - 1, 0, pages - 7]], dtype=torch.int32, device="cuda")
    for x in (cache.keys, cache.values):
        x[table[0].long()] = torch.randn(3, 2, 128, 128, device="cuda", generator=g).to(BF16)
    for tokens in (1, 150):
        q = torch.randn(tokens, 4, 128, device="cuda", generator=g).to(BF16)
        b = U.Batch(cache, table, torch.tensor([380], dtype=torch.int32, device="cuda"), torch.tensor([0, tokens], dtype=torch.int32, device="cuda"), [tokens], q, 0)
        out, lse = risa.paged_attention(q, cache, table, b.lengths, query_offsets=b.offsets, return_lse=True)
        U.assert_attention(b, out, lse)


@pytest.mark.parametrize("chunk", [1, 50])
def test_attention_over_codes_of_any_scale(chunk):
    """Scales of values that differ by 2^60 or more within a sequence, zeros among them: what is rounded is relative to the
    largest contribution, and the sums hold."""
    b = U.batch_of([300], [chunk], q_heads=4, kv_heads=2, head_dim=128, page=16, quantized=True, seed=4)
    used = b.table[0].long()
    g = torch.Generator("cuda").manual_seed(0)
    scales = torch.pow(2.0, torch.randint(-30, 31, b.cache.value_scales[used].shape, device="cuda", generator=g).float())
    scales[0, :, 3:9] = 0
    if chunk > 1:  # there what is rounded is relative to the largest scale of a tile: below 2^-14 of it steps are 2^-24 of it
        scales = scales.clamp(2.0 ** -6, 2.0 ** 6)
    b.cache.value_scales[used] = scales
    out, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    U.assert_attention(b, out, lse)


@pytest.mark.parametrize("chunk", [1, 18])
def test_values_that_are_not_finite_leave_lse_and_other_heads(chunk):
    b = U.batch_of([40], [chunk], q_heads=4, kv_heads=2, head_dim=64, page=16, quantized=True)
    want, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
    for bad in (math.inf, math.nan):
        b.cache.value_scales[b.table[0, 1].long(), 0, 5] = bad
        out, same = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True)
        assert not torch.isfinite(out[:, :2]).any() and torch.equal(out[:, 2:], want[:, 2:])
        # the sum of two numbers of up to 16 each, one of them a logarithm of 32 bits
        assert ((same - lse).abs() <= 3 * 2.0 ** -23 * 16).all()


# ---- key weights ------------------------------------------------------------------------------------------------
def assert_weights(b, got, lse, previous=None, **options):
    """An exponent is off by the score's error (see assert_attention) and lse's, whose rounding is the input's own; a sum of
    n terms of one sign adds 2^-24 n at most."""
    want, size = U.weights(b, lse, **options)
    terms = max(b.chunks) * b.q.shape[1]
    score = size * b.q.shape[-1] * 2.0 ** -23 + 2.0 ** -20 * (1 + size)
    bound = want * (1.1 * score + terms * 2.0 ** -24)
    if previous is not None:
        want = want + previous.double()
        bound = bound + 2.0 ** -24 * want
    error = (got.double() - want).abs()
    assert (error <= bound + 1e-37).all(), f"{float((error / bound.clamp_min(1e-300)).max()):.2f} of the bound"


@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("heads", [(4, 2), (8, 1), (20, 1)])
@pytest.mark.parametrize("head_dim,page,dtype,quantized", [(64, 16, BF16, False), (64, 32, BF16, True), (128, 32, F16, False), (128, 128, BF16, True), (256, 64, F16, True), (256, 16, BF16, False)])
def test_key_weights(step, heads, head_dim, page, dtype, quantized):
    lengths, chunks = STEPS[step]
    b = U.batch_of(lengths, chunks, q_heads=heads[0], kv_heads=heads[1], head_dim=head_dim, page=page, dtype=dtype, quantized=quantized, seed=len(step))
    offsets = None if chunks == [1] * len(chunks) else b.offsets
    _, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=offsets, return_lse=True)
    got = risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=offsets)
    assert_weights(b, got, lse)
    g = torch.Generator("cuda").manual_seed(1)
    previous = torch.rand(got.shape, device="cuda", generator=g)
    assert_weights(b, risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=offsets, previous=previous), lse, previous)
    assert torch.equal(risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=offsets), got)


@pytest.mark.parametrize("options", [{"is_causal": False}, {"window": 1}, {"window": 40}, {"scale": -0.1}])
@pytest.mark.parametrize("step", ["single_tokens", "chunks", "long_chunk", "empty"])
def test_key_weights_masks(options, step):
    lengths, chunks = STEPS[step]
    b = U.batch_of(lengths, chunks, q_heads=8, kv_heads=2, head_dim=128, page=16, seed=5, extra_rows=2, width=25 + max(lengths) // 16)
    _, lse = risa.paged_attention(b.q, b.cache, b.table, b.lengths, query_offsets=b.offsets, return_lse=True, **options)
    got = risa.cached_key_weights(b.q, lse, b.cache, b.table, b.lengths, query_offsets=b.offsets, **options)
    assert_weights(b, got, lse, causal=options.get("is_causal", True), window=options.get("window"), scale=options.get("scale"))


# ---- eviction -----------------------------------------------------------------------------------------------------
def evict(b, weights, budget, recent):
    """Runs the call on fresh target pages; returns (result, target table)."""
    page = b.cache.page_size
    per = -(-budget // page)
    g = torch.Generator().manual_seed(6)
    first = b.cache.keys.shape[0]
    grown = []
    for x in b.cache.tensors:
        grown.append(None if x is None else torch.cat((x, torch.full((len(b.chunks) * per + 1, *x.shape[1:]), 9, dtype=x.dtype, device="cuda"))))
    cache = risa.KeyValueCache(*grown)
    target = (first + torch.randperm(len(b.chunks) * per, generator=g)).int().view(len(b.chunks), per).cuda()
    before = [None if x is None else x.clone() for x in cache.tensors]
    result = risa.evict_from_cache(cache, b.table, b.lengths, weights, target, budget=budget, recent=recent)
    lengths = b.lengths.tolist()
    for s, n in enumerate(lengths):
        count = min(n, budget)
        assert int(result.lengths[s]) == count
        for h in range(cache.keys.shape[1]):
            want = U.evicted(weights[s, h].tolist(), n, budget, recent)
            assert result.kept[s, h].tolist() == want + [-1] * (budget - count)
            kept = torch.tensor(want, dtype=torch.long, device="cuda")
            place = torch.arange(count, device="cuda")
            assert torch.equal(result.weights[s, h, :count], weights[s, h][kept]) or torch.isnan(weights[s, h][kept]).any()
            assert (result.weights[s, h, count:] == 0).all()
            for x, old in zip(cache.tensors, before):
                if x is None:
                    continue
                moved = x[target[s].long()[place // page], h, place % page]
                assert torch.equal(moved, old[b.table[s].long()[kept // page], h, kept % page])
                for j in range(count, per * page):  # what is behind the last stays as it was
                    assert (x[int(target[s, j // page]), h, j % page] == 9).all()
                    break
    for x, old in zip(cache.tensors, before):
        if x is not None:
            assert torch.equal(torch.nan_to_num(x[:first].float(), nan=5), torch.nan_to_num(old[:first].float(), nan=5))
            assert (x[-1] == 9).all()
    return cache, target, result


@pytest.mark.parametrize("lengths,budget,recent", [([200, 33, 5, 1], 32, 8), ([100], 1, 0), ([100], 1, 1), ([64, 65], 64, 64), ([0, 3], 2, 1), ([5000, 2100], 1000, 100),
                                                   ([333], 333, 3), ([70], 40, 0)])
@pytest.mark.parametrize("head_dim,page,dtype,quantized", [(64, 16, BF16, False), (128, 32, F16, False), (128, 16, BF16, True), (256, 64, BF16, True)])
@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
def test_eviction(lengths, budget, recent, head_dim, page, dtype, quantized, kind):
    b = U.batch_of(lengths, [0] * len(lengths), q_heads=2, kv_heads=2, head_dim=head_dim, page=page, dtype=dtype, quantized=quantized, stale=1.0, extra_rows=1)
    g = torch.Generator("cuda").manual_seed(budget)
    shape = (len(lengths), 2, b.table.shape[1] * page)
    weights = torch.exp(5 * torch.randn(shape, device="cuda", generator=g))
    if kind == "ties":
        weights = (weights * 2).round().clamp_max(3)
    if kind == "special":
        odd = torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, 1e-45, -1.0, 3e38], device="cuda")
        weights = torch.where(torch.rand(shape, device="cuda", generator=g) < 0.5, odd[torch.randint(0, 8, shape, device="cuda", generator=g)], weights)
    evict(b, weights, budget, recent)


def test_eviction_skips_pages_outside_the_pool():
    cache = risa.allocate_key_value_cache(4, 1, 16, 64)
    cache.keys.fill_(1)
    table = torch.tensor([[0, 9]], dtype=torch.int32, device="cuda")
    target = torch.tensor([[2, -1]], dtype=torch.int32, device="cuda")
    weights = torch.zeros(1, 1, 32, device="cuda")
    risa.evict_from_cache(cache, table, torch.tensor([32], dtype=torch.int32, device="cuda"), weights, target, budget=32)
    with pytest.raises(RuntimeError, match="outside the pool"):
        _backend._C.device_status()


# ---- together ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,quantized", [(BF16, False), (F16, True)])
def test_a_run(dtype, quantized):
    """Two requests: their prompts, weights of the prompts, eviction, further tokens; each step against the 64-bit forms on
    what the cache then holds."""
    g = torch.Generator("cuda").manual_seed(11)
    q_heads, kv_heads, d, page = 8, 2, 128, 16
    cache = risa.allocate_key_value_cache(40, kv_heads, page, d, dtype=torch.int8 if quantized else dtype)
    table = torch.randperm(24, generator=torch.Generator().manual_seed(0)).int().view(2, 12).cuda()
    rotary = risa.rotary_table(d)
    int32 = dict(dtype=torch.int32, device="cuda")
    chunks, lengths = [150, 70], torch.tensor([150, 70], **int32)
    offsets = torch.tensor([0, 150, 220], **int32)
    new = lambda n, h: torch.randn(n, h, d, device="cuda", generator=g).to(dtype)  # noqa: E731
    q = risa.append_to_cache(cache, new(220, kv_heads), new(220, kv_heads), table, lengths, query_offsets=offsets, q=new(220, q_heads), rotary=rotary)
    b = U.Batch(cache, table, lengths, offsets, chunks, q, 0)
    out, lse = risa.paged_attention(q, cache, table, lengths, query_offsets=offsets, return_lse=True)
    U.assert_attention(b, out, lse)
    weights = risa.cached_key_weights(q, lse, cache, table, lengths, query_offsets=offsets)
    # every query row gives one in all
    assert torch.allclose(weights.sum((1, 2)), torch.tensor([150.0, 70.0], device="cuda") * q_heads, rtol=1e-4)
    target = torch.arange(24, 34, **int32).view(2, 5)
    result = risa.evict_from_cache(cache, table, lengths, weights, target, budget=64, recent=16)
    assert result.lengths.tolist() == [64, 64]
    table, weights, lengths = target, result.weights, result.lengths
    for step in range(3):
        lengths = lengths + 1
        positions = torch.tensor([150 + step, 70 + step], device="cuda")
        q = risa.append_to_cache(cache, new(2, kv_heads), new(2, kv_heads), table, lengths, q=new(2, q_heads), rotary=rotary, positions=positions)
        b = U.Batch(cache, table, lengths, torch.arange(3, **int32), [1, 1], q, 0)
        out, lse = risa.paged_attention(q, cache, table, lengths, return_lse=True)
        U.assert_attention(b, out, lse)
        previous = weights
        weights = risa.cached_key_weights(q, lse, cache, table, lengths, previous=previous)
        assert_weights(b, weights, lse, previous)
