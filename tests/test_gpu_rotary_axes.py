"""Rotation by positions of several axes (time, height, width), alone and on the way into the cache, against 64 bits."""
import pytest
import serving_util as U
import torch
from test_gpu_serving import rotation_bound

import risaattention_b200 as risa
from risaattention_b200 import _backend

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def no_status():
    yield
    torch.cuda.synchronize()
    _backend._C.device_status()


def frequencies_of(table):
    """Radians per position: the table's own whole numbers, in 64 bits."""
    return [u % 2 ** 64 / 2 ** 64 * 2 * torch.pi for u in table.turns.tolist()]


def turned(x, positions, table, interleaved, sign=1):
    """positions [axes, ...] broadcast against x.shape[:-1]; one axis' pairs at a time, the others standing still."""
    out = torch.zeros_like(x, dtype=torch.float64)
    axes = table.axes.tolist()
    r = table.rotary_dim
    channel_axis = [axes[c // 2] if interleaved else axes[c % (r // 2)] for c in range(r)]
    for axis in range(table.axis_count):
        whole = U.turned(x, positions[axis].expand(x.shape[:-1]), frequencies_of(table), table.magnitude, interleaved, sign)
        mine = [c for c in range(r) if channel_axis[c] == axis]
        out[..., mine] = whole[..., mine]
    out[..., r:] = x[..., r:].double()
    return out


CASES = [
    # dtype, shape, sections, dealt, restart, interleaved, magnitude
    (BF16, (64, 32, 128), (16, 24, 24), False, False, False, 1.0),
    (F16, (1, 3, 64), (8, 12, 12), True, False, True, 1.0),
    (F32, (2, 5, 33, 128), (22, 21, 21), False, True, False, 1.25),
    (BF16, (3, 16, 70, 256), (1, 2, 3, 4, 5, 6, 7, 36), True, True, False, 1.0),
    (F32, (7, 2, 20), (3, 1), True, False, False, 1.0),     # ten pairs of twenty channels: one thread a pair
    (F16, (1, 1, 9, 24), (8,), False, False, True, 1.0),    # one axis, half of the channels stay
    (BF16, (2, 16, 1000, 64), (16, 16), False, False, False, 1.0),
]


@pytest.mark.parametrize("dtype,shape,sections,dealt,restart,interleaved,magnitude", CASES)
@pytest.mark.parametrize("positions64", [False, True])
def test_axes(dtype, shape, sections, dealt, restart, interleaved, magnitude, positions64):
    g = torch.Generator("cuda").manual_seed(11)
    x = torch.randn(shape, device="cuda", generator=g).to(dtype)
    table = risa.rotary_table(2 * sum(sections), sections=sections, dealt=dealt, restart=restart, magnitude=magnitude)
    tokens = shape[0] if len(shape) == 3 else shape[2]
    where = (len(sections), tokens) if len(shape) == 3 else (len(sections), shape[0], tokens)
    positions = torch.randint(-5, 200000, where, device="cuda", generator=g)
    positions = positions if positions64 else positions.int()
    spread = positions[..., None] if len(shape) == 3 else positions[:, :, None, :]
    for transposed in (False, True):
        out = risa.rotate_positions(x, positions, table, interleaved=interleaved, transposed=transposed)
        want = turned(x, spread, table, interleaved, -1 if transposed else 1)
        assert ((out.double() - want).abs() <= rotation_bound(x, want, magnitude)).all()
    # the same position on all axes is one axis' rotation, whichever way it is given
    same = positions[0, 0] if len(shape) == 4 else positions[0]
    plain = risa.RotaryTable(table.turns, table.magnitude)
    want = risa.rotate_positions(x, same, plain, interleaved=interleaved)
    assert torch.equal(risa.rotate_positions(x, same, table, interleaved=interleaved), want)
    assert torch.equal(risa.rotate_positions(x, same.expand(len(sections), tokens), table, interleaved=interleaved), want)


def test_views_strides_and_bytes_that_start_anywhere():
    g = torch.Generator("cuda").manual_seed(12)
    table = risa.rotary_table(64, sections=(8, 12, 12))
    x = torch.randn(2, 19, 6 * 128, device="cuda", generator=g).bfloat16().view(2, 19, 6, 128).transpose(1, 2)
    positions = torch.randint(0, 5000, (2, 19, 3), device="cuda", generator=g, dtype=torch.int32).movedim(-1, 0)  # axes innermost
    want = risa.rotate_positions(x.contiguous(), positions.contiguous(), table)
    assert torch.equal(risa.rotate_positions(x, positions, table), want)
    shifted = torch.empty(33, dtype=torch.uint8, device="cuda")[1:]
    shifted.copy_(table.axes)
    assert torch.equal(risa.rotate_positions(x, positions, risa.RotaryTable(table.turns, 1.0, shifted, 3)), want)
    risa.rotate_positions(x, positions, table, out=x)
    assert torch.equal(x, want)


def test_an_axis_that_is_not_there_counts_as_the_last():
    x = torch.randn(5, 2, 64, device="cuda")
    positions = torch.arange(10, device="cuda", dtype=torch.int32).view(2, 5)
    table = risa.rotary_table(64, sections=(16, 16))
    beyond = table.axes.clone()
    beyond[16:] = 255
    assert torch.equal(risa.rotate_positions(x, positions, risa.RotaryTable(table.turns, 1.0, beyond, 2)), risa.rotate_positions(x, positions, table))


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient(interleaved):
    g = torch.Generator("cuda").manual_seed(13)
    table = risa.rotary_table(16, sections=(2, 3, 3), dealt=True, magnitude=1.5)
    positions = torch.randint(0, 9000, (3, 2, 3), device="cuda", generator=g)
    x = torch.randn(2, 2, 3, 24, device="cuda", generator=g).requires_grad_()
    grad = torch.randn(x.shape, device="cuda", generator=g)
    got, = torch.autograd.grad(risa.rotate_positions(x, positions, table, interleaved=interleaved), x, grad)
    want = turned(grad, positions[:, :, None], table, interleaved, -1)
    assert ((got.double() - want).abs() <= rotation_bound(grad, want, 1.5)).all()
    # differences: the map is linear, so they are exact but for the two values' rounding (2^-24 of about 8 each)
    direction = torch.randn(x.shape, device="cuda", generator=g)
    f = lambda y: (risa.rotate_positions(y, positions, table, interleaved=interleaved).double() * grad.double()).sum()  # noqa: E731
    with torch.no_grad():
        difference = f(x + direction) - f(x - direction)
    slope = 2 * (got.double() * direction.double()).sum()
    assert abs(float(difference - slope)) <= 2 * x.numel() * 8 * 4 * 2.0 ** -22
    risa.rotate_positions(x, positions, table, interleaved=interleaved).sum().backward()  # an expanded gradient
    ones = turned(torch.ones_like(x), positions[:, :, None], table, interleaved, -1)
    assert ((x.grad.double() - ones).abs() <= rotation_bound(torch.ones_like(x), ones, 1.5)).all()
    v = grad.clone().requires_grad_()
    first, = torch.autograd.grad(risa.rotate_positions(x, positions, table, interleaved=interleaved), x, v, create_graph=True)
    second, = torch.autograd.grad(first, v, direction)
    with torch.no_grad():
        assert torch.equal(second, risa.rotate_positions(direction, positions, table, interleaved=interleaved))


def test_gradient_in_a_graph():
    table = risa.rotary_table(64, sections=(8, 12, 12))
    positions = torch.arange(120, device="cuda").view(3, 40)
    leaf = torch.randn(40, 3, 64, device="cuda").requires_grad_()
    grad = torch.randn_like(leaf)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want, = torch.autograd.grad(risa.rotate_positions(leaf, positions, table), leaf, grad)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured, = torch.autograd.grad(risa.rotate_positions(leaf, positions, table), leaf, grad)
    grad.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, 2 * want)


@pytest.mark.parametrize("dtype,quantized,interleaved", [(BF16, False, False), (F16, True, True)])
def test_append_turns_by_axes(dtype, quantized, interleaved):
    g = torch.Generator("cuda").manual_seed(14)
    b = U.batch_of([40, 17, 90], [40, 1, 33], q_heads=4, kv_heads=2, head_dim=128, page=16, dtype=dtype, quantized=quantized, stale=0.0)
    q, k, v = (torch.randn(74, h, 128, device="cuda", generator=g).to(dtype) for h in (4, 2, 2))
    table = risa.rotary_table(96, sections=(16, 16, 16), dealt=True)
    positions = torch.randint(0, 30000, (3, 74), device="cuda", generator=g)
    place = torch.cat([torch.arange(n - c, n) for n, c in zip([40, 17, 90], [40, 1, 33])]).cuda()
    page = torch.cat([b.table[s, p // 16].view(-1) for s, p in zip([0] * 40 + [1] + [2] * 33, place.tolist())]).long()

    def check(angles, **options):
        """Rotation as its bound has it; codes half a step and the scale's rounding further."""
        out = risa.append_to_cache(b.cache, k, v, b.table, b.lengths, query_offsets=b.offsets, q=q, rotary=table, interleaved=interleaved, **options)
        want = turned(q, angles[..., None], table, interleaved)
        assert bool(((out.double() - want).abs() <= rotation_bound(q, want, 1.0)).all())
        want = turned(k, angles[..., None], table, interleaved)
        got, slack = b.cache.keys[page, :, place % 16].double(), 0.0
        if quantized:
            scale = b.cache.key_scales[page, :, place % 16].double()[..., None]
            got, slack = got * scale, scale * (0.5 + 127 * 2.0 ** -22)
        assert bool(((got - want).abs() <= rotation_bound(k, want, 1.0) + slack).all())

    check(positions, positions=positions)
    check(positions[:1].expand(3, 74), positions=positions[0].contiguous().int())
    check(place.expand(3, 74))  # without positions every axis has the place
