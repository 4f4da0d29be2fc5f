"""More operators of language-model serving whose time is measured: a cache held in 4 bits, attention with a window and first tokens that stay visible,
positions with several axes, and the pages of a cache shared, handed out, given back and moved together.

Sequences, pages and steps are as in ``operators.py``.  Four bits of a cache: pages ``[pages, kv_heads, page_size, head_dim / 2]`` of bytes, and in
``[pages, kv_heads, page_size * (1 + head_dim / 16)]`` bytes first the scale of each token of the page, a power of two as the exponent of a 32-bit number
(0: a scale of zero), then for each token one e4m3 scale for each 16 of its channels.  A value is code * group scale * token scale with codes -7..7; those
of channels ``8 w .. 8 w + 7`` lie in the 32-bit word ``w`` of a row as ``code + 8``, channel ``8 w + 2 i + j`` in bits ``16 j + 4 i``.  The families:

``rotate``   queries rotated by positions of several axes; with ``train`` also the gradient
``append``   one step's queries and keys rotated, keys and values written in 4 bits; what was stored is read back
``attend``   the new tokens' attention over the cached keys; with ``window`` over the last ones and the first ``sinks``
``fork``     sequences shared by several children that grow (pages they must not share are copied) and are given up again
``compact``  the pages in use copied together to the front of another pool
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BASE = 10000.0
DEFAULTS = {"head_dim": 128, "dtype": "bf16", "page": 16, "bits": 16, "batch": 1, "chunk": 1, "window": 0, "sinks": 0, "interleaved": False,
            "dealt": False, "restart": False}
SECTIONS = {3: (1 / 4, 3 / 8, 3 / 8), 2: (1 / 2, 1 / 2), 4: (1 / 4, 1 / 4, 1 / 4, 1 / 4)}  # shares of the pairs that follow each axis


def _case(family, name=None, **more):
    case = {"family": family, **DEFAULTS, **more}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # The queries of one generation step of 64 requests of a model that sees images: time, height and width.
        _case("rotate", "rotate_axes_step_b64", layout="tokens", q_heads=32, length=64, rotary_dim=128, axes=3, dealt=True),
        # A training pass of a video model: each axis has frequencies of its own, with the gradient.
        _case("rotate", "rotate_axes_train_16k", layout="hnd", q_heads=16, length=16384, batch=2, rotary_dim=128, axes=3, restart=True, train=True),
        # One generation step of 64 requests: one token of each goes into the cache.
        _case("append", "append_step_b64_4bit", q_heads=32, kv_heads=8, batch=64, length=4096, rotary_dim=128, axes=1, bits=4, dtype="f16"),
        # Prompts of ragged length with images in them, 8192 tokens together.
        _case("append", "append_prompts_8k_4bit", q_heads=32, kv_heads=8, batch=5, chunk=2720, length=2720, rotary_dim=128, axes=3, bits=4),
        # A single request in conversation: one token, time is latency.
        _case("attend", "attend_step_b1_8k_4bit", q_heads=16, kv_heads=4, length=8192, page=64, bits=4),
        # A full server: 32 requests of ragged length up to 32K keys.
        _case("attend", "attend_step_b32_32k_4bit", q_heads=32, kv_heads=8, batch=32, length=32768, bits=4),
        # Endless conversations: 64 requests that see their last 4096 keys and the first four.
        _case("attend", "attend_sinks_step_b64_32k", q_heads=32, kv_heads=8, batch=64, length=32768, window=4096, sinks=4),
        # 1024 tokens of a long prompt that is taken in with a window.
        _case("attend", "attend_sinks_chunk_1k_of_32k_4bit", q_heads=32, kv_heads=8, chunk=1024, length=32768, page=64, bits=4, window=8192, sinks=64),
        # Four prompts from which four answers each are drawn.
        _case("fork", "fork_b4_x4", kv_heads=8, batch=4, children=4, length=2023, grow=1, dtype="f16"),
        # Beams of 64 long requests, four tokens ahead.
        _case("fork", "fork_b64_x4_8k", kv_heads=8, batch=64, children=4, length=8192, grow=4, page=32),
        # A small server's pool after most requests have left.
        _case("compact", "compact_b4_4k", kv_heads=8, batch=4, length=4096, spare=3.0, dtype="f16"),
        # A large one, half empty.
        _case("compact", "compact_b32_8k", kv_heads=8, batch=32, length=8192, spare=1.0, page=64),
    ]


def draw(rng):
    most_flops = max(work(c)["flops"] for c in listed())
    most_bytes = max(work(c)["bytes"] for c in listed())

    def spread(low, high):
        return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))

    while True:
        family = rng.choice(("rotate", "rotate", "append", "append", "attend", "attend", "attend", "attend", "fork", "compact"))
        q_heads, kv_heads = rng.choice(((16, 4), (16, 16), (32, 8), (40, 40), (8, 1)))
        head_dim, dtype, page = rng.choice((64, 128, 128, 128, 256)), rng.choice(("bf16", "bf16", "f16")), rng.choice((16, 16, 32, 64, 128))
        if family == "rotate":
            case = _case(family, layout=rng.choice(("tokens", "hnd")), q_heads=q_heads, length=spread(1, 32768), head_dim=head_dim,
                         rotary_dim=rng.choice((head_dim, head_dim, head_dim // 2)), interleaved=rng.random() < 0.5, dtype=rng.choice(("bf16", "f16", "f32")),
                         axes=rng.choice((2, 3, 3, 4)), dealt=rng.random() < 0.5, restart=rng.random() < 0.5, train=rng.random() < 0.5)
            if case["layout"] == "hnd":
                case["batch"] = rng.choice((1, 2, 4))
        else:
            case = _case(family, kv_heads=kv_heads, batch=spread(1, 64), length=spread(64, 32768), head_dim=head_dim, dtype=dtype, page=page)
            if family == "fork":
                case.update(children=rng.choice((1, 2, 3, 4, 8)), grow=spread(1, 256))
            elif family == "compact":
                case["spare"] = round(rng.uniform(0.1, 4.0), 2)
            else:
                case["q_heads"] = q_heads
                case["chunk"] = 1 if rng.random() < 0.4 else spread(2, min(2048, case["length"]))
            if family == "append":
                case.update(bits=4, rotary_dim=rng.choice((head_dim, head_dim // 2)), interleaved=rng.random() < 0.3, axes=rng.choice((1, 3)))
            if family == "attend":
                case["bits"] = rng.choice((4, 4, 8, 16))
                if case["bits"] != 4 or rng.random() < 0.4:
                    case["window"], case["sinks"] = spread(16, case["length"]), spread(1, 256)
        # what the plain form holds at once: scores of padded chunks, the gathered cache in 32 bits, a pool and its copies
        plain = 0
        if family == "attend":
            plain = 4 * case["batch"] * case["length"] * (3 * q_heads * case["chunk"] + 4 * kv_heads * head_dim)
        elif family == "append":
            plain = 8 * case["batch"] * case["length"] * kv_heads * head_dim
        elif family == "fork":
            plain = 8 * case["batch"] * (case["length"] + case["children"] * (case["grow"] + 2 * page)) * kv_heads * head_dim
        elif family == "compact":
            plain = 12 * case["batch"] * case["length"] * kv_heads * head_dim * (1 + case["spare"])
        w = work(case)
        if w["flops"] <= most_flops and w["bytes"] <= most_bytes and plain <= 26e9:
            return case


# ---- what the cases' sequences look like: the same for every seed, in another order -----------------------------------------
def _lengths(case):
    """Cached tokens of each sequence, the new ones among them: spread evenly from a quarter of the longest to the longest."""
    b, n = case["batch"], case["length"]
    return [max(1, round(n * (1.0 if b == 1 else 0.25 + 0.75 * i / (b - 1)))) for i in range(b)]


def _chunks(case):
    """New tokens of each sequence: one each, or for chunks half of the sequences one and the others from half of a chunk to a whole one."""
    b, n = case["batch"], case["chunk"]
    if n == 1 or b == 1:
        return [n] * b
    if case["family"] == "append":
        return [min(length, round(n * (0.2 + 0.8 * i / (b - 1)))) or 1 for i, length in enumerate(_lengths(case))]
    return [1 if i % 2 == 0 else max(1, min(length, round(n * (0.5 + 0.5 * i / (b - 1))))) for i, length in enumerate(_lengths(case))]


def _sections(case):
    """Pairs that follow each axis."""
    pairs = case["rotary_dim"] // 2
    if case["axes"] == 1:
        return (pairs,)
    out = [round(pairs * share) for share in SECTIONS[case["axes"]][1:]]
    return (pairs - sum(out), *out)


def _pairs(case):
    """(frequency, axis) of each pair: one section behind the other, or dealt out in turn while the sections last; the frequencies go on
    through all the pairs, or start again with each section."""
    sections = _sections(case)
    if case["dealt"]:
        axes, left = [], list(sections)
        while len(axes) < sum(sections):
            for axis in range(len(sections)):
                if left[axis]:
                    left[axis] -= 1
                    axes.append(axis)
    else:
        axes = [axis for axis, n in enumerate(sections) for _ in range(n)]
    if not case["restart"]:
        return [BASE ** (-i / len(axes)) for i in range(len(axes))], axes
    seen, frequencies = [0] * len(sections), []
    for axis in axes:
        frequencies.append(BASE ** (-seen[axis] / sections[axis]))
        seen[axis] += 1
    return frequencies, axes


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _grid_positions(axes, shape, g):
    """Positions as a text with images gives them: whole rows, columns and frames of a grid behind a place of its own."""
    n = shape[-1]
    place = torch.arange(n, device="cuda")
    side = max(1, round(n ** 0.5 / 2))
    start = torch.randint(0, 65536, (*shape[:-1], 1), device="cuda", generator=g)
    frame, row, column = place // (side * side), place // side % side, place % side
    return torch.stack([start + step for step in {2: (row, column), 3: (frame, row, column), 4: (frame, row, column, place)}[axes]]).int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, d = DTYPES[case["dtype"]], case["head_dim"]

    def normal(*shape, type=dtype):
        return torch.randn(*shape, device="cuda", generator=g).to(type)

    state = {"case": case}
    if "rotary_dim" in case:
        frequencies, axes = _pairs(case)
        state["frequencies"] = torch.tensor(frequencies, dtype=torch.float64, device="cuda")
        state["axes"] = torch.tensor(axes, device="cuda")
        if own:
            import risaattention_b200 as risa
            more = {} if case["axes"] == 1 else {"sections": _sections(case), "dealt": case["dealt"], "restart": case["restart"]}
            state["rotary"] = risa.rotary_table(case["rotary_dim"], base=BASE, device="cuda", **more)
    if case["family"] == "rotate":
        n, heads, batch = case["length"], case["q_heads"], case["batch"]
        if case["layout"] == "tokens":
            x = normal(n, heads, d)
            positions = torch.randint(0, 131072, (case["axes"], n), device="cuda", generator=g, dtype=torch.int32)
        else:
            x = normal(batch, heads, n, d)
            positions = _grid_positions(case["axes"], (batch, n), g)
        state.update(x=x, positions=positions)
        if case.get("train"):
            state["x"].requires_grad_()
            state["grad"] = normal(*x.shape)
        return state

    family, kv_heads, page, batch = case["family"], case["kv_heads"], case["page"], case["batch"]
    order = torch.randperm(batch, generator=torch.Generator().manual_seed(seed)).tolist()
    lengths, chunks = [_lengths(case)[i] for i in order], [_chunks(case)[i] for i in order]
    counts = [-(-n // page) for n in lengths]
    used = sum(counts)
    # room for what the children need of their own, or what stands empty between the pages in use
    if family == "fork":
        pages = used + sum(case["children"] * (-(-(n + case["grow"]) // page) - n // page) for n in lengths)
    else:
        pages = used + math.ceil(used * case.get("spare", 0.0))
    ids = torch.randperm(pages, device="cuda", generator=g)[:used].int()
    table = torch.full((batch, max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = ids[at:at + n]
        at += n
    shape = (pages, kv_heads, page, d)
    if case["bits"] == 4:
        codes = [torch.randint(-7, 8, shape, device="cuda", generator=g, dtype=torch.int8) for _ in range(2)]
        # codes that fill their range have a deviation of 4.3 steps; the largest group scale of a row lies between 224 and 448, and rows differ
        groups = [(448 * (0.2 + 0.8 * torch.rand(*shape[:3], d // 16, device="cuda", generator=g))).to(torch.float8_e4m3fn) for _ in range(2)]
        tokens = [torch.randint(127 - 12, 127 - 9, shape[:3], device="cuda", generator=g, dtype=torch.uint8) for _ in range(2)]
        keys, values = (_packed_codes(c) for c in codes)
        scales = [_packed_scales(t, s) for t, s in zip(tokens, groups)]
    elif case["bits"] == 8:
        keys, values = (torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8) for _ in range(2))
        scales = [(torch.rand(shape[:3], device="cuda", generator=g) + 0.5) / 73.0 for _ in range(2)]
    else:
        keys, values, scales = normal(*shape), normal(*shape), [None, None]
    offsets = torch.tensor([0] + chunks).cumsum(0).int()
    tokens = int(offsets[-1])
    state.update(keys=keys, values=values, key_scales=scales[0], value_scales=scales[1], table=table,
                 lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), offsets=offsets.cuda(), most=max(chunks), tokens=tokens)
    if family in ("fork", "compact"):
        references = torch.zeros(pages, dtype=torch.int32, device="cuda")
        references[ids.long()] = 1
        state["references"] = references
        if family == "fork":
            parents = torch.arange(batch, device="cuda", dtype=torch.int32).repeat_interleave(case["children"])
            state["parents"] = parents[torch.randperm(len(parents), device="cuda", generator=g)]
            # the table has columns for what the children will hold
            wide = max(-(-(n + case["grow"]) // page) for n in lengths)
            state["table"] = torch.nn.functional.pad(table, (0, wide - table.shape[1]), value=-1).contiguous()
        else:
            state["target"] = [torch.zeros(used, kv_heads, page, d, dtype=dtype, device="cuda") for _ in range(2)]
    else:
        state["q"] = normal(tokens, case["q_heads"], d)
        if family == "append":
            state["k"], state["v"] = normal(tokens, kv_heads, d), normal(tokens, kv_heads, d)
            if case["axes"] > 1:
                state["positions"] = _grid_positions(case["axes"], (tokens,), g)
    if own:
        import risaattention_b200 as risa
        state["cache"] = risa.KeyValueCache(keys, values, *scales)
        if family == "compact":
            state["target_cache"] = risa.KeyValueCache(*state["target"])
    return state


# ---- four bits ----------------------------------------------------------------------------------------------------------------
def _packed_codes(codes):
    """int8 codes [..., channels] as bytes [..., channels / 2]."""
    u = (codes.int() + 8).unflatten(-1, (-1, 4, 2))
    shifts = torch.tensor([[0, 16], [4, 20], [8, 24], [12, 28]], device=codes.device)
    words = (u.long() << shifts).sum((-1, -2))
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int()
    return words.view(torch.uint8)


def _unpacked_codes(data):
    """32-bit floats [..., channels] of bytes [..., channels / 2]."""
    words = data.contiguous().view(torch.int32)
    shifts = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=data.device, dtype=torch.int32)
    return ((words[..., None] >> shifts) & 15).sub_(8).flatten(-2).float()


def _packed_scales(tokens, groups):
    """Exponents [pages, heads, page] and scales [pages, heads, page, groups] (e4m3) as bytes [pages, heads, ...]."""
    return torch.cat((tokens, groups.view(torch.uint8).flatten(-2)), -1)


def _power(exponents):
    return torch.where(exponents > 0, torch.exp2(exponents.float() - 127.0), 0.0)


def _scales_of(data, page):
    groups = data[..., page:].contiguous().view(torch.float8_e4m3fn).float()
    return _power(data[..., :page]), groups.unflatten(-1, (page, -1))


def _quantized(x):
    """Codes, group scales (e4m3) and token scales (exponents) of rows x, all in 64 bits: a value next to a border goes to its own side."""
    most = x.abs().amax(-1)
    # the smallest power of two of which the row's largest value is at most 7 * 448
    fraction, exponent = torch.frexp(most / 3136.0)
    exponent = (exponent - (fraction == 0.5).int()).clamp_min(-126)
    token = torch.where(most > 0, torch.exp2(exponent.double()), 0.0)[..., None]
    grouped = x.unflatten(-1, (-1, 16))
    ratio = torch.where(token > 0, grouped.abs().amax(-1) / (7.0 * token), 0.0)
    # three bits behind the point from 2^-6 on, steps of 2^-9 below
    step = torch.exp2((torch.frexp(ratio).exponent - 1).clamp_min(-6).double() - 3.0)
    group = (ratio / step).round() * step
    size = (token * group)[..., None]
    codes = torch.where(size > 0, grouped / size, 0.0).round().clamp(-7, 7)
    return codes.flatten(-2), group.float().to(torch.float8_e4m3fn), torch.where(most > 0, exponent + 127, 0).to(torch.uint8)


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _turned(x, angles, interleaved, transposed=False):
    """x [..., tokens, channels] with its first 2 * angles.shape[-1] channels rotated by angles [..., tokens, pairs] (64 bits), in the type of x."""
    cos, sin = angles.cos().to(x.dtype), angles.sin().to(x.dtype)
    sin = -sin if transposed else sin
    r = 2 * cos.shape[-1]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    first, second = a * cos - b * sin, b * cos + a * sin
    both = torch.stack((first, second), -1).flatten(-2) if interleaved else torch.cat((first, second), -1)
    return torch.cat((both, x[..., r:]), -1)


def _sequences(state):
    """(sequence, place in its chunk, place in the cache) of every new token."""
    token = torch.arange(state["tokens"], device="cuda")
    s = torch.searchsorted(state["offsets"][1:], token, right=True)
    i = token - state["offsets"][s]
    n = state["offsets"][1:] - state["offsets"][:-1]
    return s, i, state["lengths"][s] - n[s] + i


def _cached(state, what):
    """Keys or values of every sequence in 32 bits: [batch, kv_heads, keys, head_dim]."""
    case, table = state["case"], state["table"].clamp_min(0).long()
    data = state[what][table]
    if case["bits"] == 4:
        tokens, groups = _scales_of(state[what[:-1] + "_scales"][table], case["page"])
        pages = (_unpacked_codes(data).unflatten(-1, (-1, 16)) * groups[..., None]).flatten(-2) * tokens[..., None]
    elif case["bits"] == 8:
        pages = data.float() * state[what[:-1] + "_scales"][table][..., None]
    else:
        pages = data.float()
    return pages.transpose(1, 2).flatten(2, 3)


def _attend(state):
    case = state["case"]
    s, i, place = _sequences(state)
    batch, kv_heads, d = case["batch"], case["kv_heads"], case["head_dim"]
    group = case["q_heads"] // kv_heads
    q = torch.zeros(batch, state["most"], case["q_heads"], d, device="cuda")
    q[s, i] = state["q"].float() * d ** -0.5
    position = torch.full((batch, state["most"]), -1, device="cuda")
    position[s, i] = place.long()
    q = q.view(batch, -1, kv_heads, group, d).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = (q @ _cached(state, "keys").transpose(-1, -2)).view(batch, kv_heads, group, state["most"], -1)
    key = torch.arange(scores.shape[-1], device="cuda")
    hidden = key > position[..., None]
    if case["window"]:
        hidden |= (key <= position[..., None] - case["window"]) & (key >= case["sinks"])
    scores.masked_fill_(hidden[:, None, None], -torch.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)  # rows that see nothing
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = (scores.flatten(2, 3) @ _cached(state, "values")).view(*scores.shape[:-1], -1) / total.clamp_min(1e-30)
    out, lse = (x.movedim(3, 1).flatten(2, 3)[s, i] for x in (out, (total.log() + top).squeeze(-1)))
    return out.to(state["q"].dtype), lse


def _append(state):
    case = state["case"]
    s, _, place = _sequences(state)
    page, slot = state["table"][s, place // case["page"]].long(), (place % case["page"]).long()
    position = state["positions"][state["axes"]].T if "positions" in state else place[:, None]  # [tokens, pairs], or one for all of them
    angles = (position.double() * state["frequencies"])[:, None]
    q = _turned(state["q"].float(), angles, case["interleaved"]).to(state["q"].dtype)
    out = [q]
    for what, x in (("keys", _turned(state["k"].double(), angles, case["interleaved"])), ("values", state["v"].double())):
        codes, groups, tokens = _quantized(x)
        state[what][page, :, slot] = _packed_codes(codes.to(torch.int8))
        n = case["page"]
        token_scales, group_scales = state[what[:-1] + "_scales"].split((n, n * case["head_dim"] // 16), -1)
        group_scales = group_scales.unflatten(-1, (n, -1))
        token_scales[page, :, slot], group_scales[page, :, slot] = tokens, groups.view(torch.uint8)
        # read back from where they lie
        codes = _unpacked_codes(state[what][page, :, slot])
        groups = group_scales[page, :, slot].view(torch.float8_e4m3fn).float()
        out.append(((codes.unflatten(-1, (-1, 16)) * groups[..., None]).flatten(-2) * _power(token_scales[page, :, slot])[..., None]).to(q.dtype))
    return tuple(out)


def _fork(state):
    """Children of every sequence, grown, and given up."""
    case, page = state["case"], state["case"]["page"]
    references, width = state["references"], state["table"].shape[1]
    parent = state["parents"].long()
    table, lengths = state["table"][parent], state["lengths"][parent].long()
    column = torch.arange(width, device="cuda")
    held = column < ((lengths + page - 1) // page)[:, None]
    table = torch.where(held, table, -1)
    references.index_add_(0, table[held].long(), torch.ones_like(table[held]))
    # growth: a last page that is shared and not full is replaced by a copy, and new pages follow; the lowest free ones, in the order of the children
    grown = lengths + case["grow"]
    last = ((lengths - 1).clamp_min(0) // page)[:, None]
    copied = (lengths % page != 0) & (references[table.gather(1, last)[:, 0].long()] > 1)
    wanted = (column >= ((lengths + page - 1) // page)[:, None]) & (column < ((grown + page - 1) // page)[:, None])
    wanted |= copied[:, None] & (column == last)
    free = (references == 0).nonzero()[:, 0].int()
    was = table.clone()
    child, at = wanted.nonzero(as_tuple=True)  # in the order of the children, then of their columns
    fresh = free[:len(child)]
    table[child, at] = fresh
    references[fresh.long()] = 1
    rows = copied.nonzero()[:, 0]
    old, new = was.gather(1, last)[rows, 0].long(), table.gather(1, last)[rows, 0].long()
    references.index_add_(0, old, -torch.ones_like(old, dtype=torch.int32))
    there = (torch.arange(page, device="cuda") < (lengths[rows] % page)[:, None])[:, None, :, None]
    for pool in (state["keys"], state["values"]):
        pool[new] = torch.where(there, pool[old], pool[new])
    now = references.clone()
    kept = table.clone()
    held = column < ((grown + page - 1) // page)[:, None]
    references.index_add_(0, table[held].long(), -torch.ones_like(table[held]))
    return kept, grown.int(), now, references, state["keys"], state["values"]


def _compact(state):
    references, table, page = state["references"], state["table"], state["case"]["page"]
    in_use = references > 0
    place = (in_use.cumsum(0) - 1).int()
    held = torch.arange(table.shape[1], device="cuda") < ((state["lengths"] + page - 1) // page)[:, None]
    new = torch.where(held, place[table.clamp_min(0).long()], -1)
    old = in_use.nonzero()[:, 0]
    for target, source in zip(state["target"], ("keys", "values")):
        target[:len(old)] = state[source][old]
    moved = torch.zeros(state["target"][0].shape[0], dtype=torch.int32, device="cuda")
    moved[:len(old)] = references[old]
    return new, moved, *state["target"]


def run(state):
    case, family = state["case"], state["case"]["family"]
    if own:
        import risaattention_b200 as risa
    if family == "rotate":
        x, train = state["x"], case.get("train")
        if own:
            out = risa.rotate_positions(x, state["positions"], state["rotary"], interleaved=case["interleaved"])
            return (out.detach(), torch.autograd.grad(out, x, state["grad"])[0]) if train else out
        angles = state["positions"][state["axes"]].movedim(0, -1).double() * state["frequencies"]
        angles = angles[:, None]  # [tokens, 1, pairs] beside [tokens, heads, channels], [batch, 1, tokens, pairs] beside [batch, heads, tokens, channels]
        out = _turned(x.detach().float(), angles, case["interleaved"]).to(x.dtype)
        return (out, _turned(state["grad"].float(), angles, case["interleaved"], True).to(x.dtype)) if train else out
    if not own:
        return {"append": _append, "attend": _attend, "fork": _fork, "compact": _compact}[family](state)
    cache, table, lengths = state["cache"], state["table"], state["lengths"]
    # a step of one token for each sequence needs no offsets
    offsets = state["offsets"] if state["most"] > 1 else None
    if family == "append":
        q = risa.append_to_cache(cache, state["k"], state["v"], table, lengths, query_offsets=offsets, q=state["q"], rotary=state["rotary"],
                                 positions=state.get("positions"), interleaved=case["interleaved"])
        return q, *risa.read_from_cache(cache, table, lengths, query_offsets=offsets, tokens=state["tokens"], dtype=q.dtype)
    if family == "attend":
        return risa.paged_attention(state["q"], cache, table, lengths, query_offsets=offsets, window=case["window"] or None, sinks=case["sinks"], return_lse=True)
    references = state["references"]
    if family == "fork":
        children, lengths = risa.fork_sequences(cache, references, table, lengths, state["parents"])
        grown = risa.resize_sequences(cache, references, children, lengths, lengths + case["grow"])
        now, kept = references.clone(), children.clone()
        risa.resize_sequences(cache, references, children, grown, torch.zeros_like(grown))
        return kept, grown, now, references, state["keys"], state["values"]
    new, moved, _ = risa.compact_cache(cache, references, table, lengths, state["target_cache"])
    return new, moved, *state["target"]


def work(case):
    """Inputs read once and outputs written once; two operations per multiply-add of a visible (query, key, channel)."""
    size, d = 4 if case["dtype"] == "f32" else 2, case["head_dim"]
    if case["family"] == "rotate":
        values = case["batch"] * case["q_heads"] * case["length"] * d
        positions = case["axes"] * case["batch"] * case["length"]
        passes = 2 if case.get("train") else 1
        return {"bytes": passes * (2 * values * size) + 4 * positions + 6 * case["rotary_dim"], "flops": passes * 3 * values * case["rotary_dim"] / d}
    lengths, kv_heads, page = _lengths(case), case["kv_heads"], case["page"]
    counts = [-(-n // page) for n in lengths]
    row = {4: d // 2 + 1 + d // 16, 8: d + 4, 16: 2 * d}[case["bits"]]  # one token of one head in the cache
    if case["family"] == "compact":
        return {"bytes": sum(counts) * (4 * kv_heads * page * row + 8 + 4) + 4 * math.ceil(sum(counts) * (1 + case["spare"])), "flops": sum(counts)}
    if case["family"] == "fork":
        children, grown = case["children"], [-(-(n + case["grow"]) // page) for n in lengths]
        copied = children * sum(n % page for n in lengths)
        # entries read from the parents and written for the children; the references of the pages in use, and of those handed out, read, written and reported
        return {"bytes": copied * 4 * kv_heads * row + 4 * sum(counts) + 8 * children * sum(grown) + 16 * (sum(counts) + children * sum(g - c + 1 for g, c in zip(grown, counts))),
                "flops": 3 * children * sum(grown)}
    chunks, window, sinks = _chunks(case), case["window"], case["sinks"]
    tokens, q_heads = sum(chunks), case["q_heads"]
    table = 4 * sum(counts)
    if case["family"] == "append":
        # queries in and out, keys and values in, stored, read back and returned
        moved = tokens * (2 * q_heads * d * size + 2 * kv_heads * (2 * d * size + 2 * row))
        return {"bytes": moved, "flops": 3 * tokens * (q_heads + kv_heads) * case["rotary_dim"]}
    pairs = keys = 0
    for n, c in zip(lengths, chunks):
        seen = [n - c + i + 1 for i in range(c)]
        if window:
            seen = [min(p, window + min(sinks, max(0, p - window))) for p in seen]
            table += 4 * (min(n, window + c - 1 + sinks) // page - n // page)
        pairs += q_heads * sum(seen)
        keys += kv_heads * (n if not window else min(n, window + c - 1 + sinks))
    return {"bytes": 2 * keys * row + tokens * q_heads * (2 * d * size + 4) + table, "flops": 4 * pairs * d}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["family"] == "fork":
        return None, None, None, None, *_exact_fork(state)
    if case["family"] == "compact":
        used = sorted({p for row in state["table"].tolist() for p in row if p >= 0})
        return None, None, *(torch.stack([state[what][p] for p in used]).double() for what in ("keys", "values"))
    if case["family"] == "rotate":
        out = _exact_rotation(state["x"].detach(), state["positions"], state, 1)
        return (out, _exact_rotation(state["grad"], state["positions"], state, -1)) if case.get("train") else out
    offsets, lengths = state["offsets"].tolist(), state["lengths"].tolist()
    if case["family"] == "append":
        place = torch.cat([torch.arange(n - (b - a), n, device="cuda") for n, a, b in zip(lengths, offsets, offsets[1:])])
        positions = state["positions"] if "positions" in state else place[None]
        return (_exact_rotation(state["q"], positions, state, 1), _nearest(_exact_rotation(state["k"], positions, state, 1)), _nearest(state["v"].double()))
    d, group, page = case["head_dim"], case["q_heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(state["q"].shape[:2], dtype=torch.float64, device="cuda")
    for s, n in enumerate(lengths):
        rows = slice(offsets[s], offsets[s + 1])
        pages = state["table"][s, :-(-n // page)].long()
        position = torch.arange(n - (offsets[s + 1] - offsets[s]), n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        seen = key <= position
        if case["window"]:
            seen &= (position - key < case["window"]) | (key < case["sinks"])
        for h in range(case["kv_heads"]):
            k, v = (_exact_rows(state, w, pages, h)[:n] for w in ("keys", "values"))
            for head in range(h * group, (h + 1) * group):
                x = state["q"][rows, head].double() @ k.T / math.sqrt(d)
                x[~seen] = -torch.inf
                lse[rows, head] = x.logsumexp(-1)
                out[rows, head] = (x - lse[rows, head][:, None]).exp() @ v
    return out, lse


def _exact_rows(state, what, pages, head):
    case, data = state["case"], state[what][pages, head]
    if case["bits"] == 16:
        return data.double().flatten(0, 1)
    scales = state[what[:-1] + "_scales"][pages, head]
    if case["bits"] == 8:
        return (data.double() * scales.double()[..., None]).flatten(0, 1)
    n, d = case["page"], case["head_dim"]
    words = data.view(torch.int32).long()
    rows = torch.zeros(*data.shape[:2], d, dtype=torch.float64, device="cuda")
    for j in range(2):
        for i in range(4):
            rows[..., 2 * i + j::8] = ((words >> (16 * j + 4 * i)) % 16 - 8).double()
    rows *= scales[:, n:].reshape(-1, n, d // 16).view(torch.float8_e4m3fn).double().repeat_interleave(16, -1)
    rows *= 2.0 ** (scales[:, :n].double() - 127)[..., None]
    return rows.flatten(0, 1)


def _nearest(x):
    """What a row becomes in 4 bits: the nearest of 15 steps up to a group's scale, which is the nearest of the numbers that a table of e4m3 holds
    in units of the token's power of two."""
    table = torch.tensor([m / 8 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8) if (e, m) != (8, 7)],
                         dtype=torch.float64, device="cuda")
    y = x.unflatten(-1, (-1, 16))
    most = x.abs().amax(-1)
    token = torch.full_like(most, 2.0 ** -126)
    for e in range(-125, 20):
        token = torch.where(most > 3136 * 2.0 ** (e - 1), 2.0 ** e, token)
    token = token[..., None, None]
    size = y.abs().amax(-1, keepdim=True) / 7 / token
    above = torch.searchsorted(table, size.contiguous()).clamp(1, len(table) - 1)
    low, high = table[above - 1], table[above]
    up = (high - size < size - low) | ((high - size == size - low) & (above % 2 == 0))  # at ties the one whose last bit is 0
    scale = torch.where(up, high, low) * token
    steps = torch.floor(y / scale + 0.5)
    steps = torch.where((steps - y / scale == 0.5) & (steps % 2 != 0), steps - 1, steps)
    return torch.where(scale > 0, steps.clamp(-7, 7) * scale, 0.0).flatten(-2)


def _exact_fork(state):
    """The pools after the children have grown: pages counted and copied one by one."""
    case, page = state["case"], state["case"]["page"]
    table, lengths, references = state["table"].tolist(), state["lengths"].tolist(), state["references"].tolist()
    pools = [state[what].double() for what in ("keys", "values")]
    free = (p for p, n in enumerate(references) if n == 0)
    for parent in state["parents"].tolist():
        full, rest = divmod(lengths[parent], page)
        if rest:
            new = next(free)
            for pool in pools:
                pool[new, :, :rest] = pool[table[parent][full], :, :rest]
        for _ in range(-(-(lengths[parent] + case["grow"]) // page) - full - (rest > 0)):
            next(free)
    return pools


def _exact_rotation(x, positions, state, sign):
    """Each pair as a complex number, times e^(i angle); positions [axes, ..., tokens]."""
    case = state["case"]
    r = case["rotary_dim"]
    y = x.double().clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    angle = torch.stack([positions[axis].double() * f * sign for axis, f in zip(state["axes"].tolist(), state["frequencies"].tolist())], -1)
    angle = angle[:, None]  # one for all heads
    turned = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * torch.polar(torch.ones_like(angle), angle)
    y[..., first], y[..., second] = turned.real, turned.imag
    return y
