"""The operators of language-model serving whose time is measured: rotary positions, a paged key/value cache, attention over it, and eviction from it.

Every sequence of a batch owns a row of a page table; its keys and values lie in pages ``[pages, kv_heads, page_size, head_dim]`` of 16-bit
values or of 8-bit codes with one scale per token and head.  The tokens of a step are packed, ``[tokens, heads, head_dim]``, those of sequence
``s`` at ``query_offsets[s]:query_offsets[s + 1]``, and are the last ones of that sequence's ``lengths[s]``.  The families:

``rotate``   queries or keys rotated by their positions; with ``train`` also the gradient
``append``   one step's queries and keys rotated, keys and values written to their pages
``attend``   the new tokens' attention over the cached keys under the causal rule (and a window)
``weigh``    what attention the cached keys of each head have received from the new tokens
``evict``    the tokens of most accumulated weight, and the most recent ones, moved to pages of their own
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BASE = 10000.0
DEFAULTS = {"head_dim": 128, "dtype": "bf16", "page": 16, "quantized": False, "batch": 1, "chunk": 1, "window": 0, "scaling": "none", "interleaved": False}


def _case(family, name=None, **more):
    case = {"family": family, **DEFAULTS, **more}
    return case if name is None else {"name": name, **case}


def listed():
    return [
        # The queries of one generation step of 64 requests of a long-context model, frequencies scaled by parts.
        _case("rotate", "rotate_step_b64", layout="tokens", q_heads=32, length=64, rotary_dim=128, scaling="parts", train=False),
        # A training pass over the first half of every head's channels, neighbours in pairs, with the gradient.
        _case("rotate", "rotate_train_16k", layout="hnd", q_heads=16, length=16384, batch=2, rotary_dim=64, interleaved=True, train=True),
        # One generation step of 64 requests: queries and keys rotated, one token of each appended.
        _case("append", "append_step_b64", q_heads=32, kv_heads=8, batch=64, length=4096, rotary_dim=128, dtype="f16"),
        # Prompts of ragged length, 8192 tokens together, stored as 8-bit codes.
        _case("append", "append_prompts_8k_int8", q_heads=32, kv_heads=8, batch=5, chunk=2720, length=2720, rotary_dim=128, quantized=True),
        # A single request in conversation: one token, time is latency.
        _case("attend", "attend_step_b1_8k", q_heads=16, kv_heads=4, length=8192, page=64),
        # A full server: 32 requests of ragged length up to 32K keys held as 8-bit codes.
        _case("attend", "attend_step_b32_32k_int8", q_heads=32, kv_heads=8, batch=32, length=32768, quantized=True),
        # A step in which half of the requests generate and half take in up to 512 tokens of their prompts; sliding window, heads of 64.
        _case("attend", "attend_mixed_8k_d64", q_heads=32, kv_heads=8, batch=8, chunk=512, length=8192, head_dim=64, dtype="f16", window=2048),
        # 2048 tokens of a long prompt over what is cached of it.
        _case("attend", "attend_chunk_2k_of_32k", q_heads=32, kv_heads=8, chunk=2048, length=32768, page=64),
        # The weight that a generation step of 16 requests gives to what they hold.
        _case("weigh", "weigh_step_b16_16k", q_heads=16, kv_heads=4, batch=16, length=16384, page=32),
        # The weight that the last 1024 tokens of two prompts give to all 16K.
        _case("weigh", "weigh_prompt_1k_of_16k", q_heads=32, kv_heads=8, batch=2, chunk=1024, length=16384, dtype="f16", page=64),
        # One request shortened to a quarter.
        _case("evict", "evict_b1_4k", kv_heads=8, length=4096, budget=1024, recent=128, dtype="f16"),
        # A batch of long requests cut down together.
        _case("evict", "evict_b16_16k", kv_heads=8, batch=16, length=16384, budget=4096, recent=256, page=32),
    ]


def draw(rng):
    most_flops = max(work(c)["flops"] for c in listed())
    most_bytes = max(work(c)["bytes"] for c in listed())

    def spread(low, high):
        return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))

    while True:
        family = rng.choice(("rotate", "append", "attend", "attend", "attend", "weigh", "weigh", "evict"))
        q_heads, kv_heads = rng.choice(((16, 4), (16, 16), (32, 8), (40, 40), (8, 1)))
        head_dim, dtype, page = rng.choice((64, 128, 128, 128, 256)), rng.choice(("bf16", "bf16", "f16")), rng.choice((16, 16, 32, 64, 128))
        if family == "rotate":
            case = _case(family, layout=rng.choice(("tokens", "hnd")), q_heads=q_heads, length=spread(1, 32768), batch=1, head_dim=head_dim,
                         rotary_dim=rng.choice((head_dim, head_dim, head_dim // 2)), interleaved=rng.random() < 0.5, dtype=rng.choice(("bf16", "f16", "f32")),
                         scaling=rng.choice(("none", "linear", "base", "parts")), train=rng.random() < 0.5)
            if case["layout"] == "hnd":
                case["batch"] = rng.choice((1, 2, 4))
        else:
            case = _case(family, kv_heads=kv_heads, batch=spread(1, 64), length=spread(64, 32768), head_dim=head_dim, dtype=dtype, page=page,
                         quantized=rng.random() < 0.35)
            if family == "evict":
                case["budget"] = spread(32, case["length"])
                case["recent"] = rng.randrange(0, case["budget"] + 1)
            else:
                case["q_heads"] = q_heads
                case["chunk"] = 1 if rng.random() < 0.4 else spread(2, min(2048, case["length"]))
            if family == "append":
                case.update(rotary_dim=rng.choice((head_dim, head_dim // 2)), interleaved=rng.random() < 0.3, scaling=rng.choice(("none", "linear", "parts")))
            if family == "attend" and rng.random() < 0.25:
                case["window"] = spread(16, case["length"])
        # what the plain form holds at once: scores of padded chunks, the gathered cache in 32 bits
        plain = 0
        if family in ("attend", "weigh"):
            plain = 4 * case["batch"] * case["length"] * (3 * q_heads * case["chunk"] + 4 * kv_heads * head_dim)
        elif family in ("evict", "append"):
            plain = 8 * case["batch"] * case["length"] * kv_heads * head_dim
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
    if case["family"] == "weigh":
        return [min(n, length) for length in _lengths(case)]
    if case["family"] == "append":
        return [min(length, round(n * (0.2 + 0.8 * i / (b - 1)))) or 1 for i, length in enumerate(_lengths(case))]
    return [1 if i % 2 == 0 else max(1, min(length, round(n * (0.5 + 0.5 * i / (b - 1))))) for i, length in enumerate(_lengths(case))]


def _frequencies(case):
    """Angle per position of each rotated pair, as Python floats: 64 bits."""
    half = case["rotary_dim"] // 2
    base = BASE
    if case["scaling"] == "base":  # the base raised so that the slowest pair turns a fourth as fast
        base *= 4.0 ** (case["rotary_dim"] / (case["rotary_dim"] - 2))
    plain = [base ** (-i / half) for i in range(half)]
    if case["scaling"] == "linear":
        return [f / 4.0 for f in plain]
    if case["scaling"] == "parts":  # fast pairs stay, slow pairs turn a fourth as fast, those between are blended by their turns over the original length
        out = []
        for f in plain:
            turns = 8192 * f / (2 * math.pi)
            blend = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
            out.append(f / 4.0 * (1 - blend) + f * blend)
        return out
    return plain


def _scaling(case):
    return {"none": {}, "linear": {"scaling": "linear", "factor": 4.0}, "base": {"scaling": "base", "factor": 4.0},
            "parts": {"scaling": "parts", "factor": 4.0, "original_length": 8192, "slow_turns": 1.0, "fast_turns": 4.0}}[case["scaling"]]


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, d = DTYPES[case["dtype"]], case["head_dim"]

    def normal(*shape, type=dtype):
        return torch.randn(*shape, device="cuda", generator=g).to(type)

    state = {"case": case}
    if "rotary_dim" in case:
        state["frequencies"] = torch.tensor(_frequencies(case), dtype=torch.float64, device="cuda")
        if own:
            import risaattention_b200 as risa
            state["rotary"] = risa.rotary_table(case["rotary_dim"], base=BASE, device="cuda", **_scaling(case))
    if case["family"] == "rotate":
        n, heads, batch = case["length"], case["q_heads"], case["batch"]
        if case["layout"] == "tokens":
            x = normal(n, heads, d)
            positions = torch.randint(0, 131072, (n,), device="cuda", generator=g, dtype=torch.int32)
        else:
            x = normal(batch, heads, n, d)
            positions = torch.arange(n, device="cuda", dtype=torch.int32) + torch.randint(0, 4096, (batch, 1), device="cuda", generator=g, dtype=torch.int32)
        state.update(x=x, positions=positions)
        if case["train"]:
            state["x"].requires_grad_()
            state["grad"] = normal(*x.shape)
        return state

    kv_heads, page, batch = case["kv_heads"], case["page"], case["batch"]
    order = torch.randperm(batch, generator=torch.Generator().manual_seed(seed)).tolist()
    lengths, chunks = [_lengths(case)[i] for i in order], [_chunks(case)[i] for i in order]
    width = max(-(-n // page) for n in lengths)
    # pages of old tokens lie anywhere in the pool, those that take new tokens (and those that eviction fills) were handed out last
    if case["family"] == "evict":
        fresh = [0] * batch
        targets = -(-case["budget"] // page)
    else:
        fresh = [-(-n // page) - (n - c) // page for n, c in zip(lengths, chunks)]
        targets = 0
    old = [-(-n // page) - f for n, f in zip(lengths, fresh)]
    first = sum(old)
    last = batch * targets if targets else sum(fresh)
    ids = torch.cat((torch.randperm(first, device="cuda", generator=g), first + torch.randperm(last, device="cuda", generator=g))).int()
    table = torch.zeros(batch, width, dtype=torch.int32, device="cuda")
    at_old, at_fresh = 0, first
    for s in range(batch):
        table[s, :old[s]] = ids[at_old:at_old + old[s]]
        at_old += old[s]
        if not targets:
            table[s, old[s]:old[s] + fresh[s]] = ids[at_fresh:at_fresh + fresh[s]]
            at_fresh += fresh[s]
    shape = (first + last, kv_heads, page, d)
    if case["quantized"]:
        keys, values = (torch.randint(-127, 128, shape, device="cuda", generator=g, dtype=torch.int8) for _ in range(2))
        # codes spread over their whole range have a deviation of 73 steps
        scales = [(torch.rand(shape[:3], device="cuda", generator=g) + 0.5) / 73.0 for _ in range(2)]
    else:
        keys, values, scales = normal(*shape), normal(*shape), [None, None]
    if targets:
        for x in (keys, values, *scales):
            if x is not None:
                x[first:] = 0
    offsets = torch.tensor([0] + chunks).cumsum(0).int()
    tokens = int(offsets[-1])
    state.update(keys=keys, values=values, key_scales=scales[0], value_scales=scales[1], table=table, first=first,
                 lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"), offsets=offsets.cuda(), most=max(chunks), tokens=tokens)
    if own:
        import risaattention_b200 as risa
        state["cache"] = risa.KeyValueCache(keys, values, *scales)
    if case["family"] == "evict":
        state["target"] = ids[first:].view(batch, targets)
        # weights as attention gives them: a few keys hold most, many hold next to nothing, some exactly nothing
        weights = torch.exp(3 * torch.randn(batch, kv_heads, width * page, device="cuda", generator=g))
        state["weights"] = weights * (torch.rand(weights.shape, device="cuda", generator=g) < 0.9)
    else:
        state["q"] = normal(tokens, case["q_heads"], d)
        if case["family"] == "append":
            state["k"], state["v"] = normal(tokens, kv_heads, d), normal(tokens, kv_heads, d)
        if case["family"] == "weigh":
            state["lse"] = _attend(state)[1]
    return state


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _turned(x, angles, interleaved, transposed=False):
    """x [..., tokens, channels] in 32 bits with its first 2 * angles.shape[-1] channels rotated by angles [..., tokens, pairs] (64 bits)."""
    cos, sin = angles.cos().float(), angles.sin().float()
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
    pages = state[what][state["table"].long()].float()
    if state["case"]["quantized"]:
        pages *= state[what[:-1] + "_scales"][state["table"].long()][..., None]
    return pages.transpose(1, 2).flatten(2, 3)


def _scores(state):
    """Scaled scores [batch, kv_heads, group, chunk, keys] of the padded chunks, -inf where a key is hidden or a query does not exist."""
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
        hidden |= key <= position[..., None] - case["window"]
    return scores.masked_fill_(hidden[:, None, None], -torch.inf)


def _packed(x, state):
    """[batch, kv_heads, group, chunk, ...] of the padded chunks as [tokens, q_heads, ...]."""
    s, i, _ = _sequences(state)
    return x.movedim(3, 1).flatten(2, 3)[s, i]


def _attend(state):
    scores = _scores(state)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)  # rows that see nothing
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    value = _cached(state, "values")
    out = (scores.flatten(2, 3) @ value).view(*scores.shape[:-1], -1) / total.clamp_min(1e-30)
    return _packed(out, state).to(state["q"].dtype), _packed((total.log() + top).squeeze(-1), state)


def _weigh(state):
    s, i, _ = _sequences(state)
    case = state["case"]
    group = case["q_heads"] // case["kv_heads"]
    lse = torch.zeros(case["batch"], state["most"], case["q_heads"], device="cuda")
    lse[s, i] = state["lse"]
    lse = lse.view(case["batch"], -1, case["kv_heads"], group).permute(0, 2, 3, 1)
    return _scores(state).sub_(lse[..., None]).exp_().sum((2, 3))


def _quantized(x):
    """Codes (as 32-bit floats) and scales of every row: absolute maximum over 127, rounded to nearest even."""
    scale = x.abs().amax(-1) / 127.0
    return torch.where(scale[..., None] > 0, x / scale[..., None], 0.0).round(), scale


def _append(state):
    case = state["case"]
    s, _, place = _sequences(state)
    page, slot = state["table"][s, place // case["page"]].long(), (place % case["page"]).long()
    angles = (place.double()[:, None] * state["frequencies"])[:, None]
    q = _turned(state["q"].float(), angles, case["interleaved"]).to(state["q"].dtype)
    k, v = _turned(state["k"].float(), angles, case["interleaved"]), state["v"].float()
    if case["quantized"]:
        (k, ks), (v, vs) = _quantized(k), _quantized(v)
        state["key_scales"][page, :, slot], state["value_scales"][page, :, slot] = ks, vs
    state["keys"][page, :, slot], state["values"][page, :, slot] = k.to(state["keys"].dtype), v.to(state["values"].dtype)
    return q


def _stored(state, dtype):
    """The last pages of the pool, which took what was written, as the values they stand for."""
    first = state["first"]
    if not state["case"]["quantized"]:
        return state["keys"][first:], state["values"][first:]
    return tuple((state[w][first:] * state[w[:-1] + "_scales"][first:, ..., None]).to(dtype) for w in ("keys", "values"))


def _evict(state):
    case, weights = state["case"], state["weights"]
    batch, kv_heads, width = weights.shape
    length = state["lengths"].long()[:, None, None]
    key = torch.arange(width, device="cuda")
    count = length.clamp_max(case["budget"])
    # most recent first, then by weight; equal weights from the lowest index on
    rank = torch.where(key < length, (key >= length - case["recent"]).int(), -1).expand(batch, kv_heads, width)
    by_weight = weights.sort(dim=-1, descending=True, stable=True).indices
    order = by_weight.gather(-1, rank.gather(-1, by_weight).sort(dim=-1, descending=True, stable=True).indices)[..., :case["budget"]]
    place = torch.arange(order.shape[-1], device="cuda")
    kept = torch.where(place < count, order, width).sort(-1).values
    there = place < count
    source = torch.where(there, kept, 0)
    kept = torch.where(there, kept, -1)
    if order.shape[-1] < case["budget"]:
        kept = torch.nn.functional.pad(kept, (0, case["budget"] - order.shape[-1]), value=-1)
    b, h = torch.arange(batch, device="cuda")[:, None, None], torch.arange(kv_heads, device="cuda")[:, None]
    page, slot = state["table"][b, source // case["page"]].long(), source % case["page"]
    to_page, to_slot = state["target"][b, place // case["page"]].long(), place % case["page"]
    pools = [state[w] for w in ("keys", "values", "key_scales", "value_scales") if state[w] is not None]
    for pool in pools:
        seen = there[..., None] if pool.ndim == 4 else there
        pool[to_page, h, to_slot] = torch.where(seen, pool[page, h, slot], pool[to_page, h, to_slot])
    new = torch.zeros(batch, kv_heads, state["target"].shape[1] * case["page"], device="cuda")
    new[..., :order.shape[-1]] = torch.where(there, weights.gather(-1, source), 0.0)
    return kept.int(), count.view(-1).int(), new


def run(state):
    case, family = state["case"], state["case"]["family"]
    window = case["window"] or None
    if own:
        import risaattention_b200 as risa
    if family == "rotate":
        x = state["x"]
        if own:
            out = risa.rotate_positions(x, state["positions"], state["rotary"], interleaved=case["interleaved"])
            return (out.detach(), torch.autograd.grad(out, x, state["grad"])[0]) if case["train"] else out
        angles = state["positions"].double()[..., None] * state["frequencies"]
        angles = angles[:, None]  # [tokens, 1, pairs] beside [tokens, heads, channels], [batch, 1, tokens, pairs] beside [batch, heads, tokens, channels]
        out = _turned(x.detach().float(), angles, case["interleaved"]).to(x.dtype)
        return (out, _turned(state["grad"].float(), angles, case["interleaved"], True).to(x.dtype)) if case["train"] else out
    if family == "append":
        if own:
            q = risa.append_to_cache(state["cache"], state["k"], state["v"], state["table"], state["lengths"], query_offsets=state["offsets"], q=state["q"],
                                     rotary=state["rotary"], interleaved=case["interleaved"])
        else:
            q = _append(state)
        return (q, *_stored(state, q.dtype))
    if family == "attend":
        # a step of one token for each sequence needs no offsets
        offsets = state["offsets"] if state["most"] > 1 else None
        if own:
            return risa.paged_attention(state["q"], state["cache"], state["table"], state["lengths"], query_offsets=offsets, window=window, return_lse=True)
        return _attend(state)
    if family == "weigh":
        if own:
            offsets = state["offsets"] if state["most"] > 1 else None
            return risa.cached_key_weights(state["q"], state["lse"], state["cache"], state["table"], state["lengths"], query_offsets=offsets, window=window)
        return _weigh(state)
    if own:
        result = risa.evict_from_cache(state["cache"], state["table"], state["lengths"], state["weights"], state["target"], budget=case["budget"], recent=case["recent"])
    else:
        result = _evict(state)
    return (*result, *_stored(state, DTYPES[case["dtype"]]))


def work(case):
    """Inputs read once and outputs written once; two operations per multiply-add of a visible (query, key, channel)."""
    size, d = 4 if case["dtype"] == "f32" else 2, case["head_dim"]
    if case["family"] == "rotate":
        values = case["batch"] * case["q_heads"] * case["length"] * d
        positions = case["batch"] * case["length"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * (2 * values * size) + 4 * positions + 4 * case["rotary_dim"], "flops": passes * 3 * values * case["rotary_dim"] / d}
    lengths, kv_heads = _lengths(case), case["kv_heads"]
    row = d + 4 if case["quantized"] else d * size  # one token of one head in the cache
    if case["family"] == "evict":
        kept = kv_heads * sum(min(n, case["budget"]) for n in lengths)
        return {"bytes": 4 * row * kept + 4 * kv_heads * sum(lengths) + 8 * kept + 4 * kept / case["page"], "flops": kv_heads * sum(lengths)}
    chunks, window = _chunks(case), case["window"]
    tokens, q_heads = sum(chunks), case["q_heads"]
    table = 4 * sum(-(-n // case["page"]) for n in lengths)
    if case["family"] == "append":
        moved = tokens * (2 * q_heads * d * size + 2 * kv_heads * (d * size + row))
        return {"bytes": moved, "flops": 3 * tokens * (q_heads + kv_heads) * case["rotary_dim"]}
    pairs = keys = 0
    for n, c in zip(lengths, chunks):
        seen = [min(n - c + i + 1, window or n) for i in range(c)]
        pairs += q_heads * sum(seen)
        keys += kv_heads * (n if not window else min(n, window + c - 1))
    if case["family"] == "attend":
        return {"bytes": 2 * keys * row + tokens * q_heads * (2 * d * size + 4) + table, "flops": 4 * pairs * d}
    width = max(-(-n // case["page"]) for n in lengths) * case["page"]
    return {"bytes": keys * row + tokens * q_heads * (d * size + 4) + table + 4 * kv_heads * case["batch"] * width, "flops": 2 * pairs * d}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["family"] == "rotate":
        positions = state["positions"].double()
        positions = positions[:, None] if case["layout"] == "tokens" else positions[:, None, :]  # one per head
        out = _exact_rotation(state["x"].detach(), positions, state["frequencies"], case, 1)
        return (out, _exact_rotation(state["grad"], positions, state["frequencies"], case, -1)) if case["train"] else out
    if case["family"] == "evict":
        return _exact_eviction(state)
    offsets, lengths = state["offsets"].tolist(), state["lengths"].tolist()
    if case["family"] == "append":
        return _exact_append(state, offsets, lengths)
    d, group = case["head_dim"], case["q_heads"] // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(state["q"].shape[:2], dtype=torch.float64, device="cuda")
    weights = torch.zeros(case["batch"], case["kv_heads"], state["table"].shape[1] * case["page"], dtype=torch.float64, device="cuda")
    for s, n in enumerate(lengths):
        rows = slice(offsets[s], offsets[s + 1])
        pages = state["table"][s, :-(-n // case["page"])].long()
        position = torch.arange(n - (offsets[s + 1] - offsets[s]), n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        seen = (key <= position) & ((key > position - case["window"]) if case["window"] else True)
        for h in range(case["kv_heads"]):
            k, v = (_exact_rows(state, w, pages, h)[:n] for w in ("keys", "values"))
            for head in range(h * group, (h + 1) * group):
                x = state["q"][rows, head].double() @ k.T / math.sqrt(d)
                x[~seen] = -torch.inf
                if case["family"] == "weigh":
                    weights[s, h, :n] += (x - state["lse"][rows, head].double()[:, None]).exp().sum(0)
                else:
                    lse[rows, head] = x.logsumexp(-1)
                    out[rows, head] = (x - lse[rows, head][:, None]).exp() @ v
    return weights if case["family"] == "weigh" else (out, lse)


def _exact_rows(state, what, pages, head):
    rows = state[what][pages, head].double()
    if state["case"]["quantized"]:
        rows = rows * state[what[:-1] + "_scales"][pages, head].double()[..., None]
    return rows.flatten(0, 1)


def _exact_rotation(x, positions, frequencies, case, sign):
    """Each pair as a complex number, times e^(i angle)."""
    r = case["rotary_dim"]
    y = x.double().clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if case["interleaved"] else (slice(0, r // 2), slice(r // 2, r))
    angle = positions[..., None] * frequencies * sign
    turned = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * torch.polar(torch.ones_like(angle), angle)
    y[..., first], y[..., second] = turned.real, turned.imag
    return y


def _exact_append(state, offsets, lengths):
    case, dtype = state["case"], torch.float64
    place = torch.cat([torch.arange(n - (b - a), n, device="cuda") for n, a, b in zip(lengths, offsets, offsets[1:])])
    owner = torch.cat([torch.full((b - a,), s, device="cuda") for s, (a, b) in enumerate(zip(offsets, offsets[1:]))])
    page, slot = state["table"][owner, place // case["page"]].long() - state["first"], place % case["page"]
    turned = [_exact_rotation(state[x], place.double()[:, None], state["frequencies"], case, 1) for x in ("q", "k")]
    new = {"keys": turned[1], "values": state["v"].double()}
    out = [turned[0]]
    for what in ("keys", "values"):
        stored = state[what][state["first"]:].to(dtype)
        if case["quantized"]:
            stored *= state[what[:-1] + "_scales"][state["first"]:].to(dtype)[..., None]
            step = new[what].abs().amax(-1, keepdim=True) / 127
            new[what] = (new[what] / step).round() * step
        stored[page, :, slot] = new[what]
        out.append(stored)
    return tuple(out)


def _exact_eviction(state):
    case, lengths = state["case"], state["lengths"].tolist()
    weights = torch.zeros(case["batch"], case["kv_heads"], state["target"].shape[1] * case["page"], dtype=torch.float64, device="cuda")
    stored = {w: state[w][state["first"]:].double() for w in ("keys", "values")}
    for s, n in enumerate(lengths):
        pages, to = state["table"][s, :-(-n // case["page"])].long(), state["target"][s].long() - state["first"]
        count, recent = min(n, case["budget"]), min(n, case["recent"])
        for h in range(case["kv_heads"]):
            w = state["weights"][s, h, :n]
            chosen = w[:n - recent].sort(descending=True, stable=True).indices[:count - recent]
            kept = torch.cat((chosen.sort().values, torch.arange(n - recent, n, device="cuda")))
            weights[s, h, :count] = w[kept].double()
            place = torch.arange(count, device="cuda")
            for what, pool in stored.items():
                pool[to[place // case["page"]], h, place % case["page"]] = _exact_rows(state, what, pages, h)[kept]
    return None, None, weights, stored["keys"], stored["values"]
