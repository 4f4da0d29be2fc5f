"""Pages of a cache shared, handed out, given back and moved, against a plain account of them kept on the host."""
import four_bits_util as F
import pytest
import serving_util as U
import torch

import risaattention_b200 as risa
from risaattention_b200 import _backend

pytestmark = pytest.mark.gpu

KINDS = [torch.bfloat16, torch.float16, torch.int8, torch.uint8]


@pytest.fixture(autouse=True)
def no_status():
    yield
    torch.cuda.synchronize()
    _backend._C.device_status()


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def filled(pages, heads, page, d, kind, seed=0):
    """A cache with something else in every byte that is compared, and no NaN."""
    cache = risa.allocate_key_value_cache(pages, heads, page, d, dtype=kind)
    g = torch.Generator("cuda").manual_seed(seed)
    for x in cache.tensors:
        if x is not None:
            x.copy_(torch.randn(x.shape, device="cuda", generator=g) if x.is_floating_point() else torch.randint(0, 120, x.shape, device="cuda", generator=g))
    return cache


def rows_of(cache, page, n):
    """Everything that the first n tokens of a page hold, [heads, n, bytes]."""
    out = []
    for pool, scales in ((cache.keys, cache.key_scales), (cache.values, cache.value_scales)):
        out.append(pool[page, :, :n].contiguous().view(torch.uint8))
        if cache.keys.dtype == torch.int8:
            out.append(scales[page, :, :n, None].contiguous().view(torch.uint8))
        elif cache.keys.dtype == torch.uint8:
            p = cache.page_size
            out += [scales[page, :, :n, None], scales[page, :, p:].unflatten(-1, (p, -1))[:, :n]]
    return torch.cat([x.flatten(2) for x in out], -1).cpu()


class Account:
    """Tables, lengths and counts kept in Python, and what rows a page must hold."""

    def __init__(self, pages, page, width):
        self.references, self.page, self.width = [0] * pages, page, width
        self.copies = []

    def pages_for(self, n):
        return -(-n // self.page)

    def fork(self, table, lengths, parents):
        rows, out = [], []
        for p in parents:
            n = lengths[p] if 0 <= p < len(lengths) else 0
            held = table[p][:self.pages_for(n)] if n else []
            for i in held:
                self.references[i] += 1
            rows.append(held + [-1] * (self.width - len(held)))
            out.append(n)
        return rows, out

    def resize(self, table, lengths, wanted):
        free = [i for i, n in enumerate(self.references) if n == 0]
        before = list(self.references)
        granted = []
        for row, n, m in zip(table, lengths, wanted):
            m = min(max(m, 0), self.width * self.page)
            held, needed = self.pages_for(n), self.pages_for(m)
            if m > n:
                shared = n % self.page and before[row[held - 1]] > 1
                if shared:
                    if not free:
                        granted.append(n)
                        continue
                    new = free.pop(0)
                    self.copies.append((row[held - 1], new, n % self.page))
                    self.references[row[held - 1]] -= 1
                    self.references[new] = 1
                    row[held - 1] = new
                while held < needed and free:
                    row[held] = free.pop(0)
                    self.references[row[held]] = 1
                    held += 1
                granted.append(min(m, held * self.page))
            else:
                for i in range(needed, held):
                    self.references[row[i]] -= 1
                    row[i] = -1
                granted.append(m)
        return granted


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page,d", [(16, 64), (64, 128), (32, 256)])
def test_a_history_of_forks_and_sizes(kind, page, d):
    pages, width = 60, 12
    cache = filled(pages, 3, page, d, kind)
    references = torch.zeros(pages, dtype=torch.int32, device="cuda")
    account = Account(pages, page, width)
    table, lengths = [[-1] * width for _ in range(3)], [0, 0, 0]
    device_table, device_lengths = ints(table), ints(lengths)
    g = torch.Generator().manual_seed(page)

    def resize(wanted):
        nonlocal lengths, device_lengths
        account.copies = []
        was = [rows_of(cache, p, page) for p in range(pages)]
        lengths = account.resize(table, lengths, wanted)
        device_lengths = risa.resize_sequences(cache, references, device_table, device_lengths, ints(wanted))
        assert device_lengths.tolist() == lengths and references.tolist() == account.references
        for row, got, n in zip(table, device_table.tolist(), lengths):
            assert got[:account.pages_for(n)] == row[:account.pages_for(n)]
        changed = {}
        for source, to, n in account.copies:
            assert torch.equal(rows_of(cache, to, n), was[source][:, :n])
            changed[to] = n
        for p in range(pages):  # nothing else was written
            n = changed.get(p, 0)
            assert torch.equal(rows_of(cache, p, page)[:, n:], was[p][:, n:])

    def fork(parents):
        nonlocal table, lengths, device_table, device_lengths
        table, lengths = account.fork(table, lengths, parents)
        device_table, device_lengths = risa.fork_sequences(cache, references, device_table, device_lengths, ints(parents))
        assert device_table.tolist() == table and device_lengths.tolist() == lengths and references.tolist() == account.references

    resize([page * 2 + 5, page, 3])
    fork([0, 0, 1, 2, -1, 0, 99])
    resize([n + 1 for n in lengths])
    resize([n + 3 * page if i % 2 else max(0, n - page - 2) for i, n in enumerate(lengths)])
    fork([1, 1, 3, 0])
    resize([0, lengths[1] + 2, lengths[2] - 1, page * 100])      # more than a row of the table holds
    fork([3, 1, 2, 3, 1])
    resize([n + 5 * page for n in lengths])                      # more than there are pages
    resize([int(x) for x in torch.randint(0, width * page, (5,), generator=g)])
    resize([0] * 5)


def test_lowest_pages_first_and_none_given_back_in_the_same_call():
    cache = filled(6, 1, 16, 64, torch.bfloat16)
    references, table = ints([0, 1, 0, 1, 0, 0]), ints([[1, -1], [3, -1], [-1, -1]])
    granted = risa.resize_sequences(cache, references, table, ints([16, 10, 0]), ints([0, 32, 20]))
    assert granted.tolist() == [0, 32, 20] and table.tolist() == [[-1, -1], [3, 0], [2, 4]]
    assert references.tolist() == [1, 0, 1, 1, 1, 0]


def test_no_page_for_a_shared_one():
    cache = filled(2, 1, 16, 64, torch.bfloat16)
    references, table = ints([2, 1]), ints([[0, 1], [0, -1]])
    granted = risa.resize_sequences(cache, references, table, ints([32, 7]), ints([32, 9]))
    assert granted.tolist() == [32, 7] and references.tolist() == [2, 1] and table.tolist() == [[0, 1], [0, -1]]


def test_many_sequences_and_pages():
    """More sequences than a block has threads, more pages than it looks at in a round."""
    batch, pages = 2500, 40000
    cache = filled(pages, 1, 16, 64, torch.uint8)
    references = torch.ones(pages, dtype=torch.int32, device="cuda")
    g = torch.Generator("cuda").manual_seed(1)
    free = torch.randperm(pages, device="cuda", generator=g)[:9000]
    references[free] = 0
    wanted = torch.randint(0, 7 * 16, (batch,), device="cuda", generator=g, dtype=torch.int32)
    table = torch.full((batch, 6), -1, dtype=torch.int32, device="cuda")
    zero = torch.zeros(batch, dtype=torch.int32, device="cuda")
    granted = risa.resize_sequences(cache, references, table, zero, wanted)
    order = free.sort().values.tolist()
    account = Account(pages, 16, 6)
    account.references = [1] * pages
    for i in order:
        account.references[i] = 0
    rows = [[-1] * 6 for _ in range(batch)]
    want = account.resize(rows, [0] * batch, wanted.tolist())
    assert granted.tolist() == want and references.tolist() == account.references
    assert [r[:-(-n // 16)] for r, n in zip(table.tolist(), want)] == [r[:-(-n // 16)] for r, n in zip(rows, want)]
    target = risa.allocate_key_value_cache(int((references > 0).sum()) + 5, 1, 16, 64, dtype=torch.uint8)
    new, counts, used = risa.compact_cache(cache, references, table, granted, target)
    in_use = (references > 0).nonzero()[:, 0]
    place = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
    place[in_use] = torch.arange(len(in_use), device="cuda", dtype=torch.int32)
    assert int(used) == len(in_use) and torch.equal(counts[:len(in_use)], references[in_use]) and not bool(counts[len(in_use):].any())
    held = torch.arange(6, device="cuda") < ((granted + 15) // 16)[:, None]
    assert torch.equal(new, torch.where(held, place[table.clamp_min(0).long()], -1))
    for to, source in zip(target.tensors, cache.tensors):
        assert torch.equal(to[:len(in_use)], source[in_use]) and not bool(to[len(in_use):].any())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,page,d", [(3, 16, 64), (8, 128, 128), (1, 32, 256)])
def test_compaction(kind, heads, page, d):
    cache = filled(23, heads, page, d, kind)
    references = ints([0, 2, 0, 0, 1, 1, 0, 0, 0, 3, 1, 0, 0, 0, 0, 0, 0, 1, 0, 0, 0, 0, 1])
    table, lengths = ints([[9, 4, 1], [9, 22, 7], [17, 3, 3], [5, 10, 9]]), ints([3 * page, page + 1, page, 2 * page + 1])
    used = [1, 4, 5, 9, 10, 17, 22]
    for room in (7, 9, 4):
        target = filled(room, heads, page, d, kind, seed=5)
        before = [None if x is None else x.clone() for x in target.tensors]
        new, counts, n = risa.compact_cache(cache, references, table, lengths, target)
        assert int(n) == 7
        place = {p: i for i, p in enumerate(used) if i < room}
        assert counts.tolist() == ([references[p].item() for p in used] + [0] * room)[:room]
        assert new.tolist() == [[place.get(9, -1), place.get(4, -1), place.get(1, -1)], [place.get(9, -1), place.get(22, -1), -1], [place.get(17, -1), -1, -1],
                                [place.get(5, -1), place.get(10, -1), place.get(9, -1)]]
        for to, source, old in zip(target.tensors, cache.tensors, before):
            if to is not None:
                kept = min(room, 7)
                assert torch.equal(to[:kept], source[used[:kept]]) and torch.equal(to[kept:], old[kept:])


def test_entries_outside_the_pool_are_reported():
    cache = filled(4, 1, 16, 64, torch.bfloat16)
    table, lengths = ints([[0, 9], [-3, 1]]), ints([20, 20])
    for call in (lambda r: risa.fork_sequences(cache, r, table, lengths, ints([1, 0])), lambda r: risa.resize_sequences(cache, r, table.clone(), lengths, ints([0, 0])),
                 lambda r: risa.resize_sequences(cache, r, ints([[0, 9], [1, -7]]), lengths, ints([21, 21])),
                 lambda r: risa.compact_cache(cache, r, table, lengths, filled(4, 1, 16, 64, torch.bfloat16))):
        references = ints([1, 1, 0, 0])
        call(references)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside the pool"):
            _backend._C.device_status()


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.uint8])
def test_children_of_a_prompt(kind, monkeypatch):
    """A prompt read once and answered four times, from pages that the answers share, captured and replayed; then one answer moves
    to a smaller pool.  Every answer is what it would be over a cache of its own."""
    monkeypatch.setattr(U, "cached", F.cached)
    d, page, heads, q_heads = 64, 16, 2, 4
    cache = risa.allocate_key_value_cache(40, heads, page, d, dtype=kind)
    references = torch.zeros(40, dtype=torch.int32, device="cuda")
    table, lengths = torch.full((1, 8), -1, dtype=torch.int32, device="cuda"), ints([0])
    lengths = risa.resize_sequences(cache, references, table, lengths, ints([53]))
    k, v = (torch.randn(53, heads, d, device="cuda").bfloat16() for _ in range(2))
    risa.append_to_cache(cache, k, v, table, lengths, query_offsets=ints([0, 53]))
    tables, sizes = risa.fork_sequences(cache, references, table, lengths, ints([0, 0, 0, 0]))
    risa.resize_sequences(cache, references, table, lengths, ints([0]))  # the prompt itself leaves
    assert int(references.max()) == 4
    k, v = (torch.randn(4, heads, d, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(4, q_heads, d, device="cuda").bfloat16()

    def step():
        grown = risa.resize_sequences(cache, references, tables, sizes, sizes + 1)
        risa.append_to_cache(cache, k, v, tables, grown)
        out, lse = risa.paged_attention(q, cache, tables, grown, return_lse=True)
        sizes.copy_(grown)
        return out, lse
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = step()
    torch.cuda.synchronize()
    own = [[] for _ in range(4)]

    def check():
        torch.cuda.synchronize()
        F.assert_attention(U.Batch(cache, tables, sizes, torch.arange(5), [1] * 4, q, 0), out, lse)
        keys, values = risa.read_from_cache(cache, tables, sizes, dtype=torch.bfloat16)
        for s in range(4):
            own[s].append((keys[s].clone(), values[s].clone()))
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for _ in range(14):
        for x in (k, v, q):
            x.normal_()
        graph.replay()
        check()
    assert sizes.tolist() == [68] * 4 and sorted(references.tolist())[-8:] == [1] * 5 + [4] * 3
    # every child still holds the prompt and its own tokens
    offsets = ints([0, 68, 136, 204, 272])
    keys, values = risa.read_from_cache(cache, tables, sizes, query_offsets=offsets, tokens=272, dtype=torch.bfloat16)
    for s in range(4):
        for i, (a, b) in enumerate(own[s]):
            assert torch.equal(keys[68 * s + 53 + i], a) and torch.equal(values[68 * s + 53 + i], b)
        assert torch.equal(keys[68 * s:68 * s + 53], keys[:53])
    left = risa.resize_sequences(cache, references, tables, sizes, ints([0, 68, 0, 0]))
    target = risa.allocate_key_value_cache(6, heads, page, d, dtype=kind)
    new, counts, used = risa.compact_cache(cache, references, tables, left, target)
    assert int(used) == 5 and counts.tolist() == [1] * 5 + [0]
    out, lse = risa.paged_attention(q, target, new, left, return_lse=True)
    assert left.tolist() == [0, 68, 0, 0]
    F.assert_attention(U.Batch(target, new, left, torch.arange(5), [1] * 4, q, 0), out, lse)
    again = risa.read_from_cache(target, new, left, query_offsets=ints([0, 0, 68, 68, 68]), tokens=68, dtype=torch.bfloat16)
    assert torch.equal(again[0], keys[68:136]) and torch.equal(again[1], values[68:136])


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_another_device_than_the_current_one():
    for device in ("cuda:0", "cuda:1"):
        cache = risa.allocate_key_value_cache(9, 2, 16, 64, dtype=torch.uint8, device=device)
        references, table = torch.zeros(9, dtype=torch.int32, device=device), torch.full((2, 3), -1, dtype=torch.int32, device=device)
        sizes = risa.resize_sequences(cache, references, table, torch.zeros(2, dtype=torch.int32, device=device), torch.tensor([20, 40], dtype=torch.int32, device=device))
        children, lengths = risa.fork_sequences(cache, references, table, sizes, torch.tensor([1], dtype=torch.int32, device=device))
        moved = risa.compact_cache(cache, references, children, lengths, risa.allocate_key_value_cache(5, 2, 16, 64, dtype=torch.uint8, device=device))
        assert table.tolist() == [[0, 1, -1], [2, 3, 4]] and children.tolist() == [[2, 3, 4]] and moved.page_table.tolist() == [[2, 3, 4]]
